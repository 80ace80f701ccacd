// Products of float matrices (fp32, fp16, bf16) with fp32 sums: what the kernels and the entries share.
//
//     forward   y[t][n]  = act(sum_k x[t][k] w[n][k] + b[n]) + r[t][n]
//     SwiGLU    mid[t][i] = silu(x[t] . w_gate[i]) * (x[t] . w_up[i])
//     input     gx[t][k] = sum_n gz[t][n] w[n][k]
//     weight    gw[n][k] = sum_t gz[t][n] x[t][k]
//
// of one matrix, or of stacked experts' matrices and rows sorted by expert.
#pragma once

#include "mxfp4_common.hpp"

namespace jjo {

enum RowsMode { kRowsForward, kRowsSwiglu, kRowsInput, kRowsWeight };

// What follows a sum: bias, the sum kept, activation, residual.  SwiGLU: pre is gate|up.
struct RowsEpilogue {
    const void *bias = nullptr, *residual = nullptr;
    int64_t residual_stride = 0;
    void *pre = nullptr;
    int act = JJO_ACT_NONE;
};

// out[Q rows][P columns] = Qmat . Pmat^T over K: of either operand either the sums' elements of a row
// are contiguous (forward), or the rows' of an element are (weight; input: of P).
struct RowsMm {
    const void *p, *p2;  // p2: the up matrix (SwiGLU), or the operand of the sums' second half (input)
    const void *q, *rest;  // rest: q's other terms, terms - 1 matrices (weight)
    int64_t rest_plane;    // elements from one of these to the next
    float first_scale;     // of the sums over q, before those over rest are added (terms 2)
    int64_t ldp, ldq;  // elements from one memory row to the next
    void *y, *y2;      // y2: of the second half's output rows (weight)
    int64_t ldy;
    int P, Q, K;
    int halves;              // 2: input sums over p, then over p2; weight has rows of y, then of y2
    int terms;               // of q in a weight's sums, the smallest first: q, then those of rest
    const int32_t *offsets;  // [n_experts + 1], or nullptr
    int n_experts, M;        // M: sorted rows
    int64_t expert_stride;   // elements of a matrix (of an expert's part of y: weight)
    bool wide;               // y is fp32 (weight)
    int slices;              // of the sums, each in its own part[Q][P] (SwiGLU: [Q][2P])
    float *part;
    RowsEpilogue epi;
    int tiles_p, tiles_q;  // of the launch
};

// ---- activations.  sigmoid and tanh through the hardware's exp2 and reciprocal (1 ulp each):
// 0.5 (1 + tanh u) = sigmoid(2u).  The normal distribution by erfc, so that its lower tail keeps its
// relative precision, for results of 16 bits as well.
__device__ __forceinline__ float rows_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896f * z));
}
constexpr float kGeluC = 0.797884560802865f, kGeluA = 0.044715f;  // sqrt(2 / pi)

// erfc(x).  For results of 16 bits e^(x^2) erfc(x) = t P(t), t = 1 / (1 + 3x/8), x >= 0: P fitted here by weighted
// least squares, the weights raised where the relative error was largest until it was even, over 0 <= x <= 10 (erfc
// leaves fp32 at 9.2).  Relative error at most 1.1e-6, and that of e^(-x^2), whose argument is rounded once: 2^-24 of
// it, 6e-6 at x = 9.  (A third of the instructions of erfcf.)
template <class T>
__device__ __forceinline__ float rows_erfc(float x) {
    if constexpr (sizeof(T) == 4) return erfcf(x);
    const float a = fabsf(x), t = __builtin_amdgcn_rcpf(1.0f + 0.375f * a);
    constexpr float kP[] = {0.21133944f,  0.21568918f, 0.16666459f, 0.28306147f,
                            -0.12959719f, 0.38793775f, -0.13509588f};
    float poly = kP[6];
#pragma unroll
    for (int i = 5; i >= 0; --i) poly = poly * t + kP[i];
    const float tail = t * poly * __builtin_amdgcn_exp2f(-1.44269504088896f * (a * a));
    return x < 0.0f ? 2.0f - tail : tail;
}

template <class T>
__device__ __forceinline__ float rows_act(float z, int act) {
    switch (act) {
        case JJO_ACT_RELU: return z > 0.0f ? z : z != z ? z : 0.0f;
        case JJO_ACT_GELU: return 0.5f * z * rows_erfc<T>(-0.707106781186548f * z);
        case JJO_ACT_GELU_TANH: return z * rows_sigmoid(2.0f * kGeluC * (z + kGeluA * z * z * z));
        case JJO_ACT_SILU: return z * rows_sigmoid(z);
    }
    return z;
}

// The activation's derivative at z (not of relu).
template <class T>
__device__ __forceinline__ float rows_slope(float z, int act) {
    switch (act) {
        case JJO_ACT_GELU:
            return 0.5f * rows_erfc<T>(-0.707106781186548f * z) +
                   z * 0.398942280401433f * __builtin_amdgcn_exp2f(-0.721347520444482f * z * z);
        case JJO_ACT_GELU_TANH: {
            const float s = rows_sigmoid(2.0f * kGeluC * (z + kGeluA * z * z * z));
            // The second term is nothing beyond |z| = 32, where its z^3 would leave fp32 later on.
            const float c = fminf(fmaxf(z, -32.0f), 32.0f);
            return s + c * 2.0f * s * (1.0f - s) * kGeluC * (1.0f + 3.0f * kGeluA * c * c);
        }
        case JJO_ACT_SILU: {
            const float s = rows_sigmoid(z);
            return s * (1.0f + z * (1.0f - s));
        }
    }
    return 1.0f;
}
// A gradient g through an activation: times its derivative at z; of relu g or 0, also where g is infinite.
template <class T>
__device__ __forceinline__ float rows_through(float g, float z, int act) {
    if (act == JJO_ACT_RELU) return z > 0.0f ? g : z != z ? z : 0.0f;
    return g * rows_slope<T>(z, act);
}

// ---- eight consecutive values of a row, n of them inside it, at any alignment
template <class T>
__device__ __forceinline__ void rows_load8(const T *p, int n, float *v) {
    if (n >= 8) {
        const MxVec<T, 8> a = load_any<MxVec<T, 8>>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
    }
}
// A value is rounded to fp32 before it is to T, on every path alike (the compiler would give some paths
// an instruction that multiplies and rounds to fp16 at once, and so results that depend on the path).
template <class T>
__device__ __forceinline__ T rows_round(float v) {
    asm("" : "+v"(v));
    return (T)v;
}
template <class T>
__device__ __forceinline__ void rows_store8(T *p, int n, const float *v) {
    if (n >= 8) {
        MxVec<T, 8> a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a.v[i] = rows_round<T>(v[i]);
        store_any(p, a);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < n) p[i] = rows_round<T>(v[i]);
    }
}
// Eight values as 16 bytes of T, and 16 bytes to any address past the caches.
template <class T>
__device__ __forceinline__ u32x4v rows_pack8(const float *v) {
    MxVec<T, 8> a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] = rows_round<T>(v[i]);
    return __builtin_bit_cast(u32x4v, a);
}
__device__ __forceinline__ void rows_store_past(void *p, u32x4v v) {
    typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));
    __builtin_nontemporal_store((Any)v, (Any *)p);
}

// Sums of columns col.. of a row (n of them) to the output.
template <class T>
__device__ __forceinline__ void rows_finish(const RowsEpilogue &e, float *v, int64_t row, int col, int n, int cols,
                                            void *y, int64_t ldy, bool wide) {
    if (e.bias != nullptr) {
        float b[8];
        rows_load8((const T *)e.bias + col, n, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += b[i];
    }
    if (e.pre != nullptr) rows_store8((T *)e.pre + row * cols + col, n, v);
    if (e.act != JJO_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = rows_act<T>(v[i], e.act);
    }
    if (e.residual != nullptr) {
        float r[8];
        rows_load8((const T *)e.residual + row * e.residual_stride + col, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    if (wide) rows_store8((float *)y + row * ldy + col, n, v);
    else rows_store8((T *)y + row * ldy + col, n, v);
}

__device__ __forceinline__ void rows_swiglu(float *gate, const float *up) {
#pragma unroll
    for (int i = 0; i < 8; ++i) gate[i] = gate[i] * rows_sigmoid(gate[i]) * up[i];
}

template <class T>
__device__ __forceinline__ void rows_finish_swiglu(const RowsEpilogue &e, float *gate, const float *up, int64_t row,
                                                   int col, int n, int cols, void *y) {
    if (e.pre != nullptr) {
        T *const at = (T *)e.pre + row * 2 * cols + col;
        rows_store8(at, n, gate);
        rows_store8(at + cols, n, up);
    }
    rows_swiglu(gate, up);
    rows_store8((T *)y + row * cols + col, n, gate);
}

// ---- launchers (asynchronous; arguments validated by the entries)
// The kernel of a product: LDS tiles of 64 x 64, 128 x 128, 256 columns x 160 rows (forward and input) or 256 x 256
// (the last two 16 bits only), or the direct kernel with `waves` that cut the sums between them (forward and
// SwiGLU); and the slices of the sums that join their fp32 outputs in a second launch.
enum RowsTileKind { kRowsDirect = -1, kRowsTile64, kRowsTile128, kRowsTile160, kRowsTile256, kRowsTileKinds };
struct RowsChoice {
    int tile, waves, slices;
};
// By the sizes alone (the workspace depends on it).  n_experts 0: one matrix.
RowsChoice rows_mm_choose(RowsMode mode, int dtype, int P, int Q, int K, int halves, int n_experts);
hipError_t launch_rows_mm(RowsMode mode, int dtype, const RowsMm &p, hipStream_t stream,
                          const RowsChoice *pinned = nullptr);
// Rows of a product's output (weight: of all matrices), and the bytes of its slices' sums.
int64_t rows_output_rows(RowsMode mode, const RowsMm &p);
int64_t rows_part_bytes(RowsMode mode, const RowsMm &p);


template <class E>
hipError_t rows_mm_run(RowsMode mode, const RowsMm &p, const RowsChoice &c, hipStream_t stream);

// What the rounding of a value to fp16 left is kept times this.  It is below 2^-11 of the value, so that it would be a
// subnormal of fp16 for all values below 2^-3, and lost below 2^-14; of 65504 it is 16, and so 2^15 at most.
constexpr float kRowsRestScale = 2048.0f;
// gz[t] = grad_y[t] * act'(pre[t]) (act none: not written; planes - 1 more matrices behind it: what the rounding
// left, rounded again) and the columns' sums of gz (sums nullable; column_part: rows_column_chunks(T, N) * N floats).
constexpr int kRowsColumns = 512;  // of a workgroup
int rows_column_chunks(int T, int N);
hipError_t launch_rows_act_backward(const void *grad_y, int64_t grad_y_stride, const void *pre, void *gz, int planes,
                                    int64_t plane, int dtype, int act, void *sums, bool sums_wide,
                                    float *column_part, int T, int N, hipStream_t stream);
// grad_gate_up [R][2I] from grad_mid and the saved gate|up, rows below offsets[n_experts].
hipError_t launch_rows_swiglu_backward(const void *grad_mid, const void *gate_up, void *grad_gate_up, int planes,
                                       int64_t plane, int dtype, const int32_t *offsets, int n_experts, int I, int R,
                                       hipStream_t stream);

}  // namespace jjo
