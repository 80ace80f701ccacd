// Shared pieces of the MXFP4 kernels: element types of the activations, the block
// quantizer, and the launchers each translation unit provides.
//
// MXFP4 matrix [rows][cols] (cols % 32 == 0), the OCP microscaling format with e2m1 elements:
//     codes : rows * cols/2 bytes, element 2j of a row in the low nibble of its byte j
//     scales: rows * cols/32 bytes e8m0 behind them; value = e2m1 * 2^(s - 127), s = 255 NaN
// Every block's codes are one aligned 16-byte load and exactly one lane's operand of the
// scaled matrix instruction, whose scale operand is the block's byte as it is stored.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "q4q8_common.hpp"

namespace jjo {

constexpr int kMxBlockBytes = 17;  // 16 bytes of codes and a scale byte

inline int64_t mx_bytes(int64_t rows, int64_t cols) { return rows * (cols / kQK) * kMxBlockBytes; }

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

// ---- activation types: fp32, fp16, bf16 (JJO_DTYPE_*), widened to fp32 exactly and rounded
// to nearest even on the way out.
struct MxF32 {
    typedef float type;
};
struct MxF16 {
    typedef _Float16 type;
};
struct MxBF16 {
    typedef __bf16 type;
};

// Calls F(tag) with the type tag of a JJO_DTYPE_* value (checked by the entries).
template <class F>
inline hipError_t mx_by_dtype(int dtype, F f) {
    if (dtype == JJO_DTYPE_F32) return f(MxF32{});
    if (dtype == JJO_DTYPE_F16) return f(MxF16{});
    return f(MxBF16{});
}

// VEC consecutive elements, loaded or stored in one access.
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) MxVec {
    T v[VEC];
};

// The same at any alignment: one access all the same, over one line more where it crosses one.
template <class V>
__device__ __forceinline__ V load_any(const void *p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <class V>
__device__ __forceinline__ void store_any(void *p, const V &v) {
    __builtin_memcpy(p, &v, sizeof(V));
}

// ---- quantizer.  The scale byte of a block whose largest |x| has the fp32 bits `amax`:
// 2^(floor(log2 amax) - 2), the exponent of e2m1's largest power of two, taken from the
// exponent field (fp32 subnormals and smaller exponents: 2^-127); 255 for a NaN or an infinity.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
    const uint32_t e = amax >> 23;
    return e == 255u ? 255u : e < 2u ? 0u : e - 2u;
}

// 2^(s - 127) as fp32, s <= 254 (s = 0: the subnormal 2^-127).
__device__ __forceinline__ float mx_scale_value(uint32_t s) {
    return __uint_as_float(s == 0u ? 0x00400000u : s << 23);
}

// Eight values to eight codes; `s` is their block's scale byte (255: all codes 0).  The
// conversion divides by the scale (exact) and rounds to nearest even, at most 6.
__device__ __forceinline__ uint32_t mx_codes8(const float *x, uint32_t s) {
    const float sc = mx_scale_value(s == 255u ? 254u : s);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], sc, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], sc, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], sc, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], sc, 3);
    return s == 255u ? 0u : c;
}

// Largest |x| of eight values as fp32 bits (ordered as unsigned; a NaN is above infinity).
__device__ __forceinline__ uint32_t mx_amax8(const float *x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
        m = u > m ? u : m;
    }
    return m;
}

// Maximum over the lane's group of four lanes.
__device__ __forceinline__ uint32_t mx_max_quad(uint32_t m) {
    uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true);  // quad_perm 1,0,3,2
    m = o > m ? o : m;
    o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, true);  // quad_perm 2,3,0,1
    return o > m ? o : m;
}

// Eight consecutive values, one 16-byte load or two.
template <class T>
__device__ __forceinline__ void mx_load8(const T *p, float *x) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const MxVec<T, 8> a = *reinterpret_cast<const MxVec<T, 8> *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a.v[i];
    }
}

// Group `i` of eight values of a matrix of n8 of them, by a quad of lanes per block (n8 % 4 == 0): its
// codes and, from one lane of four, the scale.
template <class T>
__device__ __forceinline__ void mx_quantize8(const T *p, int64_t i, int64_t n8, uint8_t *__restrict__ out) {
    float v[8];
    mx_load8(p, v);
    const uint32_t s = mx_scale_byte(mx_max_quad(mx_amax8(v)));
    reinterpret_cast<uint32_t *>(out)[i] = mx_codes8(v, s);
    if ((threadIdx.x & 3) == 0) out[4 * n8 + (i >> 2)] = (uint8_t)s;
}

// Groups of eight values of one quantizer launch, a thread each: a grid has fewer than 2^32 threads.
constexpr int64_t kMxMaxGroups = (1LL << 32) - (1 << 20);

// ---- launchers (asynchronous on `stream`; arguments validated by the C ABI)
hipError_t launch_quantize_mxfp4(const void *x, int dtype, int64_t row_stride, void *out, int64_t rows, int64_t cols,
                                 hipStream_t stream);
hipError_t launch_dequantize_mxfp4(const void *q, void *y, int dtype, int64_t row_stride, int64_t rows, int64_t cols,
                                   hipStream_t stream);

// y[t][n] = x[t] . w[n] of two MXFP4 matrices.  `groups`, where offsets is not null: x's rows are sorted by
// expert, offsets[n_experts + 1] their ranges, w the stacked experts; row p of x is x's row
// src_route[p] / top_k where src_route is not null; its output row is route_dst[p], or p.
struct MxGroups {
    const int32_t *offsets = nullptr;
    int n_experts = 0;
    const int32_t *route_dst = nullptr;
    const int32_t *src_route = nullptr;
    int top_k = 1;
    int x_rows = 0;  // rows of x where src_route is given
};
// Experts with rows, of M rows in all, as far as it is known without reading the offsets ...
inline int mx_experts(int M, const MxGroups &g) { return g.offsets == nullptr ? 1 : std::min(g.n_experts, M); }
// ... and the rows of one that has many: the mean and two standard deviations of a random share.
inline int mx_rows(int M, const MxGroups &g) {
    if (g.offsets == nullptr) return M;
    const double mean = (double)M / mx_experts(M, g);
    return std::min(M, (int)std::ceil(mean + 2 * std::sqrt(mean)));
}
// The products on the direct kernel (any shape) ...
hipError_t launch_mxfp4_direct(const void *w, const void *xq, void *y, int dtype, int K, int N, int M,
                               const MxGroups &groups, hipStream_t stream);
// One token whose row is quantized inside the product (K <= kMxFusedMaxK).
constexpr int kMxFusedMaxK = 16384;
hipError_t launch_mxfp4_gemv(const void *w, const void *x, int x_dtype, void *y, int y_dtype, int K, int N,
                             hipStream_t stream);
// mid = MXFP4 of silu(x . w_gate) * (x . w_up), [M][I] (I % 32 == 0), of grouped rows.
hipError_t launch_mxfp4_direct_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I,
                                      int M, const MxGroups &groups, hipStream_t stream);
// ... and on the kernel chosen for the shape.
hipError_t launch_mxfp4_mm(const void *w, const void *xq, void *y, int dtype, int K, int N, int M,
                           const MxGroups &groups, hipStream_t stream, int slices = 1);
// Slices of K (1 or 2) that a grouped product whose reader adds them is best cut into: y holds slices of M rows.
int mxfp4_down_slices(int K, int N, int M, int n_experts);
hipError_t launch_mxfp4_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I, int M,
                               const MxGroups &groups, hipStream_t stream);

// Rows to their experts and back (moe_rows.hip).
hipError_t launch_moe_sort(const int32_t *ids, int n_routes, int n_experts, int32_t *offsets, int32_t *src_route,
                           int32_t *dst_of_route, hipStream_t stream);
hipError_t launch_moe_dispatch_rows(const int32_t *ids, const void *x, int elem_bytes, int T, int top_k, int H, int E,
                                    int32_t *offsets, int32_t *src_route, int32_t *dst_of_route, void *rows,
                                    hipStream_t stream);
// Routing of the MXFP4 FFN: top-k, sort, and x to MXFP4, in one launch (up to kMxRouteOne routes) or two.
hipError_t launch_mxfp4_route(const void *x, int dtype, const float *logits, int T, int H, int E, int top_k,
                              float *route_w, int32_t *ids, int32_t *offsets, int32_t *src_route,
                              int32_t *dst_of_route, void *xq, hipStream_t stream);
// y[t] = sum over k of weights[t, k] * rows[dst(t, k)] (weights nullptr: 1), routes with dst outside
// [0, T * top_k) left out; fp32 rows may be the sum of two slices (T * top_k rows apart).
hipError_t launch_moe_join_rows(const void *rows, int rows_dtype, const int32_t *dst_of_route, const float *weights,
                                void *y, int dtype, int T, int H, int top_k, hipStream_t stream, int slices = 1);
hipError_t launch_moe_combine_rows_backward(const void *grad_y, const void *rows, int dtype,
                                            const int32_t *dst_of_route, const float *weights, void *grad_rows,
                                            float *grad_weights, int T, int H, int top_k, hipStream_t stream);

}  // namespace jjo
