// Around the float products: the sums of a product's slices with its epilogue, the gradient through an
// activation with the bias's gradient, and the gradient through SwiGLU.  All are bound by HBM: every
// value is read and written once, eight columns a thread.
#include <hip/hip_runtime.h>

#include "rows_mm.hpp"

namespace jjo {
namespace {

__device__ __forceinline__ int rows_limit(const int32_t *offsets, int n_experts, int rows) {
    return offsets != nullptr ? min(max(offsets[n_experts], 0), rows) : rows;
}

// Sums over slices in their order, then the epilogue.  A thread takes eight columns of a row.
template <class E, RowsMode MODE>
__global__ __launch_bounds__(256) void rows_join_kernel(RowsMm p, int chunks, int64_t rows) {
    typedef typename E::type T;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t row = id / chunks;
    if (row >= rows) return;
    const int col = (int)(id % chunks) * 8, n = min(8, p.P - col);
    if (MODE != kRowsWeight && row >= rows_limit(p.offsets, p.n_experts, p.M)) return;
    const int64_t cols = MODE == kRowsSwiglu ? 2 * (int64_t)p.P : p.P;
    const float *from = p.part + row * cols + col;
    float v[8] = {}, up[8] = {};
    for (int s = 0; s < p.slices; ++s, from += rows * cols) {
        float a[8];
        rows_load8(from, n, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += a[i];
        if constexpr (MODE == kRowsSwiglu) {
            rows_load8(from + p.P, n, a);
#pragma unroll
            for (int i = 0; i < 8; ++i) up[i] += a[i];
        }
    }
    if constexpr (MODE == kRowsSwiglu) {
        rows_finish_swiglu<T>(p.epi, v, up, row, col, n, p.P, p.y);
    } else {
        void *y = p.y;
        if (MODE == kRowsWeight && p.halves == 2 && row >= rows / 2) y = p.y2, row -= rows / 2;
        rows_finish<T>(p.epi, v, row, col, n, p.P, y, p.ldy, MODE == kRowsWeight && p.wide);
    }
}

// Eight values rounded to T and, in the planes behind, what the rounding left of them, rounded again (fp16: times
// kRowsRestScale; nothing of an infinity or a NaN, also where the rounding made it).
template <class T>
__device__ __forceinline__ void store_split(void *to, int planes, int64_t plane, int64_t at, int n, const float *v) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[i];
    for (int k = 0; k < planes; ++k) {
        rows_store8((T *)to + k * plane + at, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float kept = (float)rows_round<T>(r[i]);
            r[i] = fabsf(kept) <= 3.402823466e38f ? r[i] - kept : 0.0f;
            if (std::is_same_v<T, _Float16>) r[i] *= kRowsRestScale;
        }
    }
}

constexpr int kColumnsAtOnce = kRowsColumns;  // of a workgroup: 64 lanes x 8; its four waves take every fourth row

template <class E>
__global__ __launch_bounds__(256) void rows_act_backward_kernel(const void *grad_y, int64_t grad_y_stride,
                                                                const void *pre, void *gz, int planes,
                                                                int64_t plane, int act, float *part, int T_, int N) {
    typedef typename E::type T;
    __shared__ float sums[4][kColumnsAtOnce];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * kColumnsAtOnce + 8 * lane, n = min(8, N - col);
    const int beg = (int)((int64_t)T_ * blockIdx.y / gridDim.y);
    const int end = (int)((int64_t)T_ * (blockIdx.y + 1) / gridDim.y);
    float total[8] = {};
    if (n > 0)
        for (int t = beg + wave; t < end; t += 4) {
            float g[8], z[8];
            rows_load8((const T *)grad_y + t * grad_y_stride + col, n, g);
            if (act != JJO_ACT_NONE) {
                rows_load8((const T *)pre + (int64_t)t * N + col, n, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = rows_through<T>(g[i], z[i], act);
                store_split<T>(gz, planes, plane, (int64_t)t * N + col, n, g);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) total[i] += g[i];
        }
    if (part == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[wave][8 * lane + i] = total[i];
    __syncthreads();
    for (int c = threadIdx.x; c < kColumnsAtOnce; c += 256) {
        const int at = blockIdx.x * kColumnsAtOnce + c;
        if (at < N) part[(int64_t)blockIdx.y * N + at] = sums[0][c] + sums[1][c] + sums[2][c] + sums[3][c];
    }
}

// Column sums of the chunks: 64 columns a workgroup, its four waves every fourth chunk, eight loads in flight.
template <class T>
__global__ __launch_bounds__(256) void rows_column_join_kernel(const float *part, int chunks, int N, T *out) {
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float v = 0.0f;
    if (c < N) {
#pragma unroll 8
        for (int s = wave; s < chunks; s += 4) v += part[(int64_t)s * N + c];
    }
    sums[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < N) out[c] = rows_round<T>(sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]);
}

template <class E>
__global__ __launch_bounds__(256) void rows_swiglu_backward_kernel(const void *grad_mid, const void *gate_up,
                                                                   void *grad_gate_up, int planes, int64_t plane,
                                                                   const int32_t *offsets, int n_experts, int chunks,
                                                                   int I, int R) {
    typedef typename E::type T;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / chunks;
    if (row >= rows_limit(offsets, n_experts, R)) return;
    const int col = (int)(id % chunks) * 8, n = min(8, I - col);
    const int64_t at = row * 2 * I + col;
    float g[8], gate[8], up[8];
    rows_load8((const T *)grad_mid + row * I + col, n, g);
    rows_load8((const T *)gate_up + at, n, gate);
    rows_load8((const T *)gate_up + at + I, n, up);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = rows_sigmoid(gate[i]), gm = g[i];
        g[i] = gm * up[i] * s * (1.0f + gate[i] * (1.0f - s));
        up[i] = gm * gate[i] * s;
    }
    store_split<T>(grad_gate_up, planes, plane, at, n, g);
    store_split<T>(grad_gate_up, planes, plane, at + I, n, up);
}

bool grid_of(int64_t threads, dim3 *grid) {
    if (threads >= (1LL << 32) - 256) return false;
    *grid = dim3((unsigned)((threads + 255) / 256));
    return true;
}

}  // namespace

hipError_t launch_rows_mm(RowsMode mode, int dtype, const RowsMm &p, hipStream_t stream, const RowsChoice *pinned) {
    const RowsChoice c =
        pinned != nullptr ? *pinned : rows_mm_choose(mode, dtype, p.P, p.Q, p.K, p.halves, p.n_experts);
    if (c.slices != p.slices) return hipErrorInvalidValue;
    const hipError_t e = mx_by_dtype(dtype, [&](auto tag) {
        return rows_mm_run<decltype(tag)>(mode, p, c, stream);
    });
    if (e != hipSuccess || p.slices == 1) return e;
    const int chunks = (p.P + 7) / 8;
    const int64_t rows = rows_output_rows(mode, p);
    dim3 grid;
    if (!grid_of(rows * chunks, &grid)) return hipErrorInvalidConfiguration;
    return mx_by_dtype(dtype, [&](auto tag) {
        using E = decltype(tag);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p, chunks, rows);
            return hipGetLastError();
        };
        switch (mode) {
            case kRowsSwiglu: return go(rows_join_kernel<E, kRowsSwiglu>);
            case kRowsWeight: return go(rows_join_kernel<E, kRowsWeight>);
            default: return go(rows_join_kernel<E, kRowsForward>);
        }
    });
}

hipError_t launch_rows_act_backward(const void *grad_y, int64_t grad_y_stride, const void *pre, void *gz, int planes,
                                    int64_t plane, int dtype, int act, void *sums, bool sums_wide,
                                     float *column_part, int T, int N, hipStream_t stream) {
    const int chunks = rows_column_chunks(T, N);
    const dim3 grid((unsigned)((N + (int64_t)kColumnsAtOnce - 1) / kColumnsAtOnce), (unsigned)chunks);
    float *const part = sums != nullptr ? column_part : nullptr;
    return mx_by_dtype(dtype, [&](auto tag) {
        using E = decltype(tag);
        typedef typename E::type V;
        hipLaunchKernelGGL(rows_act_backward_kernel<E>, grid, dim3(256), 0, stream, grad_y, grad_y_stride, pre, gz,
                           planes, plane, act, part, T, N);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || sums == nullptr) return e;
        const dim3 join((unsigned)((N + 63LL) / 64));
        if (sums_wide)
            hipLaunchKernelGGL(rows_column_join_kernel<float>, join, dim3(256), 0, stream, part, chunks, N,
                               (float *)sums);
        else
            hipLaunchKernelGGL(rows_column_join_kernel<V>, join, dim3(256), 0, stream, part, chunks, N, (V *)sums);
        return hipGetLastError();
    });
}

hipError_t launch_rows_swiglu_backward(const void *grad_mid, const void *gate_up, void *grad_gate_up, int planes,
                                       int64_t plane, int dtype, const int32_t *offsets, int n_experts, int I, int R,
                                       hipStream_t stream) {
    const int chunks = (I + 7) / 8;
    dim3 grid;
    if (!grid_of((int64_t)R * chunks, &grid)) return hipErrorInvalidConfiguration;
    return mx_by_dtype(dtype, [&](auto tag) {
        hipLaunchKernelGGL(rows_swiglu_backward_kernel<decltype(tag)>, grid, dim3(256), 0, stream, grad_mid, gate_up,
                           grad_gate_up, planes, plane, offsets, n_experts, chunks, I, R);
        return hipGetLastError();
    });
}

}  // namespace jjo
