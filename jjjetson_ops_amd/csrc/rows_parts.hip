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
        rows_finish<T>(p.epi, v, row, col, n, p.P, y, p.ldy, p.wide);
    }
}

// Eight values rounded to T and, in the planes behind, what the rounding left of them, rounded again.
template <class T>
__device__ __forceinline__ void store_split(void *to, int planes, int64_t plane, int64_t at, int n, const float *v) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[i];
    for (int k = 0; k < planes; ++k) {
        rows_store8((T *)to + k * plane + at, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] -= (float)rows_round<T>(r[i]);
    }
}

constexpr int kColumnsAtOnce = 512;  // of a workgroup: 64 lanes x 8; its four waves take every fourth row

template <class E>
__global__ __launch_bounds__(256) void rows_act_backward_kernel(const void *grad_y, int64_t grad_y_stride,
                                                                const void *pre, void *gz, int planes,
                                                                int64_t plane, int act, float *part, int T_, int N) {
    typedef typename E::type T;
    __shared__ float sums[4][kColumnsAtOnce];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * kColumnsAtOnce + 8 * lane, n = min(8, N - col);
    const int beg = (int)((int64_t)T_ * blockIdx.y / gridDim.y), end = (int)((int64_t)T_ * (blockIdx.y + 1) / gridDim.y);
    float total[8] = {};
    if (n > 0)
        for (int t = beg + wave; t < end; t += 4) {
            float g[8], z[8];
            rows_load8((const T *)grad_y + t * grad_y_stride + col, n, g);
            if (act != JJO_ACT_NONE) {
                rows_load8((const T *)pre + (int64_t)t * N + col, n, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] *= rows_slope<T>(z[i], act);
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

int64_t output_rows(RowsMode mode, const RowsMm &p) {
    return mode == kRowsWeight ? (int64_t)p.Q * p.halves * std::max(p.n_experts, 1) : p.Q;
}

}  // namespace

int64_t rows_part_bytes(RowsMode mode, const RowsMm &p) {
    return p.slices == 1 ? 0 : 4LL * p.slices * output_rows(mode, p) * p.P * (mode == kRowsSwiglu ? 2 : 1);
}

// An estimate of each tile's time, the cheapest wins.  A launch is rounds of as many workgroups as the 256 CUs hold
// (the device's own number would change the workspace): two of the small tiles a CU, one of the large; a round takes
// `fixed` and one[] or two[] for each stage where a CU has one workgroup or two.  Slices of the sums divide the
// stages and cost a second launch and 8 bytes an output at 4 TB/s.  Measured (us, bf16; estimates in brackets): 2047
// x 14336 over 4096 on tiles of 256 / 160 / 128 rows 198 / 225 / 228 (191 / 232 / 267); 2048 x 4096 over 4096
// 90 / 76 / 64 (96 / 78 / 67); 64 x 4096 over 4096 on tiles of 64 x 64 in 1, 2, 4 slices 22.9 / 17.7 / 13.9
// (25 / 19 / 14).
RowsChoice rows_mm_choose(RowsMode mode, int dtype, int P, int Q, int K, int halves, int n_experts) {
    constexpr int64_t kCus = 256;
    const bool fp32 = dtype == JJO_DTYPE_F32, weight = mode == kRowsWeight;
    const int step = fp32 ? 32 : 64;
    const int64_t cols = mode == kRowsSwiglu ? 2LL * P : P;  // columns of tiles
    // Experts with rows, as far as it is known without reading the offsets, and the rows (sums) of one.
    const int M = weight ? K : Q;
    const double experts = n_experts == 0 ? 1 : std::min(n_experts, M), mean = M / experts;

    // Few rows: a matrix is best read by the direct kernel up to 16 rows, up to 12 where tiles of 64 columns
    // occupy every other CU (11008 x 4096: 1 / 8 / 16 rows 18.1 / 21.2 / 25.0 us against 23.6 / 23.9 / 23.9 on tiles;
    // 4096 x 4096 16 rows 10.6 against 12.9 in four slices).  Of experts only where the tiles leave CUs without two
    // workgroups and rows are long (8 rows of 8 experts, 4096 x 14336: 100 against 122 us; 14336 x 4096: 108
    // against 104; SwiGLU of 64 experts' 1408 x 2048: 19.5 against 16.5).
    const int64_t tiles64 = (cols + 63) / 64;
    const bool few = n_experts == 0 ? Q <= (tiles64 < kCus / 2 ? 16 : 12)
                                    : mean <= 4 && K >= 4096 && (int64_t)experts * tiles64 < 3 * kCus;
    if (few && (mode == kRowsForward || mode == kRowsSwiglu)) {
        const int64_t wgs = (int64_t)experts * ((cols + 15) / 16);
        return {kRowsDirect, wgs >= 4 * kCus ? 2 : 8, 1};  // as above on 2, 4, 8 waves: 100, 111, 110; 1 row 19.0, 18.8, 18.1
    }

    struct Cost {
        int p, q, a_cu;
        float fixed, one, two;
    };
    constexpr Cost k16[] = {{64, 64, 2, 2.2f, 0.35f, 0.5f}, {128, 128, 2, 2.9f, 0.65f, 1.0f},
                            {256, 160, 1, 5.f, 1.13f, 1.13f}, {256, 256, 1, 6.f, 1.4f, 1.4f}};
    // A stage of experts' rows, where few tiles share a matrix's rows and wait for memory.
    constexpr float kExperts[] = {0.5f, 1.3f, 1.4f, 1.9f};
    constexpr Cost k32[] = {{64, 64, 2, 2.2f, 0.62f, 1.05f}, {128, 128, 2, 2.9f, 2.0f, 4.0f}};
    const Cost *const costs = fp32 ? k32 : k16;
    RowsChoice best{kRowsTile128, 0, 1};
    double least = 0;
    for (int tile = 0; tile < (fp32 ? 2 : (int)kRowsTileKinds); ++tile) {
        if (weight && tile == kRowsTile160) continue;
        Cost c = costs[tile];
        if (n_experts > 0 && !weight && !fp32) c.two = kExperts[tile], c.one = std::max(c.one, c.two / c.a_cu);
        // Row tiles in all: of experts the mean over a spread of a third of their rows, as routers have.
        double tiles_q, stages;
        if (weight) {
            tiles_q = experts * halves * ((Q + c.q - 1) / c.q), stages = (mean + step - 1) / step;
            if (n_experts > 0) stages += 0.5;
        } else {
            stages = (double)halves * ((K + step - 1) / step);
            tiles_q = 0;
            const double spread = n_experts == 0 ? 0 : mean / 3 + std::sqrt(mean);
            for (int i = -2; i <= 2; ++i) tiles_q += std::ceil(std::max(1.0, mean + 0.6 * i * spread) / c.q) / 5;
            tiles_q *= experts;
        }
        const double tiles = tiles_q * ((cols + c.p - 1) / c.p);
        for (int slices : {1, 2, 3, 4, 6, 8}) {
            const double per = std::ceil(stages / slices), n = std::ceil(tiles * slices), slots = (double)kCus * c.a_cu;
            if (slices > 1 && (per < 8 || tile > kRowsTile128)) break;
            double us;
            if (n_experts > 0 && n > slots / 2) {  // how full the last round is nobody knows: half of one on average
                us = std::max(n / slots + 0.5, 1.0) * (c.fixed + c.two * per);
            } else {
                const double full = std::floor(n / slots), rest = n - full * slots;
                us = full * (c.fixed + c.two * per);
                if (rest > 0) us += c.fixed + (rest <= kCus ? c.one : c.two) * per;
            }
            if (slices > 1) us += 3 + 8e-6 / 4 * slices * (double)cols * (weight ? (double)Q * halves * experts : Q);
            if (least == 0 || us < least) least = us, best = {tile, 0, slices};
        }
    }
    return best;
}

hipError_t launch_rows_mm(RowsMode mode, int dtype, const RowsMm &p, hipStream_t stream, const RowsChoice *pinned) {
    const RowsChoice c = pinned != nullptr ? *pinned : rows_mm_choose(mode, dtype, p.P, p.Q, p.K, p.halves, p.n_experts);
    if (c.slices != p.slices) return hipErrorInvalidValue;
    const hipError_t e = mx_by_dtype(dtype, [&](auto tag) {
        return rows_mm_run<decltype(tag)>(mode, p, c, stream);
    });
    if (e != hipSuccess || p.slices == 1) return e;
    const int chunks = (p.P + 7) / 8;
    const int64_t rows = output_rows(mode, p);
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

// About two workgroups a CU, two rows a wave at least.
int rows_column_chunks(int T, int N) {
    const int64_t across = ((int64_t)N + kColumnsAtOnce - 1) / kColumnsAtOnce;
    return (int)std::max<int64_t>(1, std::min<int64_t>(512 / across, ((int64_t)T + 7) / 8));
}

hipError_t launch_rows_act_backward(const void *grad_y, int64_t grad_y_stride, const void *pre, void *gz, int planes,
                                    int64_t plane, int dtype, int act, void *sums, bool sums_wide, float *column_part, int T, int N,
                                    hipStream_t stream) {
    const int chunks = rows_column_chunks(T, N);
    const dim3 grid((unsigned)((N + (int64_t)kColumnsAtOnce - 1) / kColumnsAtOnce), (unsigned)chunks);
    float *const part = sums != nullptr ? column_part : nullptr;
    return mx_by_dtype(dtype, [&](auto tag) {
        using E = decltype(tag);
        typedef typename E::type V;
        hipLaunchKernelGGL(rows_act_backward_kernel<E>, grid, dim3(256), 0, stream, grad_y, grad_y_stride, pre, gz, planes,
                           plane, act, part, T, N);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || sums == nullptr) return e;
        const dim3 join((unsigned)((N + 63LL) / 64));
        if (sums_wide)
            hipLaunchKernelGGL(rows_column_join_kernel<float>, join, dim3(256), 0, stream, part, chunks, N, (float *)sums);
        else
            hipLaunchKernelGGL(rows_column_join_kernel<V>, join, dim3(256), 0, stream, part, chunks, N, (V *)sums);
        return hipGetLastError();
    });
}

hipError_t launch_rows_swiglu_backward(const void *grad_mid, const void *gate_up, void *grad_gate_up, int planes, int64_t plane, int dtype,
                                       const int32_t *offsets, int n_experts, int I, int R, hipStream_t stream) {
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
