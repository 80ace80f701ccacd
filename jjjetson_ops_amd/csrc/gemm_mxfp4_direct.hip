// MXFP4 weights x MXFP4 activations for few tokens (a decode batch, an expert's handful of
// rows) on gfx950's scaled matrix instruction, operands straight from memory to registers.
//
//     y[t][n] = sum over blocks b of 2^(sw[n,b] + sx[t,b] - 254) * sum_j cw[n,b,j] * cx[t,b,j]
//
// One v_mfma_scale_f32_16x16x128 takes 16 rows x 16 tokens x four blocks: a lane's operand is
// one block, 16 bytes as they lie in the matrix, and its scale operand that block's byte, so
// nothing is unpacked.  Sums are fp32.  Bound by reading the weights (17/32 byte a value): a
// workgroup's waves cut K between them, so that a small output still fills the chip with
// loads in flight; the slices are added through LDS in slice order.
#include <hip/hip_runtime.h>

#include "mxfp4_mm.hpp"

namespace jjo {
namespace {

struct MxProblem {
    const uint8_t *w, *w2, *x;  // w2: the up matrix (SwiGLU)
    void *y;                    // outputs, or the MXFP4 rows of the SwiGLU form
    int dtype;
    int K, N, M;
    int token_tiles;  // of the launch; workgroup i has token tile i % token_tiles
    MxGroups g;
};

// RT tiles of 16 weight rows x TT tiles of 16 tokens, W waves over K, U steps of 128 loaded ahead.
// SWIGLU: RT = 4, two tiles of gate rows and the two of the same up rows.
template <int RT, int TT, int W, int U, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(64 * W) void mxfp4_direct_kernel(MxProblem p) {
    __shared__ f32x4v part[W][RT * TT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const int tile_t = (int)(blockIdx.x % (unsigned)p.token_tiles), tile_n = (int)(blockIdx.x / (unsigned)p.token_tiles);
    int expert = 0, first = tile_t * 16 * TT, end = p.M;
    if constexpr (GROUPED) {
        if (!mx_expert_tile(p.g.offsets, p.g.n_experts, p.M, 16 * TT, tile_t, expert, first, end)) return;
    }
    constexpr int kRows = SWIGLU ? 32 : 16 * RT;  // weight rows of one matrix
    const int n0 = tile_n * kRows;
    const int nb = p.K / kQK, steps = (nb + 3) / 4;
    const int s_beg = (int)((int64_t)steps * wave / W), s_end = (int)((int64_t)steps * (wave + 1) / W);
    const size_t half = (size_t)p.K / 2;

    const uint8_t *wr[RT], *ws[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const uint8_t *m = SWIGLU && rt >= 2 ? p.w2 : p.w;
        const int tile = SWIGLU ? rt & 1 : rt;
        const size_t row = (size_t)expert * p.N + min(n0 + 16 * tile + r16, p.N - 1);
        const size_t all = (size_t)(GROUPED ? p.g.n_experts : 1) * p.N;
        wr[rt] = m + row * half;
        ws[rt] = m + all * half + row * nb;
    }
    const uint8_t *xr[TT], *xs[TT];
    const size_t x_rows = p.g.src_route != nullptr ? p.g.x_rows : p.M;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        int t = min(first + 16 * tt + r16, end - 1);
        if (GROUPED && p.g.src_route != nullptr) t = min(max(p.g.src_route[t] / p.g.top_k, 0), p.g.x_rows - 1);
        xr[tt] = p.x + (size_t)t * half;
        xs[tt] = p.x + x_rows * half + (size_t)t * nb;
    }
    f32x4v acc[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = f32x4v{0.f, 0.f, 0.f, 0.f};

    for (int s = s_beg; s < s_end; s += U) {
        u32x4v a[U][RT], b[U][TT];
        uint32_t sa[U][RT], sb[U][TT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int blk = 4 * min(s + u, s_end - 1) + q, at = min(blk, nb - 1);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                a[u][rt] = *reinterpret_cast<const u32x4v *>(wr[rt] + (size_t)at * 16);
                sa[u][rt] = ws[rt][at];
                if (blk >= nb) a[u][rt] = u32x4v{0u, 0u, 0u, 0u};  // behind the row's end (K % 128)
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                b[u][tt] = *reinterpret_cast<const u32x4v *>(xr[tt] + (size_t)at * 16);
                sb[u][tt] = xs[tt][at];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < s_end) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt)
                        acc[rt][tt] = mx_mfma(a[u][rt], b[u][tt], acc[rt][tt], sa[u][rt], sb[u][tt]);
            }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) part[wave][rt * TT + tt][lane] = acc[rt][tt];
    __syncthreads();
    auto total = [&](int tile) {
        f32x4v v = part[0][tile][lane];
#pragma unroll
        for (int k = 1; k < W; ++k) v += part[k][tile][lane];
        return v;
    };
    if constexpr (SWIGLU) {
        uint8_t *codes = (uint8_t *)p.y, *scales = codes + (size_t)p.M * (p.N / 2);
        for (int tt = wave; tt < TT; tt += W) {
            const f32x4v gate[2] = {total(tt), total(TT + tt)}, up[2] = {total(2 * TT + tt), total(3 * TT + tt)};
            const int t = first + 16 * tt + r16;
            const size_t row = min(t, p.M - 1);
            mx_swiglu_store(gate, up, codes + row * (p.N / 2) + n0 / 2, scales + row * (p.N / kQK) + n0 / kQK, t < end);
        }
    } else {
        const bool vec = p.N % 4 == 0;  // y is 16-byte aligned
        for (int tile = wave; tile < RT * TT; tile += W) {
            const f32x4v v = total(tile);
            const int t = first + 16 * (tile % TT) + r16, n = n0 + 16 * (tile / TT) + 4 * q;
            if (t >= end || n >= p.N) continue;
            const int row = GROUPED && p.g.route_dst != nullptr ? p.g.route_dst[t] : t;
            mx_store4(p.y, p.dtype, (size_t)row * p.N + n, v, p.N - n, vec);
        }
    }
}

template <int RT, int TT, int W, int U, bool SWIGLU>
hipError_t run_direct(MxProblem p, hipStream_t stream) {
    const int rows = SWIGLU ? 32 : 16 * RT;
    // token tiles of M rows, and one more for each expert that can have a rest
    p.token_tiles = (p.M + 16 * TT - 1) / (16 * TT) + (p.g.offsets != nullptr ? std::min(p.g.n_experts, p.M) : 0);
    const int64_t wgs = (int64_t)p.token_tiles * ((p.N + rows - 1) / rows);
    if (wgs * 64 * W >= 1LL << 32) return hipErrorInvalidConfiguration;
    if (p.g.offsets != nullptr)
        hipLaunchKernelGGL((mxfp4_direct_kernel<RT, TT, W, U, true, SWIGLU>), dim3((unsigned)wgs), dim3(64 * W), 0,
                           stream, p);
    else if constexpr (!SWIGLU)
        hipLaunchKernelGGL((mxfp4_direct_kernel<RT, TT, W, U, false, false>), dim3((unsigned)wgs), dim3(64 * W), 0,
                           stream, p);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

// Rows per expert expected (of M rows in all), or M.
int mean_rows(int M, const MxGroups &g) {
    if (g.offsets == nullptr) return M;
    const int active = std::min(g.n_experts, M);
    return (M + active - 1) / active;
}

}  // namespace

hipError_t launch_mxfp4_direct(const void *w, const void *xq, void *y, int dtype, int K, int N, int M,
                               const MxGroups &groups, hipStream_t stream) {
    const MxProblem p{(const uint8_t *)w, nullptr, (const uint8_t *)xq, y, dtype, K, N, M, 0, groups};
    const int mean = mean_rows(M, groups);
    if (mean <= 16) return run_direct<1, 1, 4, 8, false>(p, stream);
    if (mean <= 32) return run_direct<2, 2, 4, 4, false>(p, stream);
    return run_direct<4, 4, 4, 2, false>(p, stream);
}

hipError_t launch_mxfp4_direct_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I,
                                      int M, const MxGroups &groups, hipStream_t stream) {
    const MxProblem p{(const uint8_t *)w_gate, (const uint8_t *)w_up, (const uint8_t *)xq, mid, JJO_DTYPE_F32, K, I, M,
                      0, groups};
    if (mean_rows(M, groups) <= 16) return run_direct<4, 1, 4, 4, true>(p, stream);
    return run_direct<4, 4, 4, 2, true>(p, stream);
}

}  // namespace jjo
