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

constexpr int kFusedMaxK = kMxFusedMaxK;

struct MxProblem {
    const uint8_t *w, *w2, *x;  // w2: the up matrix (SwiGLU)
    void *y;                    // outputs, or the MXFP4 rows of the SwiGLU form
    int dtype;
    int K, N, M;
    int token_tiles;  // of the launch; workgroup i has token tile i % token_tiles
    MxGroups g;
};

// Operands of U steps of TILES tiles of 16 rows.  A row's scale bytes of the U steps are one load:
// dword u holds the bytes of step u's four lane groups.  Rows shorter than that (and only
// they) fetch each byte where it is used.
template <int TILES, int U>
struct MxChunk {
    u32x4v v[U][TILES];
    uint32_t s[TILES][U];
};
template <int TILES, int U>
__device__ __forceinline__ void load_chunk(MxChunk<TILES, U> &c, const uint8_t *const (&rows)[TILES],
                                           const uint8_t *const (&scales)[TILES], int step, int nb) {
    const int q = (threadIdx.x & 63) >> 4;
    if (nb >= 4 * U) {
        const int at = min(4 * step, nb - 4 * U);  // the last chunk's bytes end with the row
#pragma unroll
        for (int t = 0; t < TILES; ++t) __builtin_memcpy(c.s[t], scales[t] + at, 4 * U);  // whatever the alignment
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int blk = min(4 * (step + u) + q, nb - 1);
#pragma unroll
        for (int t = 0; t < TILES; ++t) c.v[u][t] = *reinterpret_cast<const u32x4v *>(rows[t] + (size_t)blk * 16);
    }
}
// The chunk's scale bytes to their places: shifted where the row ends inside the chunk (zeros
// behind it), or fetched.
template <int TILES, int U>
__device__ __forceinline__ void place_scales(MxChunk<TILES, U> &c, const uint8_t *const (&scales)[TILES], int step,
                                             int nb) {
    const int over = 4 * step + 4 * U - nb;  // uniform
    if (over <= 0) return;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        if (nb >= 4 * U) {
            unsigned __int128 b = 0;
            __builtin_memcpy(&b, c.s[t], 4 * U);
            b >>= 8 * over;
            __builtin_memcpy(c.s[t], &b, 4 * U);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                c.s[t][u] = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    c.s[t][u] |= (uint32_t)scales[t][min(4 * (step + u) + k, nb - 1)] << (8 * k);
            }
        }
    }
}

// One wave's 1024 values of the fused activation, 16 a lane, to codes and scales in LDS.
template <class T>
__device__ __forceinline__ void load16(const T *p, float *x) {
    constexpr int kVec = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kVec; ++i) {
        const MxVec<T, kVec> a = reinterpret_cast<const MxVec<T, kVec> *>(p)[i];
#pragma unroll
        for (int k = 0; k < kVec; ++k) x[kVec * i + k] = (float)a.v[k];
    }
}

// RT tiles of 16 weight rows x TT tiles of 16 tokens, W waves over K, U steps of 128 in registers
// and U more in flight.  SWIGLU: RT = 4, two tiles of gate rows and the two of the same up
// rows.  XT: void (x is MXFP4), or the type of the one token's row, which every wave quantizes
// for its own slice of K.
template <int RT, int TT, int W, int U, bool GROUPED, bool SWIGLU, class XT>
__global__ __launch_bounds__(64 * W) void mxfp4_direct_kernel(MxProblem p) {
    constexpr bool kFused = !std::is_void_v<XT>;
    constexpr int kPieces = 2;  // of 1024 values in a wave's slice of the fused form
    __shared__ f32x4v part[W][RT * TT][64];
    __shared__ u32x4v x_codes[kFused ? W : 1][kFused ? 32 * kPieces : 1];
    __shared__ uint8_t x_scales[kFused ? W : 1][kFused ? 32 * kPieces : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, q = lane >> 4;
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
    if constexpr (!kFused) {
        const size_t x_rows = p.g.src_route != nullptr ? p.g.x_rows : p.M;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            int t = min(first + 16 * tt + r16, end - 1);
            if (GROUPED && p.g.src_route != nullptr) t = min(max(p.g.src_route[t] / p.g.top_k, 0), p.g.x_rows - 1);
            xr[tt] = p.x + (size_t)t * half;
            xs[tt] = p.x + x_rows * half + (size_t)t * nb;
        }
    }
    f32x4v acc[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = f32x4v{0.f, 0.f, 0.f, 0.f};

    MxChunk<RT, U> w;
    MxChunk<TT, U> x;
    if constexpr (kFused) {
        // The token's values are asked for before the weights: loads return in order.
        typedef std::conditional_t<kFused, XT, float> T;
        const T *src = (const T *)p.x + 128 * (size_t)s_beg;
        const int live = min(128 * (s_end - s_beg), p.K - 128 * s_beg);  // a multiple of 32
        float v[kPieces][16];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (1024 * i + 16 * lane < live) load16(src + 1024 * i + 16 * lane, v[i]);
        if (s_beg < s_end) load_chunk(w, wr, ws, s_beg, nb);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (1024 * i >= 128 * (s_end - s_beg)) break;
            const bool in = 1024 * i + 16 * lane < live;
            uint32_t m = 0;
            if (in) {
                m = mx_amax8(v[i]);
                const uint32_t o = mx_amax8(v[i] + 8);
                m = o > m ? o : m;
            }
            const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true);  // lane ^ 1
            m = o > m ? o : m;
            const uint32_t s = mx_scale_byte(m);
            uint2 c = make_uint2(0u, 0u);
            if (in) c = make_uint2(mx_codes8(v[i], s), mx_codes8(v[i] + 8, s));
            reinterpret_cast<uint2 *>(&x_codes[wave][32 * i])[lane] = c;
            if ((lane & 1) == 0) x_scales[wave][32 * i + (lane >> 1)] = (uint8_t)s;
        }
    } else if (s_beg < s_end) {
        load_chunk(w, wr, ws, s_beg, nb);
        load_chunk(x, xr, xs, s_beg, nb);
    }
    for (int s = s_beg; s < s_end; s += U) {
        MxChunk<RT, U> w_next;
        MxChunk<TT, U> x_next;
        if (s + U < s_end) {
            load_chunk(w_next, wr, ws, s + U, nb);
            if constexpr (!kFused) load_chunk(x_next, xr, xs, s + U, nb);
        }
        place_scales(w, ws, s, nb);
        if constexpr (!kFused) place_scales(x, xs, s, nb);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= s_end) break;
            if (4 * (s + u) + 4 > nb) {  // the row ends inside the step (K % 128)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (4 * (s + u) + q >= nb) w.v[u][rt] = u32x4v{0u, 0u, 0u, 0u};
            }
            u32x4v xv[TT];
            uint32_t sx[TT];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                if constexpr (kFused) {
                    xv[tt] = x_codes[wave][4 * (s + u - s_beg) + q];
                    sx[tt] = x_scales[wave][4 * (s + u - s_beg) + q];
                } else {
                    xv[tt] = x.v[u][tt];
                    sx[tt] = x.s[tt][u] >> (8 * q);
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
                    acc[rt][tt] = mx_mfma(w.v[u][rt], xv[tt], acc[rt][tt], w.s[rt][u] >> (8 * q), sx[tt]);
        }
        w = w_next;
        if constexpr (!kFused) x = x_next;
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

template <int RT, int TT, int W, int U, bool SWIGLU, class XT = void>
hipError_t run_direct(MxProblem p, hipStream_t stream) {
    const int rows = SWIGLU ? 32 : 16 * RT;
    // token tiles of M rows, and one more for each expert that can have a rest
    p.token_tiles = (p.M + 16 * TT - 1) / (16 * TT) + (p.g.offsets != nullptr ? std::min(p.g.n_experts, p.M) : 0);
    const int64_t wgs = (int64_t)p.token_tiles * ((p.N + rows - 1) / rows);
    if (wgs * 64 * W >= 1LL << 32) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)wgs), block(64 * W);
    if constexpr (!std::is_void_v<XT>)
        hipLaunchKernelGGL((mxfp4_direct_kernel<RT, TT, W, U, false, false, XT>), grid, block, 0, stream, p);
    else if (p.g.offsets != nullptr)
        hipLaunchKernelGGL((mxfp4_direct_kernel<RT, TT, W, U, true, SWIGLU, void>), grid, block, 0, stream, p);
    else if constexpr (!SWIGLU)
        hipLaunchKernelGGL((mxfp4_direct_kernel<RT, TT, W, U, false, false, void>), grid, block, 0, stream, p);
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
    const int mean = mean_rows(M, groups), steps = (K + 127) / 128;
    if (mean <= 16) return steps >= 64 ? run_direct<1, 1, 8, 4, false>(p, stream) : run_direct<1, 1, 4, 4, false>(p, stream);
    if (mean <= 32) return steps >= 64 ? run_direct<1, 2, 8, 4, false>(p, stream) : run_direct<1, 2, 4, 4, false>(p, stream);
    return run_direct<2, 4, 4, 2, false>(p, stream);
}

hipError_t launch_mxfp4_direct_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I,
                                      int M, const MxGroups &groups, hipStream_t stream) {
    const MxProblem p{(const uint8_t *)w_gate, (const uint8_t *)w_up, (const uint8_t *)xq, mid, JJO_DTYPE_F32, K, I, M,
                      0, groups};
    if (mean_rows(M, groups) <= 16) return run_direct<4, 1, 4, 2, true>(p, stream);
    return run_direct<4, 2, 4, 2, true>(p, stream);
}

hipError_t launch_mxfp4_gemv(const void *w, const void *x, int x_dtype, void *y, int y_dtype, int K, int N,
                             hipStream_t stream) {
    const MxProblem p{(const uint8_t *)w, nullptr, (const uint8_t *)x, y, y_dtype, K, N, 1, 0, MxGroups{}};
    return mx_by_dtype(x_dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        return K > 8192 ? run_direct<1, 1, 8, 4, false, T>(p, stream) : run_direct<1, 1, 4, 4, false, T>(p, stream);
    });
}

}  // namespace jjo
