// MXFP4 weights x MXFP4 activations for prompts and for experts with many rows: tiles staged in
// LDS, gfx950's scaled matrix instruction.
//
//     y[t][n] = sum over blocks b of 2^(sw[n,b] + sx[t,b] - 254) * sum_j cw[n,b,j] * cx[t,b,j]
//
// A stage is 256 values (128 bytes) of every weight row and token row of the tile, two steps of the
// matrix instruction.  The codes go to LDS by DMA, 8 rows an instruction, the 16-byte pieces of a
// row permuted by its row number (piece ^ row % 8) so that the 8 lanes that LDS serves at a time
// fall in different banks; of the stage's 8 blocks lane group q of a step u takes block 2q + u,
// so that a lane's two scale bytes are one 16-bit read and the instruction picks the byte.  The
// scales (8 bytes a row and stage, of any alignment) go through a register of one thread per row.
// While a stage is computed the next one lands in the other buffer; one barrier per stage.
#include <hip/hip_runtime.h>

#include "mxfp4_mm.hpp"

namespace jjo {
namespace {

struct MxTiled {
    const uint8_t *w, *w2, *x;  // w2: the up matrix (SwiGLU)
    void *y;                    // outputs, or the MXFP4 rows of the SwiGLU form
    int dtype;
    int K, N, M;
    int tiles_n, tiles_t;  // of the launch
    MxGroups g;
};

// acc += W . X^T of step U of a stage: byte U of the scale registers.
template <int U>
__device__ __forceinline__ f32x4v mx_mfma_step(u32x4v w, u32x4v x, f32x4v acc, uint32_t sw, uint32_t sx) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, U, (int)sw, U, (int)sx);
}

// WN x WT waves of RT tiles of 16 weight rows x TT tiles of 16 tokens each.
template <int RT_, int TT_, int WN_, int WT_>
struct MxTile {
    static constexpr int RT = RT_, TT = TT_, WN = WN_, WT = WT_;
    static constexpr int kWaves = WN * WT, kThreads = 64 * kWaves;
    static constexpr int kRowsN = 16 * RT * WN, kRowsT = 16 * TT * WT, kRows = kRowsN + kRowsT;
    static constexpr int kDma = kRows / 8 / kWaves;  // instructions a wave and stage
    static constexpr int kScaleRows = (kRows + kThreads - 1) / kThreads;  // rows a thread
    static constexpr int kStage = kRows * 128;
    static constexpr int kLds = 2 * (kStage + kRows * 8);
    static_assert(kRows % (8 * kWaves) == 0 && kRowsN % 8 == 0, "whole DMA instructions");
};

template <class Tile, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(Tile::kThreads) void mxfp4_tiled_kernel(MxTiled p) {
    constexpr int RT = Tile::RT, TT = Tile::TT;
    extern __shared__ __align__(16) uint8_t lds[];
    uint8_t *const lds_scales = lds + 2 * Tile::kStage;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, q = lane >> 4;
    const int wn = wave % Tile::WN, wt = wave / Tile::WN;

    // Workgroups go to the eight XCDs in turn: each takes a contiguous run of tiles, token tiles
    // fastest, so that a weight row tile is read into one L2.
    const int total = p.tiles_n * p.tiles_t, per = total / 8, rest = total % 8;
    const int xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    const int tile = xcd * per + min(xcd, rest) + at;
    const int tile_t = tile % p.tiles_t, tile_n = tile / p.tiles_t;
    int expert = 0, first = tile_t * Tile::kRowsT, end = p.M;
    if constexpr (GROUPED) {
        if (!mx_expert_tile(p.g.offsets, p.g.n_experts, p.M, Tile::kRowsT, tile_t, expert, first, end)) return;
    }
    const int nb = p.K / kQK, stages = (nb + 7) / 8;
    const uint32_t half = (uint32_t)p.K / 2;
    constexpr int kOutN = SWIGLU ? Tile::kRowsN / 2 : Tile::kRowsN;  // rows of one matrix
    const int n0 = tile_n * kOutN;

    // Row `row` of the tile (weights first): its matrix's row, clamped to the last valid one.
    auto weight_row = [&](int row) {
        if constexpr (SWIGLU) return min(n0 + 32 * (row / 64) + row % 32, p.N - 1);
        return min(n0 + row, p.N - 1);
    };
    auto token_row = [&](int row) {
        int t = min(first + row, end - 1);
        if (GROUPED && p.g.src_route != nullptr) t = min(max(p.g.src_route[t] / p.g.top_k, 0), p.g.x_rows - 1);
        return t;
    };
    auto is_up = [&](int row) { return SWIGLU && (row & 32) != 0; };
    const size_t w_first = (size_t)expert * p.N, w_all = (size_t)(GROUPED ? p.g.n_experts : 1) * p.N;
    const size_t x_all = p.g.src_route != nullptr ? p.g.x_rows : p.M;

    // ---- this lane's part of the DMA: rows 8 * i + lane / 8, piece (lane % 8) ^ (lane / 8)
    const uint8_t *base[Tile::kDma];  // uniform
    uint32_t off[Tile::kDma];
    const uint32_t piece = 16 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (int i = 0; i < Tile::kDma; ++i) {
        const int row8 = 8 * (wave * Tile::kDma + i), row = row8 + (lane >> 3);
        if (row8 < Tile::kRowsN) {
            base[i] = (is_up(row8) ? p.w2 : p.w) + w_first * half;
            base[i] += (size_t)n0 * half;
            off[i] = (uint32_t)(weight_row(row) - n0) * half + piece;
        } else {
            const int t0 = GROUPED && p.g.src_route != nullptr ? 0 : first;
            base[i] = p.x + (size_t)t0 * half;
            off[i] = (uint32_t)(token_row(row - Tile::kRowsN) - t0) * half + piece;
        }
    }
    // ---- and of the scales: one row, or kScaleRows
    const uint8_t *srow[Tile::kScaleRows];
#pragma unroll
    for (int i = 0; i < Tile::kScaleRows; ++i) {
        const int row = min((int)threadIdx.x + i * Tile::kThreads, Tile::kRows - 1);
        if (row < Tile::kRowsN)
            srow[i] = (is_up(row) ? p.w2 : p.w) + w_all * half + (w_first + weight_row(row)) * nb;
        else
            srow[i] = p.x + x_all * half + (size_t)token_row(row - Tile::kRowsN) * nb;
    }
    uint64_t sv[Tile::kScaleRows];
    auto load_scales = [&](int st) {  // the last stage's bytes end with the row (nb >= 8)
#pragma unroll
        for (int i = 0; i < Tile::kScaleRows; ++i) __builtin_memcpy(&sv[i], srow[i] + min(8 * st, nb - 8), 8);
    };
    auto store_scales = [&](int st) {
        const int over = max(8 * st + 8 - nb, 0);  // zeros behind the row's end
#pragma unroll
        for (int i = 0; i < Tile::kScaleRows; ++i) {
            const int row = threadIdx.x + i * Tile::kThreads;
            if (row < Tile::kRows)
                *reinterpret_cast<uint64_t *>(lds_scales + (st & 1) * (Tile::kRows * 8) + row * 8) = sv[i] >> (8 * over);
        }
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    auto dma = [&](int st) {
        const uint32_t left = 16u * (uint32_t)(nb - 8 * st);  // bytes of the row from the stage on
        const uint32_t back = piece + 16 > left ? piece + 16 - left : 0;
#pragma unroll
        for (int i = 0; i < Tile::kDma; ++i) {
            const uint32_t m0v = __builtin_amdgcn_readfirstlane(lds0 + (st & 1) * Tile::kStage +
                                                                1024 * (wave * Tile::kDma + i));
            asm volatile("global_load_lds_dwordx4 %0, %1"
                         :
                         : "v"(off[i] - back), "s"(base[i] + (size_t)st * 128), "{m0}"(m0v)
                         : "memory");
        }
    };

    f32x4v acc[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = f32x4v{0.f, 0.f, 0.f, 0.f};

    load_scales(0);
    dma(0);
    const uint32_t w_at = (uint32_t)(16 * RT * wn + r16), x_at = (uint32_t)(Tile::kRowsN + 16 * TT * wt + r16);
    const uint32_t sw0 = 16u * ((2 * q) ^ (r16 & 7)), sw1 = 16u * ((2 * q + 1) ^ (r16 & 7));
    for (int st = 0; st < stages; ++st) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // stage st has landed
        store_scales(st);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (st + 1 < stages) {
            load_scales(st + 1);
            dma(st + 1);
        }
        const uint8_t *buf = lds + (st & 1) * Tile::kStage;
        const uint8_t *sbuf = lds_scales + (st & 1) * (Tile::kRows * 8);
        uint32_t sw[RT], sx[TT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sw[rt] = *reinterpret_cast<const uint16_t *>(sbuf + (w_at + 16 * rt) * 8 + 2 * q);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) sx[tt] = *reinterpret_cast<const uint16_t *>(sbuf + (x_at + 16 * tt) * 8 + 2 * q);
        auto step = [&](auto u_tag) {
            constexpr int U = decltype(u_tag)::value;
            const uint32_t sw_off = U == 0 ? sw0 : sw1;
            u32x4v a[RT], b[TT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                a[rt] = *reinterpret_cast<const u32x4v *>(buf + (w_at + 16 * rt) * 128 + sw_off);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
                b[tt] = *reinterpret_cast<const u32x4v *>(buf + (x_at + 16 * tt) * 128 + sw_off);
            if (8 * st + 8 > nb) {  // the row ends inside the stage
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (8 * st + 2 * q + U >= nb) a[rt] = u32x4v{0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    acc[rt][tt] = mx_mfma_step<U>(a[rt], b[tt], acc[rt][tt], sw[rt], sx[tt]);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
    }

    if constexpr (SWIGLU) {
        static_assert(!SWIGLU || RT == 4, "a wave holds 32 gate rows and the same 32 up rows");
        uint8_t *codes = (uint8_t *)p.y, *scales = codes + (size_t)p.M * (p.N / 2);
        const int n = n0 + 32 * wn;
        if (n >= p.N) return;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const f32x4v gate[2] = {acc[0][tt], acc[1][tt]}, up[2] = {acc[2][tt], acc[3][tt]};
            const int t = first + 16 * (TT * wt + tt) + r16;
            const size_t row = min(t, p.M - 1);
            mx_swiglu_store(gate, up, codes + row * (p.N / 2) + n / 2, scales + row * (p.N / kQK) + n / kQK, t < end);
        }
    } else {
        const bool vec = p.N % 4 == 0;  // y is 16-byte aligned
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int t = first + 16 * (TT * wt + tt) + r16;
            if (t >= end) continue;
            const size_t row = GROUPED && p.g.route_dst != nullptr ? p.g.route_dst[t] : t;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int n = n0 + 16 * (RT * wn + rt) + 4 * q;
                if (n < p.N) mx_store4(p.y, p.dtype, row * p.N + n, acc[rt][tt], p.N - n, vec);
            }
        }
    }
}

template <class Tile, bool SWIGLU>
hipError_t run_tiled(MxTiled p, hipStream_t stream) {
    constexpr int kOutN = SWIGLU ? Tile::kRowsN / 2 : Tile::kRowsN;
    p.tiles_n = (p.N + kOutN - 1) / kOutN;
    p.tiles_t = (p.M + Tile::kRowsT - 1) / Tile::kRowsT + (p.g.offsets != nullptr ? std::min(p.g.n_experts, p.M) : 0);
    const int64_t wgs = (int64_t)p.tiles_n * p.tiles_t;
    if (wgs * Tile::kThreads >= 1LL << 32) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)wgs), block(Tile::kThreads);
    auto go = [&](auto kernel) {
        const hipError_t e = ensure_dynamic_lds((const void *)kernel, Tile::kLds);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, grid, block, Tile::kLds, stream, p);
        return hipGetLastError();
    };
    if (p.g.offsets != nullptr) return go(mxfp4_tiled_kernel<Tile, true, SWIGLU>);
    if constexpr (!SWIGLU) return go(mxfp4_tiled_kernel<Tile, false, false>);
    return hipErrorInvalidValue;
}

typedef MxTile<4, 8, 4, 2> Tile256;  // 256 rows x 256 tokens, 8 waves
typedef MxTile<4, 4, 2, 2> Tile128;  // 128 x 128, 4 waves

}  // namespace

// Rows of at least one stage; byte offsets inside a tile (and of gathered rows) fit 32 bits.
bool mxfp4_tiled_accepts(int K, const MxGroups &g) {
    return K >= 256 && K <= 1 << 23 && (g.src_route == nullptr || (int64_t)g.x_rows * (K / 2) < 1LL << 32);
}

hipError_t launch_mxfp4_tiled(const void *w, const void *xq, void *y, int dtype, int K, int N, int M,
                              const MxGroups &groups, int tile, hipStream_t stream) {
    const MxTiled p{(const uint8_t *)w, nullptr, (const uint8_t *)xq, y, dtype, K, N, M, 0, 0, groups};
    return tile == 256 ? run_tiled<Tile256, false>(p, stream) : run_tiled<Tile128, false>(p, stream);
}

hipError_t launch_mxfp4_tiled_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I,
                                     int M, const MxGroups &groups, int tile, hipStream_t stream) {
    const MxTiled p{(const uint8_t *)w_gate, (const uint8_t *)w_up, (const uint8_t *)xq, mid, JJO_DTYPE_F32, K, I, M,
                    0, 0, groups};
    return tile == 256 ? run_tiled<Tile256, true>(p, stream) : run_tiled<Tile128, true>(p, stream);
}

namespace {
// Rows per expert expected (of M rows in all), or M.
int mean_rows(int M, const MxGroups &g) {
    if (g.offsets == nullptr) return M;
    const int active = std::min(g.n_experts, M);
    return (M + active - 1) / active;
}

// Tile of the staged kernel (256 or 128), or 0 for the direct one.
int tile_for(int K, int N, int M, const MxGroups &g) {
    const int mean = mean_rows(M, g);
    if (mean <= 48 || !mxfp4_tiled_accepts(K, g)) return 0;
    const int64_t groups = g.offsets == nullptr ? 1 : std::min(g.n_experts, M);
    const int64_t t256 = groups * ((mean + 255) / 256) * ((N + 255) / 256);
    return mean > 128 && t256 >= device_cu_count() ? 256 : 128;
}
}  // namespace

hipError_t launch_mxfp4_mm(const void *w, const void *xq, void *y, int dtype, int K, int N, int M,
                           const MxGroups &groups, hipStream_t stream) {
    const int tile = tile_for(K, N, M, groups);
    return tile != 0 ? launch_mxfp4_tiled(w, xq, y, dtype, K, N, M, groups, tile, stream)
                     : launch_mxfp4_direct(w, xq, y, dtype, K, N, M, groups, stream);
}

hipError_t launch_mxfp4_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I, int M,
                               const MxGroups &groups, hipStream_t stream) {
    const int tile = tile_for(K, 2 * I, M, groups);
    return tile != 0 ? launch_mxfp4_tiled_swiglu(w_gate, w_up, xq, mid, K, I, M, groups, tile, stream)
                     : launch_mxfp4_direct_swiglu(w_gate, w_up, xq, mid, K, I, M, groups, stream);
}

}  // namespace jjo
