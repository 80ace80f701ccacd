// MXFP4 weights x MXFP4 activations for prompts and for experts with many rows: tiles staged in
// LDS, gfx950's scaled matrix instruction.
//
//     y[t][n] = sum over blocks b of 2^(sw[n,b] + sx[t,b] - 254) * sum_j cw[n,b,j] * cx[t,b,j]
//
// A stage is 256 values (128 bytes) of every weight row and token row of the tile, two steps of the
// matrix instruction.  The codes go to LDS by DMA, 8 rows of 128 bytes an instruction, the 16-byte
// pieces of a row permuted by its row number (piece ^ row / 2 % 8) so that the 16 lanes that LDS
// serves at a time fall in its 64 banks once; of the stage's 8 blocks lane group q of a step u takes
// block 2q + u, so that a lane's two scale bytes are one 16-bit read and the instruction picks the
// byte.  The scales (8 bytes a row and stage, of any alignment) go through a register of one thread
// per row, two stages at a time.  While a stage is computed the next one lands in the other buffer;
// one barrier per stage.
//
// What bounds it: for prompts the matrix instruction and LDS together (2047 tokens, 14336 x 4096:
// 79 us, 3.0 Pflop/s; 66 without any load; the instruction alone on random data in registers
// reaches 6.2 Pflop/s, a library product of 8192 cubed 3.1); a small product a stage's latency, about
// 1 us.  There the tiles are cut along K as well (KG), into groups of waves with stages of their
// own, so that two or three stages are in flight: 4096 x 4096 and 256 tokens 13.4 us, 17.3 without.
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
    int slices;            // of K, each with its own rows of y
    MxGroups g;
};

// WN x WT waves of RT tiles of 16 weight rows x TT tiles of 16 tokens each; KG groups of such waves
// cut K between them, each with stages of its own; NW stages of weights in LDS (and two of x).
template <int RT_, int TT_, int WN_, int WT_, int KG_ = 1, int NW_ = 2>
struct MxTile {
    static constexpr int RT = RT_, TT = TT_, WN = WN_, WT = WT_, KG = KG_, NW = NW_;
    static constexpr int kWaves = WN * WT, kThreads = 64 * kWaves;  // of a group
    static constexpr int kRowsN = 16 * RT * WN, kRowsT = 16 * TT * WT, kRows = kRowsN + kRowsT;
    static constexpr int kRunsN = kRowsN / 8, kRunsT = kRowsT / 8;  // DMA instructions a stage, and a wave's
    static constexpr int kDmaN = (kRunsN + kWaves - 1) / kWaves, kDmaT = (kRunsT + kWaves - 1) / kWaves;
    static constexpr int kScaleRows = (kRows + kThreads - 1) / kThreads;  // rows a thread
    static constexpr int kStageN = kRowsN * 128, kStageT = kRowsT * 128;
    static constexpr int kGroupLds = NW * kStageN + 2 * kStageT + 2 * kRows * 16;
    static constexpr int kLds = KG * kGroupLds + kRows * 4;
    static_assert(kLds <= 160 * 1024, "LDS of a CU");
    static_assert(KG == 1 || kThreads * RT * TT * 16 <= kGroupLds, "a group's sums fit its stages");
    static_assert(NW == 2 || (NW == 3 && KG == 1), "weights one stage ahead, or two in every other stage");
};

// A wave's outputs (from weight row n, token t on) through its own 4 KB of LDS, 16 tokens at a time:
// the matrix instruction leaves 4 consecutive outputs of a token in a lane, 32 bytes of a row in
// an instruction; read back a row is 16 RT outputs in whole 128-byte lines.  Any N: where rows are not
// aligned the 16-byte stores are not either (2047 tokens, 14335 x 4096: 83 us, 123 by single outputs).
template <class T, int RT, int TT>
__device__ __forceinline__ void store_rows(T *__restrict__ y, const f32x4v (&acc)[RT][TT], uint8_t *stage, int n,
                                           int t, int end, int N, const int32_t *__restrict__ route_dst) {
    constexpr int kVec = 16 / sizeof(T), kChunks = 16 * RT / kVec, kRowsAtOnce = 64 / kChunks;
    const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
    const int row = lane / kChunks, chunk = lane % kChunks;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int at = 16 * rt + 4 * q;
            MxVec<T, 4> v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v.v[i] = (T)acc[rt][tt][i];
            *reinterpret_cast<MxVec<T, 4> *>(stage + r16 * (kChunks * 16) + 16 * ((at / kVec) ^ (r16 % kChunks)) +
                                             at % kVec * sizeof(T)) = v;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < 16 / kRowsAtOnce; ++k) {
            const int r = kRowsAtOnce * k + row, token = t + 16 * tt + r;
            const MxVec<T, kVec> v =
                *reinterpret_cast<const MxVec<T, kVec> *>(stage + r * (kChunks * 16) + 16 * (chunk ^ (r % kChunks)));
            const int at = n + chunk * kVec;
            if (token < end && at < N) {
                T *const to = y + (size_t)(route_dst != nullptr ? route_dst[token] : token) * N + at;
                if (at + kVec <= N) {
                    store_any(to, v);
                } else {
#pragma unroll
                    for (int i = 0; i < kVec - 1; ++i)
                        if (at + i < N) to[i] = v.v[i];
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <class Tile, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(Tile::KG *Tile::kThreads) void mxfp4_tiled_kernel(MxTiled p) {
    constexpr int RT = Tile::RT, TT = Tile::TT;
    constexpr int KG = Tile::KG;
    extern __shared__ __align__(16) uint8_t lds_all[];
    const int lane = threadIdx.x & 63, any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = KG == 1 ? 0 : any_wave / Tile::kWaves, wave = KG == 1 ? any_wave : any_wave % Tile::kWaves;
    const int tid = KG == 1 ? (int)threadIdx.x : 64 * wave + lane;  // in the group
    uint8_t *const lds = lds_all + kg * Tile::kGroupLds, *const lds_x = lds + Tile::NW * Tile::kStageN;
    uint8_t *const lds_scales = lds_x + 2 * Tile::kStageT;
    uint32_t *const lds_rows = reinterpret_cast<uint32_t *>(lds_all + KG * Tile::kGroupLds);
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

    // ---- the DMA: instruction i of a wave takes run kDma * wave + i of 8 rows, a lane piece
    // (lane % 8) ^ (row / 2 % 8) of row lane / 8.  The rows' offsets stand in LDS (in registers
    // they would take up to eight of the 60 and more that every tile leaves).
    const int t0 = GROUPED && p.g.src_route != nullptr ? 0 : first;
    for (int row = threadIdx.x; row < Tile::kRows; row += KG * Tile::kThreads)
        lds_rows[row] = row < Tile::kRowsN ? (uint32_t)(weight_row(row) - n0) * half
                                           : (uint32_t)(token_row(row - Tile::kRowsN) - t0) * half;
    const uint64_t x_base = (uint64_t)p.x + (uint64_t)t0 * half, w_at0 = (uint64_t)(w_first + n0) * half;
    const uint64_t w_base = (uint64_t)p.w + w_at0, w2_base = SWIGLU ? (uint64_t)p.w2 + w_at0 : w_base;
    const uint32_t piece = 16 * ((lane & 7) ^ ((lane >> 4) & 3));  // of an even run of 8 rows; ^ 64 for an odd one
    // ---- and of the scales: one row, or kScaleRows
    const uint8_t *srow[Tile::kScaleRows];
#pragma unroll
    for (int i = 0; i < Tile::kScaleRows; ++i) {
        const int row = min(tid + i * Tile::kThreads, Tile::kRows - 1);
        if (row < Tile::kRowsN)
            srow[i] = (is_up(row) ? p.w2 : p.w) + w_all * half + (w_first + weight_row(row)) * nb;
        else
            srow[i] = p.x + x_all * half + (size_t)token_row(row - Tile::kRowsN) * nb;
    }
    // A pair of stages at a time: 16 bytes of each row are one request.
    uint32_t sv[Tile::kScaleRows][4];
    auto load_scales = [&](int pair) {  // the last pair's bytes end with the row (nb >= 16)
#pragma unroll
        for (int i = 0; i < Tile::kScaleRows; ++i) __builtin_memcpy(sv[i], srow[i] + min(16 * pair, nb - 16), 16);
    };
    auto store_scales = [&](int pair) {
        const int over = 16 * pair + 16 - nb;
#pragma unroll
        for (int i = 0; i < Tile::kScaleRows; ++i) {
            if (over > 0) {  // zeros behind the row's end
                unsigned __int128 v;
                __builtin_memcpy(&v, sv[i], 16);
                v >>= 8 * over;
                __builtin_memcpy(sv[i], &v, 16);
            }
            const int row = tid + i * Tile::kThreads;
            uint8_t *to = lds_scales + (pair & 1) * (Tile::kRows * 16) + row * 8;
            if (row < Tile::kRows) {
                *reinterpret_cast<uint2 *>(to) = make_uint2(sv[i][0], sv[i][1]);
                *reinterpret_cast<uint2 *>(to + Tile::kRows * 8) = make_uint2(sv[i][2], sv[i][3]);
            }
        }
    };
    // The weights' (or x's) part of stage st to its `buffer`-th place.
    auto dma = [&](auto x_tag, int st, int buffer) {
        constexpr bool X = decltype(x_tag)::value;
        constexpr int kRuns = X ? Tile::kRunsT : Tile::kRunsN, kMine = X ? Tile::kDmaT : Tile::kDmaN;
        const uint32_t to = X ? (uint32_t)(uintptr_t)lds_x + buffer * Tile::kStageT
                              : (uint32_t)(uintptr_t)lds + buffer * Tile::kStageN;
        const uint32_t left = 16u * (uint32_t)(nb - 8 * st);  // bytes of the row from the stage on
        const uint32_t most = left >= 128u ? 112u : left - 16u;
        const uint32_t even = min((uint32_t)piece, most), odd = min((uint32_t)piece ^ 64u, most);
        auto run = [&](int i) {  // of 8 rows; the last one again where they do not divide
            const int at = wave * kMine + i;
            return kRuns % Tile::kWaves == 0 ? at : min(at, kRuns - 1);
        };
        uint32_t off[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            off[i] = lds_rows[(X ? Tile::kRowsN : 0) + 8 * run(i) + (lane >> 3)] + (run(i) & 1 ? odd : even);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const uint32_t m0v = __builtin_amdgcn_readfirstlane(to + 1024 * run(i));
            // A mask, not a branch: a choice among captured addresses would go through scratch.
            const uint64_t up = -(uint64_t)is_up(8 * run(i));
            const uint64_t from = (X ? x_base : w_base + (up & (w2_base - w_base))) + (uint64_t)st * 128;
            // Five wait states: an SGPR that a VALU instruction wrote is not read by a load before, nor M0 in the
            // next cycle, and the compiler does not count them for an asm statement.
            asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
                         :
                         : "v"(off[i]), "s"(from), "{m0}"(m0v)
                         : "memory");
        }
    };
    constexpr std::integral_constant<bool, false> kW{};
    constexpr std::integral_constant<bool, true> kX{};

    f32x4v acc[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = f32x4v{0.f, 0.f, 0.f, 0.f};

    // A slice, and in it a group, takes whole pairs of stages.  All run as many rounds as the longest (barriers).
    const int pairs = (stages + 1) / 2, parts = p.slices * KG, part = (int)blockIdx.y * KG + kg;
    const int p_beg = pairs * part / parts, p_end = pairs * (part + 1) / parts;
    const int s_beg = 2 * p_beg, s_end = min(2 * p_end, stages);
    const int rounds = KG == 1 ? s_end - s_beg : 2 * ((pairs + parts - 1) / parts);
    // The last part's last round, where the row ends inside its stage.
    const bool ends = nb % 8 != 0 && (int)blockIdx.y == p.slices - 1;
    const int cut = ends ? stages - 1 - 2 * (pairs * (parts - 1) / parts) : -1;
    load_scales(p_beg);
    __syncthreads();
    dma(kW, s_beg, 0);
    dma(kX, s_beg, 0);
    if constexpr (Tile::NW == 3) dma(kW, min(s_beg + 1, s_end - 1), 1);
    const uint32_t w_at = (uint32_t)(16 * RT * wn + r16), x_at = (uint32_t)(16 * TT * wt + r16);
    int w_buffer = 0;
    const uint32_t sw0 = 16u * ((2 * q) ^ (r16 >> 1)), sw1 = 16u * ((2 * q + 1) ^ (r16 >> 1));
    for (int round = 0; round < rounds; ++round) {
        const int st = s_beg + round;  // s_beg is even
        // Stage st has landed: loads return in order, the last ones are the next stage's weights (NW == 3).  In even
        // stages the compiler waits for the scales' registers below, and not counting the asm's loads it waits for all
        // of them: there the next stage's weights have landed too.
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(Tile::NW == 3 ? Tile::kDmaN : 0) : "memory");
        if ((st & 1) == 0 && (KG == 1 || st < s_end)) store_scales(st >> 1);
        if (round == cut) {  // the row ends inside the last stage: zero weights behind it
            asm volatile("s_barrier" ::: "memory");
            const int over = 8 * stages - nb;
            if (kg == KG - 1)
                for (int i = tid; i < Tile::kRowsN * 8; i += Tile::kThreads)
                    if ((i & 7) >= 8 - over)
                        *reinterpret_cast<u32x4v *>(lds + w_buffer * Tile::kStageN + (i >> 3) * 128 +
                                                    16 * ((i & 7) ^ ((i >> 4) & 7))) = u32x4v{0u, 0u, 0u, 0u};
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        // The next stage on its way; behind the last one, the last again (nothing reads it).
        if ((st & 1) == 0) load_scales(min((st >> 1) + 1, p_end - 1));
        const int w_next = w_buffer == Tile::NW - 1 ? 0 : w_buffer + 1;
        if constexpr (Tile::NW == 2) dma(kW, min(st + 1, s_end - 1), w_next);
        dma(kX, min(st + 1, s_end - 1), (st + 1) & 1);
        if constexpr (Tile::NW == 3) dma(kW, min(st + 2, s_end - 1), w_next == 2 ? 0 : w_next + 1);
        const uint8_t *wbuf = lds + w_buffer * Tile::kStageN, *xbuf = lds_x + (st & 1) * Tile::kStageT;
        w_buffer = w_next;
        if (KG > 1 && st >= s_end) continue;
        const uint8_t *sbuf = lds_scales + (st & 3) * (Tile::kRows * 8);
        uint32_t sw[RT], sx[TT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            sw[rt] = *reinterpret_cast<const uint16_t *>(sbuf + (w_at + 16 * rt) * 8 + 2 * q);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
            sx[tt] = *reinterpret_cast<const uint16_t *>(sbuf + (Tile::kRowsN + x_at + 16 * tt) * 8 + 2 * q);
        auto step = [&](auto u_tag) {
            constexpr int U = decltype(u_tag)::value;
            const uint32_t at = U == 0 ? sw0 : sw1;
            u32x4v a[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) a[rt] = *reinterpret_cast<const u32x4v *>(wbuf + at + (w_at + 16 * rt) * 128);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const u32x4v b = *reinterpret_cast<const u32x4v *>(xbuf + at + (x_at + 16 * tt) * 128);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt][tt] = mx_mfma<U, U>(a[rt], b, acc[rt][tt], sw[rt], sx[tt]);
            }
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outlives the workgroup's LDS

    if constexpr (KG > 1) {  // the other groups' sums, in their order
        f32x4v *const sums = reinterpret_cast<f32x4v *>(lds_all) + tid;
        __syncthreads();  // no wave reads a stage any more
        if (kg > 0) {
#pragma unroll
            for (int i = 0; i < RT * TT; ++i)
                sums[(kg * Tile::kGroupLds / 16) + i * Tile::kThreads] = acc[i / TT][i % TT];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int k = 1; k < KG; ++k)
#pragma unroll
            for (int i = 0; i < RT * TT; ++i)
                acc[i / TT][i % TT] += sums[(k * Tile::kGroupLds / 16) + i * Tile::kThreads];
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
        if constexpr (KG == 1) __syncthreads();  // no wave reads a stage any more
        uint8_t *stage = lds + wave * 4096;
        const int nw = n0 + 16 * RT * wn, tw = first + 16 * TT * wt;
        const int32_t *route_dst = GROUPED ? p.g.route_dst : nullptr;
        if (p.dtype == JJO_DTYPE_F32)
            store_rows<float, RT, TT>((float *)p.y + (size_t)blockIdx.y * p.M * p.N, acc, stage, nw, tw, end, p.N,
                                      route_dst);
        else if (p.dtype == JJO_DTYPE_F16)
            store_rows<_Float16, RT, TT>((_Float16 *)p.y, acc, stage, nw, tw, end, p.N, route_dst);
        else store_rows<__bf16, RT, TT>((__bf16 *)p.y, acc, stage, nw, tw, end, p.N, route_dst);
    }
}

template <class Tile, bool SWIGLU>
hipError_t run_tiled(MxTiled p, hipStream_t stream) {
    constexpr int kOutN = SWIGLU ? Tile::kRowsN / 2 : Tile::kRowsN;
    p.tiles_n = (p.N + kOutN - 1) / kOutN;
    p.tiles_t = (p.M + Tile::kRowsT - 1) / Tile::kRowsT + (p.g.offsets != nullptr ? std::min(p.g.n_experts, p.M) : 0);
    const int64_t wgs = (int64_t)p.tiles_n * p.tiles_t;
    if (wgs * Tile::KG * Tile::kThreads >= 1LL << 32) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)wgs, (unsigned)p.slices), block(Tile::KG * Tile::kThreads);
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

struct MxTileChoice {
    int tokens;  // 0: the direct kernel
    bool split;  // K cut inside the workgroup
    float cost;  // of a whole tile's rounds: us at K = 4096
};

// 128 weight rows on four waves up to 128 tokens, 256 on eight above; there the weights come two stages
// ahead where LDS has room, in every other stage (the wait for the scales drains them in the rest; 8
// experts of 28672 rows, 128 tokens each: 152 us on tiles of 160, 159 with one stage ahead; no difference
// where several token tiles read the same weights).
template <bool SWIGLU>
hipError_t run_tile(const MxTiled &p, const MxTileChoice &tile, hipStream_t stream) {
    if (tile.split) {
        switch (tile.tokens) {
            case 32: return run_tiled<MxTile<4, 1, 2, 2, 3>, SWIGLU>(p, stream);
            case 64: return run_tiled<MxTile<4, 2, 2, 2, 2>, SWIGLU>(p, stream);
            case 96: return run_tiled<MxTile<4, 3, 2, 2, 2>, SWIGLU>(p, stream);
            case 128: return run_tiled<MxTile<4, 4, 2, 2, 2>, SWIGLU>(p, stream);
        }
        return hipErrorInvalidValue;
    }
    switch (tile.tokens) {
        case 32: return run_tiled<MxTile<4, 1, 2, 2>, SWIGLU>(p, stream);
        case 64: return run_tiled<MxTile<4, 2, 2, 2>, SWIGLU>(p, stream);
        case 96: return run_tiled<MxTile<4, 3, 2, 2>, SWIGLU>(p, stream);
        case 128: return run_tiled<MxTile<4, 4, 2, 2>, SWIGLU>(p, stream);
        case 160: return run_tiled<MxTile<4, 5, 4, 2, 1, 3>, SWIGLU>(p, stream);
        case 192: return run_tiled<MxTile<4, 6, 4, 2, 1, 3>, SWIGLU>(p, stream);
        case 256: return run_tiled<MxTile<4, 8, 4, 2>, SWIGLU>(p, stream);
    }
    return hipErrorInvalidValue;
}

// Rows of at least two stages; byte offsets inside a tile (and of gathered rows) fit 32 bits.
bool tiles_accept(int K, const MxGroups &g) {
    return K >= 512 && K <= 1 << 23 && (g.src_route == nullptr || (int64_t)g.x_rows * (K / 2) < 1LL << 32);
}

// The kernel of a product with N weight rows in all (gate and up together).
//
// The direct kernel is bound by its workgroups' work, a tile by the latency of its stages, which is
// the same for any output up to a tile per CU: 4096 x 4096 (N x K) and 64 / 128 / 256 tokens 7.6 /
// 11.7 / 18.8 us direct against 13.5 / 13.3 / 13.4 us on split tiles, 8192 x 14336 and 64 / 96 tokens
// 36 / 52 against 38 / 38 us.  They meet at 8 workgroups of 16 rows x 16 tokens a CU (4 where K <
// 2048: 32768 x 1024 and 12 tokens, 8 a CU, 8.4 against 7.2 us).  Behind that the matrix itself is the
// bound: up to 16 tokens the direct kernel reads it as fast from K = 4096 on (131072 x 4096, 16
// tokens: 59 against 63 us).
//
// Split tiles where the smallest tile that leaves at most one workgroup a CU can do it (4096 x 4096,
// 256 tokens: 13.4 against 17.3 us; 14336 x 4096, 256: 20.4 against 21.9; 4096 x 11008, 512: 27.6
// against 34).  Otherwise the tile whose rounds over the CUs cost least; kCost is a round's time in
// us at K = 4096 with each CU's share of workgroups in flight (14336 x 4096: tiles of 96 take 22 us
// for 384 tokens, 128 26 for 512, 160 31 for 640, 192 34 for 768, 256 41 for 1024, and each of the
// others there is slower; 8 experts of 28672 rows with 128 tokens each: 160 152 us, 192 163, 128 191).
MxTileChoice tile_for(int K, int64_t N, int M, const MxGroups &g, int64_t cus) {
    const int64_t experts = mx_experts(M, g), rows = mx_rows(M, g);
    const int64_t mean = (M + experts - 1) / experts;
    const int64_t small = experts * ((N + 15) / 16) * ((rows + 15) / 16);
    const int most = g.offsets == nullptr ? 16 : 10;  // an uneven share of 10 rows is 16 and more for some
    if (!tiles_accept(K, g) || mean <= 4 || small <= (K < 2048 ? 4 : 8) * cus || (mean <= most && K >= 4096))
        return {0, false, 0.f};
    auto rounds = [&](int tokens) {
        const int64_t n = tokens <= 128 ? 128 : 256;
        return (experts * ((rows + tokens - 1) / tokens) * ((N + n - 1) / n) + cus - 1) / cus;
    };
    if (K >= 2048)
        for (int tokens : {32, 64, 96, 128})
            if (rounds(tokens) == 1) return {tokens, true, 0.f};
    MxTileChoice best{0, false, 0.f};
    constexpr struct {
        int tokens;
        float cost;
    } kCost[] = {{32, 9.f}, {64, 10.f}, {96, 11.5f}, {128, 14.f}, {160, 28.5f}, {192, 31.f}, {256, 39.5f}};
    for (const auto &c : kCost) {
        const float cost = (float)rounds(c.tokens) * c.cost;
        if (best.tokens == 0 || cost < best.cost) best = {c.tokens, false, cost};
    }
    return best;
}

}  // namespace

// Two slices of K (fp32 outputs, added by the reader) for experts whose whole tiles leave
// CUs without work: the cheapest tile for half the length on twice the workgroups, against the
// cheapest for all of it (of the difference 0.4 to 0.5 was measured) and the second slice's way
// through memory, 4 bytes an output at 5 TB/s.  8 experts, K = 14336 to 4096: of 128 rows each 66 us on
// tiles of 160 rows in two slices, 80 on two tiles of 96 rows an expert; of 225 rows 84 and 99, of 512
// 199 and 225.  The workspace depends on it, so the rule takes the chip's 256 CUs and not the
// device's.
constexpr int64_t kMxCus = 256;
int mxfp4_down_slices(int K, int N, int M, int n_experts) {
    MxGroups g;
    static const int32_t grouped = 0;
    g.offsets = &grouped, g.n_experts = n_experts;
    const MxTileChoice one = tile_for(K, N, M, g, kMxCus);
    if (one.tokens == 0 || one.split || K < 4096) return 1;
    const MxTileChoice two = tile_for(K, N, M, g, kMxCus / 2);  // tiles as well, and whole ones: fewer CUs
    return 0.4f * (one.cost - 0.5f * two.cost) * (float)K / 4096.f > (float)M * (float)N * 4.f / 5e6f ? 2 : 1;
}

hipError_t launch_mxfp4_mm(const void *w, const void *xq, void *y, int dtype, int K, int N, int M,
                           const MxGroups &groups, hipStream_t stream, int slices) {
    // A tile for half the length costs half, on twice the workgroups: as if there were half the CUs.
    const MxTileChoice tile = tile_for(K, N, M, groups, slices == 1 ? device_cu_count() : kMxCus / slices);
    if (tile.tokens == 0)
        return slices == 1 ? launch_mxfp4_direct(w, xq, y, dtype, K, N, M, groups, stream) : hipErrorInvalidValue;
    const MxTiled p{(const uint8_t *)w, nullptr, (const uint8_t *)xq, y, dtype, K, N, M, 0, 0, slices, groups};
    return run_tile<false>(p, tile, stream);
}

hipError_t launch_mxfp4_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I, int M,
                               const MxGroups &groups, hipStream_t stream) {
    const MxTileChoice tile = tile_for(K, 2 * (int64_t)I, M, groups, device_cu_count());
    if (tile.tokens == 0) return launch_mxfp4_direct_swiglu(w_gate, w_up, xq, mid, K, I, M, groups, stream);
    const MxTiled p{(const uint8_t *)w_gate, (const uint8_t *)w_up, (const uint8_t *)xq, mid, JJO_DTYPE_F32, K, I, M,
                    0, 0, 1, groups};
    return run_tile<true>(p, tile, stream);
}

}  // namespace jjo
