// Products of float matrices on LDS tiles: see rows_mm.hpp for the four forms.
//
// out[Q][P] += Qmat[Q][K] . Pmat[P][K]^T.  A stage is 128 bytes of the sums' direction (64 elements of 16
// bits, 32 of 32) of every row of the tile's two operands, two steps of the matrix instruction.  Where
// a row's elements are contiguous, its 128 bytes are a row of LDS, 16-byte pieces permuted by the row
// (piece ^ row / 2 % 8); where the rows of an element are, an LDS row is one element of all the tile's
// rows, and the transposing LDS read puts four elements of a row into a lane; pieces are permuted by
// the element's number so that the lanes served together fall into different banks.
#pragma once

#include <hip/hip_runtime.h>

#include "mxfp4_mm.hpp"
#include "rows_mm.hpp"

namespace jjo {
namespace {

typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef short s16x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

// acc[16 of P][16 of Q] += 16 bytes of a row in each lane (row lane % 16, piece lane / 16 of four).  A lane's
// acc holds P rows 4 * (lane / 16) + 0..3 of Q row lane % 16.
template <class T>
__device__ __forceinline__ f32x4v rows_mfma(u32x4v p, u32x4v q, f32x4v acc) {
    if constexpr (std::is_same_v<T, __bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, p), __builtin_bit_cast(bf16x8v, q),
                                                       acc, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8v, p), __builtin_bit_cast(f16x8v, q),
                                                      acc, 0, 0, 0);
    } else {
        const f32x4v a = __builtin_bit_cast(f32x4v, p), b = __builtin_bit_cast(f32x4v, q);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
        return acc;
    }
}

// WP x WQ waves of RT tiles of 16 output columns x TT tiles of 16 output rows each, NB stages in LDS.
template <int RT_, int TT_, int WP_, int WQ_, int NB_ = 2>
struct RowsTile {
    static constexpr int RT = RT_, TT = TT_, WP = WP_, WQ = WQ_, NB = NB_;
    static constexpr int kWaves = WP * WQ, kThreads = 64 * kWaves;
    static constexpr int kP = 16 * RT * WP, kQ = 16 * TT * WQ;
    static constexpr int kStageP = kP * 128, kStageQ = kQ * 128, kStage = kStageP + kStageQ;
    static constexpr int kLds = NB * kStage;
    static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

// One operand's part of a stage: ROWS rows of the tile, TRANS: the rows of an element contiguous.
template <class T, bool TRANS, int ROWS, int THREADS>
struct RowsOperand {
    static constexpr int kPiece = 16 / sizeof(T), kStep = 128 / sizeof(T);
    static constexpr int kPitch = TRANS ? ROWS * (int)sizeof(T) : 128;  // bytes of an LDS row
    static constexpr int kRowPieces = kPitch / 16;
    static constexpr int kRuns = ROWS / 8, kWaves = THREADS / 64;  // of 64 pieces: a DMA instruction's
    static constexpr int kMine = (kRuns + kWaves - 1) / kWaves;    // of a wave
    static_assert(!TRANS || ROWS % 128 == 0 || ROWS == 64, "the permutations below");

    // The permutation of element k's pieces (of 16 bits: pairs, 16 rows each; of 32: fours).
    static __device__ __forceinline__ int swizzle(int k) {
        if constexpr (sizeof(T) == 4) return 4 * ((k >> 2) & 3);
        else if constexpr (ROWS == 64) return 2 * (((k >> 1) & 1) + 2 * ((k >> 3) & 1));
        else return 2 * ((k & 3) + 4 * ((k >> 3) & 1));
    }
    // What stands in the piece at place `at` of LDS: row i and element k of the stage (the first ones).
    static __device__ __forceinline__ void piece(int at, int &i, int &k) {
        const int line = at / kRowPieces, place = at % kRowPieces;
        if constexpr (TRANS) k = line, i = (place ^ swizzle(line)) * kPiece;
        else i = line, k = (place ^ ((line >> 1) & 7)) * kPiece;
    }
    // A wave's n-th run; the last one again where they do not divide.
    static __device__ __forceinline__ int run(int wave, int n) {
        return kRuns % kWaves == 0 ? wave * kMine + n : min(wave * kMine + n, kRuns - 1);
    }
    static __device__ __forceinline__ int64_t offset(int i, int k, int64_t ld) {
        return TRANS ? k * ld + i : i * ld + k;
    }

    // ---- through registers: any address.  `from`(i, k, have) is the address of a piece, `have` the elements
    // from it on that exist (zeros behind them).
    template <class F>
    static __device__ __forceinline__ void copy(F from, uint8_t *lds) {
        u32x4v v[kMine];
        const int tid = threadIdx.x;
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            int i, k, have;
            piece(64 * run(tid >> 6, n) + (tid & 63), i, k);
            const T *const at = from(i, k, have);
            v[n] = u32x4v{0u, 0u, 0u, 0u};
            if (have >= kPiece) {
                v[n] = load_any<u32x4v>(at);
            } else if (have > 0) {
                MxVec<T, kPiece> e;
#pragma unroll
                for (int j = 0; j < kPiece; ++j) e.v[j] = j < have ? at[j] : (T)0.0f;
                v[n] = __builtin_bit_cast(u32x4v, e);
            }
        }
#pragma unroll
        for (int n = 0; n < kMine; ++n)
            *reinterpret_cast<u32x4v *>(lds + 16 * (64 * run(tid >> 6, n) + (tid & 63))) = v[n];
    }

    // ---- by DMA, 64 pieces an instruction: a lane's offsets; rows behind the last are the last again.
    template <class F>
    static __device__ __forceinline__ void dma_offsets(uint32_t (&off)[kMine], int wave, int64_t ld, F row) {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            int i, k;
            piece(64 * run(wave, n) + (threadIdx.x & 63), i, k);
            off[n] = (uint32_t)(offset(row(i), k, ld) * sizeof(T));
        }
    }

    // ---- a lane's 16 bytes of a step's operand, rows base + 16 * t + lane % 16
    // (base a multiple of 16 times the tiles that are read from it; those are a power of two where TRANS).
    struct Reader {
        uint32_t at[TRANS ? 1 : 2];
        __device__ __forceinline__ explicit Reader(int base) {
            const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
            if constexpr (!TRANS) {
#pragma unroll
                for (int u = 0; u < 2; ++u) at[u] = (base + r16) * 128 + 16 * ((4 * u + q) ^ (r16 >> 1));
            } else if constexpr (sizeof(T) == 4) {
                at[0] = 4 * q * kPitch + 64 * ((base / 16) ^ q) + 4 * r16;
            } else {
                at[0] = (8 * q + (r16 >> 2)) * kPitch + 32 * ((base / 16) ^ (swizzle(8 * q + (r16 >> 2)) / 2)) +
                        8 * (r16 & 3);
            }
        }
        template <int U>
        __device__ __forceinline__ u32x4v read(const uint8_t *lds, int t) const {
            if constexpr (!TRANS) {
                return *reinterpret_cast<const u32x4v *>(lds + at[U] + t * 2048);
            } else if constexpr (sizeof(T) == 4) {
                const uint8_t *const from = lds + (at[0] ^ (64 * t));
                u32x4v v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t *>(from + (16 * U + j) * kPitch);
                return v;
            } else {
                typedef __attribute__((address_space(3))) s16x4v Lds;
                const uint8_t *const from = lds + (at[0] ^ (32 * t)) + 32 * U * kPitch;
                const u32x2v a = __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds *)from));
                const u32x2v b =
                    __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds *)(from + 4 * kPitch)));
                return u32x4v{a[0], a[1], b[0], b[1]};
            }
        }
    };
};

// Of tiles a and b (a lane holds columns 4 * (lane / 16) + 0..3 of both) eight columns of one: lanes 0..15
// columns 0..7 of a, the next 16 those of b, then columns 8..15 of a and of b.
__device__ __forceinline__ void rows_exchange(f32x4v a, f32x4v b, float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[i]), __float_as_uint(b[i]), false, false);
        v[i] = __uint_as_float(s[0]), v[4 + i] = __uint_as_float(s[1]);
    }
}

// 64 pieces of 16 bytes to LDS.
__device__ __forceinline__ void rows_dma(uint32_t off, uint64_t from, uint32_t lds) {
    const uint32_t m0v = __builtin_amdgcn_readfirstlane(lds);
    from = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(from >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)from);
    // Five wait states: an SGPR that a VALU instruction wrote is not read by a load before, nor M0 in the
    // next cycle, and the compiler does not count them for an asm statement.
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(from), "{m0}"(m0v) : "memory");
}

// Workgroups go to the eight XCDs in turn: each takes a contiguous run of `total` tiles, so that tiles
// that read the same rows follow each other in one L2.  -1 behind the last.
__device__ __forceinline__ int rows_xcd_run(int block, int total) {
    const int per = total / 8, rest = total % 8, xcd = block % 8, at = block / 8;
    return at < per + (xcd < rest) ? xcd * per + min(xcd, rest) + at : -1;
}

// The workgroup's tile of `rows` sorted rows x one of tiles_p of their expert's columns: expert by expert, its
// row tiles fastest; false behind the last.  Ranges are clamped to [0, M], so a malformed table
// drops rows instead of leaving the buffers.  All lanes of a wave call it together.
__device__ __forceinline__ bool rows_expert_tile(const int32_t *__restrict__ offsets, int n_experts, int M, int rows,
                                                 int tiles_p, int &expert, int &first, int &end, int &tile_p) {
    const int lane = threadIdx.x & 63;
    int beg = 0, fin = 0, incl = 0, mine = 0, total = 0;
    auto count = [&](int e0) {
        const int e = e0 + lane;
        beg = fin = 0;
        if (e < n_experts) {
            beg = min(max(offsets[e], 0), M);
            fin = min(max(offsets[e + 1], beg), M);
        }
        mine = (fin - beg + rows - 1) / rows;
        incl = mx_scan(mine);
    };
    for (int e0 = 0; e0 < n_experts; e0 += 64) {
        count(e0);
        total += __builtin_amdgcn_readlane(incl, 63);
    }
    const int64_t all = (int64_t)total * tiles_p;
    if (all > gridDim.x) return false;  // only the sums of a malformed table
    const int tile = rows_xcd_run(blockIdx.x, (int)all);
    if (tile < 0) return false;
    int base = 0;
    for (int e0 = 0; e0 < n_experts; e0 += 64) {
        if (n_experts > 64) count(e0);
        const uint64_t past = __ballot((int64_t)(base + incl) * tiles_p > tile);
        if (past != 0) {
            const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
            const int tiles = __builtin_amdgcn_readlane(mine, l);
            const int local = tile - (base + __builtin_amdgcn_readlane(incl, l) - tiles) * tiles_p;
            if (tiles <= 0 || local < 0) return false;
            expert = e0 + l;
            first = __builtin_amdgcn_readlane(beg, l) + local % tiles * rows;
            end = __builtin_amdgcn_readlane(fin, l);
            tile_p = local / tiles;
            return first < end && tile_p < tiles_p;
        }
        base += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// The same from an address of each lane's own.
__device__ __forceinline__ void rows_dma(const void *from, uint32_t lds) {
    const uint32_t m0v = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "{m0}"(m0v) : "memory");
}

__device__ const uint32_t rows_zeros[4] = {0u, 0u, 0u, 0u};  // the pieces behind the sums' end

// DMA: the operands' memory rows are 16-byte aligned, the sums' elements whole pieces, and a tile's offsets
// fit 32 bits; other operands go through registers.
template <class E, RowsMode MODE, class Tile, bool DMA>
__global__ __launch_bounds__(Tile::kThreads) void rows_mm_kernel(RowsMm p) {
    typedef typename E::type T;
    constexpr int RT = Tile::RT, TT = Tile::TT, kStep = 128 / sizeof(T);
    constexpr bool PT = MODE == kRowsInput || MODE == kRowsWeight, QT = MODE == kRowsWeight;
    using OpP = RowsOperand<T, PT, Tile::kP, Tile::kThreads>;
    using OpQ = RowsOperand<T, QT, Tile::kQ, Tile::kThreads>;
    // SwiGLU: a wave's first columns are gate's, the other half up's of the same.
    constexpr int kOutP = MODE == kRowsSwiglu ? Tile::kP / 2 : Tile::kP;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, q4 = lane >> 4;
    const int wp = wave % Tile::WP, wq = wave / Tile::WP;

    int expert = 0, first = 0, end = p.Q, half = 0, q0, tile_p, length = p.K;
    if constexpr (MODE == kRowsWeight) {
        const int each = p.tiles_p * p.tiles_q;
        int tile = rows_xcd_run(blockIdx.x, gridDim.x);
        if (p.offsets != nullptr) {
            expert = tile / each, tile %= each;
            first = min(max(p.offsets[expert], 0), p.M);
            length = min(max(p.offsets[expert + 1], first), p.M) - first;
        }
        const int tiles_half = p.tiles_q / p.halves, tile_q = tile % p.tiles_q;
        half = tile_q / tiles_half;
        q0 = tile_q % tiles_half * Tile::kQ;
        tile_p = tile / p.tiles_q;
    } else if (p.offsets == nullptr) {
        const int tile = rows_xcd_run(blockIdx.x, gridDim.x);
        q0 = tile % p.tiles_q * Tile::kQ;
        tile_p = tile / p.tiles_q;
    } else if (!rows_expert_tile(p.offsets, p.n_experts, p.M, Tile::kQ, p.tiles_p, expert, q0, end, tile_p)) {
        return;
    }
    const int p0 = tile_p * kOutP;
    const int rows_p = min(p.P - p0, kOutP), rows_q = min(end - q0, Tile::kQ);

    // The operands from the tile's first row and the sums' first element on.
    const T *const pm = (const T *)p.p + (MODE == kRowsWeight ? first * p.ldp + p0
                                                              : expert * p.expert_stride + (PT ? p0 : p0 * p.ldp));
    const T *const pm2 = MODE == kRowsWeight ? pm : (const T *)p.p2 + (pm - (const T *)p.p);
    const T *const qm = (const T *)p.q + (QT ? first * p.ldq + (int64_t)half * p.Q + q0 : q0 * p.ldq);
    const T *const qm2 = MODE == kRowsWeight ? (const T *)p.q2 + (qm - (const T *)p.q) : qm;

    const int stages_half = (length + kStep - 1) / kStep;
    const int stages = MODE == kRowsInput ? p.halves * stages_half : MODE == kRowsWeight ? p.terms * stages_half : stages_half;
    const int s_beg = (int)((int64_t)stages * blockIdx.y / p.slices);
    const int s_end = (int)((int64_t)stages * (blockIdx.y + 1) / p.slices);

    // Row i of the P operand's part of a stage: of SwiGLU a wave's first 8 * RT are gate's, the others up's.
    auto is_up = [&](int i) { return MODE == kRowsSwiglu && i % (16 * RT) >= 8 * RT; };
    auto row_p = [&](int i) { return MODE == kRowsSwiglu ? i / (16 * RT) * (8 * RT) + i % (8 * RT) : i; };
    uint32_t off_p[OpP::kMine], off_q[OpQ::kMine];
    if constexpr (DMA) {
        OpP::dma_offsets(off_p, wave, p.ldp, [&](int i) { return min(row_p(i), PT ? rows_p - OpP::kPiece : rows_p - 1); });
        OpQ::dma_offsets(off_q, wave, p.ldq, [&](int i) { return min(i, QT ? rows_q - OpQ::kPiece : rows_q - 1); });
    }
    auto bring = [&](int st, int buffer) {
        const bool second = (MODE == kRowsInput || MODE == kRowsWeight) && st >= stages_half;
        const int k0 = (second ? st - stages_half : st) * kStep, left = length - k0;
        uint8_t *const to = lds + buffer * Tile::kStage;
        const T *const from_p = (second ? pm2 : pm) + (PT ? k0 * p.ldp : k0);
        const T *const from_up = MODE == kRowsSwiglu ? pm2 + k0 : from_p;
        const T *const from_q = (MODE == kRowsWeight && second ? qm2 : qm) +
                                (QT ? k0 * p.ldq : (second ? p.K : 0) + (int64_t)k0);
        if constexpr (DMA) {
            const uint32_t at = (uint32_t)(uintptr_t)to;
            if (left >= kStep) {
#pragma unroll
                for (int n = 0; n < OpP::kMine; ++n) {
                    const int run = OpP::run(wave, n);  // of SwiGLU 8 rows of one matrix
                    rows_dma(off_p[n], (uint64_t)(is_up(8 * run) ? from_up : from_p), at + 1024 * run);
                }
#pragma unroll
                for (int n = 0; n < OpQ::kMine; ++n) {
                    const int run = OpQ::run(wave, n);
                    rows_dma(off_q[n], (uint64_t)from_q, at + Tile::kStageP + 1024 * run);
                }
            } else {  // the sums end inside the stage
                int in_run = lane;
                asm volatile("" : "+v"(in_run));  // one stage of many: nothing kept in registers for it
#pragma unroll
                for (int n = 0; n < OpP::kMine; ++n) {
                    int i, k;
                    const int run = OpP::run(wave, n);
                    OpP::piece(64 * run + in_run, i, k);
                    const T *const from = (is_up(8 * run) ? from_up : from_p) + off_p[n] / sizeof(T);
                    rows_dma(k < left ? (const void *)from : rows_zeros, at + 1024 * run);
                }
#pragma unroll
                for (int n = 0; n < OpQ::kMine; ++n) {
                    int i, k;
                    const int run = OpQ::run(wave, n);
                    OpQ::piece(64 * run + in_run, i, k);
                    rows_dma(k < left ? (const void *)(from_q + off_q[n] / sizeof(T)) : rows_zeros,
                             at + Tile::kStageP + 1024 * run);
                }
            }
        } else {
            OpP::copy([&](int i, int k, int &have) {
                const int row = row_p(i);
                have = PT ? (k < left ? rows_p - row : 0) : (row < rows_p ? left - k : 0);
                return (is_up(i) ? from_up : from_p) + OpP::offset(row, k, p.ldp);
            }, to);
            OpQ::copy([&](int i, int k, int &have) {
                have = QT ? (k < left ? rows_q - i : 0) : (i < rows_q ? left - k : 0);
                return from_q + OpQ::offset(i, k, p.ldq);
            }, to + Tile::kStageP);
        }
    };

    f32x4v acc[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = f32x4v{0.f, 0.f, 0.f, 0.f};

    const typename OpP::Reader read_p(16 * RT * wp);
    const typename OpQ::Reader read_q(16 * TT * wq);
    constexpr int kDma = OpP::kMine + OpQ::kMine;  // of a wave and stage
    constexpr int kAhead = Tile::NB - 1;           // stages on their way while one is multiplied
    u32x4v a[RT], b[TT];
    auto read = [&](auto u_tag, int buffer) {
        constexpr int U = decltype(u_tag)::value;
        const uint8_t *const in_p = lds + buffer * Tile::kStage, *const in_q = in_p + Tile::kStageP;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) a[rt] = read_p.template read<U>(in_p, rt);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) b[tt] = read_q.template read<U>(in_q, tt);
    };
    auto multiply = [&]() {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][tt] = rows_mfma<T>(a[rt], b[tt], acc[rt][tt]);
    };
    constexpr std::integral_constant<int, 0> kU0{};
    constexpr std::integral_constant<int, 1> kU1{};
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (s_beg + i < s_end) bring(s_beg + i, i);
    int buffer = 0;
    if constexpr (Tile::kWaves == 8) {
        // Two waves a SIMD, one half of the waves a slot behind the other: while one reads its operands of a step,
        // the other multiplies.  A barrier ends each slot.
        auto slot_end = [&]() {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        // The next stage has landed (stages behind it may be on their way).
        auto landed = [&](int next) {
            if (next + kAhead - 1 < s_end) asm volatile("s_waitcnt vmcnt(%0)" ::"i"((kAhead - 1) * kDma) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        };
        auto products = [&]() {
            __builtin_amdgcn_s_setprio(1);
            multiply();
            __builtin_amdgcn_s_setprio(0);
        };
        if (s_beg < s_end) landed(s_beg);
        slot_end();
        if (wave >= 4) slot_end();
        for (int st = s_beg; st < s_end; ++st) {
            // Into the buffer of stage st - 1, whose last readers' slot has ended.
            if (st + kAhead < s_end) bring(st + kAhead, buffer == 0 ? Tile::NB - 1 : buffer - 1);
            read(kU0, buffer);
            slot_end();
            products();
            slot_end();
            read(kU1, buffer);
            if (wave >= 4 && st + 1 < s_end) landed(st + 1);
            slot_end();
            products();
            if (wave < 4 && st + 1 < s_end) landed(st + 1);
            slot_end();
            buffer = buffer == Tile::NB - 1 ? 0 : buffer + 1;
        }
        if (wave < 4) slot_end();
    } else {
        for (int st = s_beg; st < s_end; ++st) {
            // Stage st has landed, and no wave reads the buffer of stage st - 1 any more.
            if (st + kAhead - 1 < s_end)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((kAhead - 1) * kDma) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (st + kAhead < s_end) bring(st + kAhead, buffer == 0 ? Tile::NB - 1 : buffer - 1);
            read(kU0, buffer);
            multiply();
            read(kU1, buffer);
            multiply();
            buffer = buffer == Tile::NB - 1 ? 0 : buffer + 1;
        }
    }

    // ---- outputs straight from the registers: of two tiles side by side lanes exchange halves, so that each
    // holds eight columns of a row and a row's four lanes 64 contiguous bytes (of 16 bits).
    const bool parts = p.slices > 1;
    void *const y = MODE == kRowsWeight ? (void *)((uint8_t *)(half == 0 ? p.y : p.y2) +
                                                   expert * p.expert_stride * (p.wide ? 4 : sizeof(T)))
                                        : p.y;
    auto finish = [&](int in_tile, int column, float *v, float *up) {
        const int col = p0 + column, n = min(8, p.P - col);
        if (in_tile >= rows_q || n <= 0) return;
        const int64_t row = q0 + in_tile;
        if (parts) {
            const int64_t cols = MODE == kRowsSwiglu ? 2 * (int64_t)p.P : p.P;
            // A slice's rows: of weight those of all matrices.
            const int64_t matrices = max(p.n_experts, 1);
            const int64_t all = MODE == kRowsWeight ? p.Q * p.halves * matrices : p.Q;
            const int64_t mine = MODE == kRowsWeight ? (half * matrices + expert) * p.Q + row : row;
            float *const to = p.part + (blockIdx.y * all + mine) * cols + col;
            rows_store8(to, n, v);
            if constexpr (MODE == kRowsSwiglu) rows_store8(to + p.P, n, up);
        } else if constexpr (MODE == kRowsSwiglu) {
            rows_finish_swiglu<T>(p.epi, v, up, row, col, n, p.P, y);
        } else {
            rows_finish<T>(p.epi, v, row, col, n, p.P, y, p.ldy, p.wide);
        }
    };
    constexpr int kWaveP = MODE == kRowsSwiglu ? 8 * RT : 16 * RT;  // columns of a wave
    if constexpr (kWaveP % 32 == 0) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int rt = 0; rt < kWaveP / 16; rt += 2) {
                float v[8], up[8];
                rows_exchange(acc[rt][tt], acc[rt + 1][tt], v);
                if constexpr (MODE == kRowsSwiglu) rows_exchange(acc[RT / 2 + rt][tt], acc[RT / 2 + rt + 1][tt], up);
                finish(16 * (TT * wq + tt) + r16, kWaveP * wp + 16 * (rt + (q4 & 1)) + 8 * (q4 >> 1), v, up);
            }
    } else {  // one tile of columns: of two tiles of rows
        static_assert(TT % 2 == 0 && RT == 2 && MODE == kRowsSwiglu, "the small tile's gate and up");
#pragma unroll
        for (int tt = 0; tt < TT; tt += 2) {
            float v[8], up[8];
            rows_exchange(acc[0][tt], acc[0][tt + 1], v);
            rows_exchange(acc[1][tt], acc[1][tt + 1], up);
            finish(16 * (TT * wq + tt + (q4 & 1)) + r16, 16 * wp + 8 * (q4 >> 1), v, up);
        }
    }
}

template <class E, RowsMode MODE, class Tile, bool DMA>
hipError_t run_rows(RowsMm p, hipStream_t stream) {
    constexpr int kOutP = MODE == kRowsSwiglu ? Tile::kP / 2 : Tile::kP;
    p.tiles_p = (p.P + kOutP - 1) / kOutP;
    p.tiles_q = (p.Q + Tile::kQ - 1) / Tile::kQ;
    int64_t wgs;
    if (MODE == kRowsWeight) {
        p.tiles_q *= p.halves;
        wgs = (int64_t)p.tiles_p * p.tiles_q * (p.offsets != nullptr ? p.n_experts : 1);
        if ((int64_t)p.tiles_p * p.tiles_q > INT32_MAX) return hipErrorInvalidConfiguration;
    } else {
        if (p.offsets != nullptr) p.tiles_q += std::min(p.n_experts, p.M);
        wgs = (int64_t)p.tiles_p * p.tiles_q;
    }
    if (wgs * Tile::kThreads >= 1LL << 32) return hipErrorInvalidConfiguration;
    const auto kernel = rows_mm_kernel<E, MODE, Tile, DMA>;
    const hipError_t e = ensure_dynamic_lds((const void *)kernel, Tile::kLds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)wgs, (unsigned)p.slices), dim3(Tile::kThreads), Tile::kLds, stream, p);
    return hipGetLastError();
}

// DMA where every memory row of both operands is 16-byte aligned, a tile's rows and a stage's elements
// are within 4 GiB of its first, and (where rows of an element are contiguous) rows come in whole pieces.
inline bool rows_dma_accepts(RowsMode mode, int es, const RowsMm &p) {
    const int piece = 16 / es;
    auto fits = [&](const void *m, int64_t ld) {
        return (uintptr_t)m % 16 == 0 && ld % piece == 0 && ld * es < (1LL << 32) / 512;
    };
    if (!fits(p.p, p.ldp) || !fits(p.q, p.ldq)) return false;
    if (p.p2 != nullptr && !fits(p.p2, p.ldp)) return false;
    if (p.q2 != nullptr && !fits(p.q2, p.ldq)) return false;
    if (mode == kRowsWeight) return p.P % piece == 0 && p.Q % piece == 0;
    return p.K % piece == 0 && (mode != kRowsInput || p.P % piece == 0);
}

template <class E, RowsMode MODE>
hipError_t rows_by_tile(const RowsMm &p, int tile, hipStream_t stream) {
    if (!rows_dma_accepts(MODE, (int)sizeof(typename E::type), p)) return run_rows<E, MODE, RowsTile<4, 4, 2, 2>, false>(p, stream);
    switch (tile) {
        case 0: return run_rows<E, MODE, RowsTile<2, 2, 2, 2>, true>(p, stream);
        case 1: return run_rows<E, MODE, RowsTile<4, 4, 2, 2>, true>(p, stream);
        case 2: return run_rows<E, MODE, RowsTile<8, 4, 2, 4>, true>(p, stream);
        case 3: return run_rows<E, MODE, RowsTile<4, 8, 4, 2>, true>(p, stream);
        case 4: return run_rows<E, MODE, RowsTile<4, 4, 4, 2, 3>, true>(p, stream);
        case 5: return run_rows<E, MODE, RowsTile<2, 2, 2, 2, 4>, true>(p, stream);
        case 6: return run_rows<E, MODE, RowsTile<4, 4, 2, 2, 3>, true>(p, stream);
    }
    if constexpr (MODE != kRowsWeight) {
        if (tile == 7) return run_rows<E, MODE, RowsTile<4, 5, 4, 2, 3>, true>(p, stream);
        if (tile == 8) return run_rows<E, MODE, RowsTile<4, 6, 4, 2>, true>(p, stream);
        if (tile == 9) return run_rows<E, MODE, RowsTile<4, 3, 4, 2, 3>, true>(p, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace
}  // namespace jjo
