// Products of float matrices on LDS tiles: see rows_mm.hpp for the four forms.
//
// out[Q][P] += Qmat[Q][K] . Pmat[P][K]^T.  A stage is 128 bytes of the sums' direction (64 elements of 16
// bits, 32 of 32) of every row of the tile's two operands, two steps of the matrix instruction.  Where
// a row's elements are contiguous, its 128 bytes are a row of LDS, 16-byte pieces permuted by the row
// (piece ^ row / 2 % 8); where the rows of an element are, an LDS row is one element of all the tile's
// rows, and the transposing LDS read puts four elements of a row into a lane; pieces are permuted by
// the element's number so that the lanes served together fall into different banks.
//
// What bounds it (bf16, us and Tflop/s): dense products the matrix cores with LDS behind them, 8192 cubed 816 to 845
// (1300 to 1347; a library product 700 to 840 with the card's clock, its input gradient 825, its weights' 960 to 990),
// 2047 x 14336 over 4096 197 to 210 (448 tiles are 1.75 rounds; the library 170 to 182), gradients of the weights
// 4096 x 4096 over 2048 60 (1150; the library 66).  Experts with few rows: reading their matrices (64 x 1408 x 2048,
// 25 rows each, 72 us, 5.3 TB/s on tiles of 64 x 64).  Short sums of large outputs: writing them (8 x 28672 x 4096
// over 256 tokens each 733: 1.9 GB, which a fill writes in 273; a tile's output, 128 KB a CU at 5.8 TB/s, and its
// stages do not overlap, see rows_stream_kernel).  Rows without 16-byte alignment: fp32 as with it, 512 x 4095 over 4095
// 148 us (134); 16 bits the caches, 45 us (28), see RowsWay.
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

// 16 bytes less their first n of eight elements, zeros behind them.
__device__ __forceinline__ u32x4v rows_shift(u32x4v v, int n) {
    if (n & 1) v = u32x4v{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    if (n & 2) v = u32x4v{v[1], v[2], v[3], 0u};
    if (n & 4) v = u32x4v{v[2], v[3], 0u, 0u};
    return v;
}

// One operand's part of a stage: ROWS rows of the tile, TRANS: the rows of an element contiguous.  A DMA instruction
// moves UNIT bytes a lane, a piece or a word of one.
template <class T, bool TRANS, int ROWS, int THREADS, int UNIT = 16>
struct RowsOperand {
    static constexpr int kPiece = 16 / sizeof(T), kStep = 128 / sizeof(T);
    static constexpr int kPitch = TRANS ? ROWS * (int)sizeof(T) : 128;  // bytes of an LDS row
    static constexpr int kRowPieces = kPitch / 16;
    static constexpr int kRuns = ROWS / 8, kWaves = THREADS / 64;  // of 64 pieces: a DMA instruction's
    static constexpr int kMine = (kRuns + kWaves - 1) / kWaves;    // of a wave
    static constexpr int kUnits = 16 / UNIT, kDmaMine = kMine * kUnits;
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

    // ---- through registers, a stage ahead, any alignment.  A piece that the rows' or the sums' end cuts is loaded
    // as the last whole one and shifted on its way to LDS; rows behind the last are any values, sums behind theirs
    // zeros.  `lead`: columns that the tile lacks of a piece, by which its first address is moved back (TRANS).
    static __device__ __forceinline__ void fetch(u32x4v (&v)[kMine], const T *from, const uint32_t (&off)[kMine]) {
#pragma unroll
        for (int n = 0; n < kMine; ++n) v[n] = load_any<u32x4v>((const uint8_t *)from + off[n]);
    }
    // ... `left` elements of a stage.
    template <class F>
    static __device__ __forceinline__ void fetch_last(u32x4v (&v)[kMine], int n, const T *from, int64_t ld, int left,
                                                      int wave, F row) {
        int i, k;
        piece(64 * run(wave, n) + (threadIdx.x & 63), i, k);
        v[n] = load_any<u32x4v>(from + (TRANS ? min(k, left - 1) * ld + row(i) : row(i) * ld + min(k, left - kPiece)));
    }
    static __device__ __forceinline__ void put(u32x4v (&v)[kMine], uint8_t *lds, int left, int rows, int wave) {
        const int in_run = threadIdx.x & 63;
        if (left < kStep || (TRANS && rows < ROWS && rows % kPiece != 0)) {
#pragma unroll
            for (int n = 0; n < kMine; ++n) {
                int i, k;
                piece(64 * run(wave, n) + in_run, i, k);
                const int cut = TRANS ? max(i - (rows - kPiece), 0) : max(k - (left - kPiece), 0);
                if (k >= left) v[n] = u32x4v{0u, 0u, 0u, 0u};
                else v[n] = rows_shift(v[n], cut);
            }
        }
#pragma unroll
        for (int n = 0; n < kMine; ++n) *reinterpret_cast<u32x4v *>(lds + 16 * (64 * run(wave, n) + in_run)) = v[n];
    }

    // ---- piece by piece: any address and size.  `from`(i, k, have) is the address of a piece, `have` the elements
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

    // ---- by DMA, 64 units an instruction: what the n-th one of a wave moves into this lane's unit, and where to.
    static __device__ __forceinline__ void dma_unit(int wave, int n, int in_run, int &i, int &k) {
        const int at = n % kUnits * 64 + in_run;
        piece(64 * run(wave, n / kUnits) + at / kUnits, i, k);
        (TRANS ? i : k) += at % kUnits;
    }
    static __device__ __forceinline__ uint32_t dma_to(int wave, int n) {
        return 1024 * run(wave, n / kUnits) + 64 * UNIT * (n % kUnits);
    }
    // A lane's offsets; rows behind the last are the last again.
    template <class F>
    static __device__ __forceinline__ void dma_offsets(uint32_t (&off)[kDmaMine], int wave, int64_t ld, F row) {
#pragma unroll
        for (int n = 0; n < kDmaMine; ++n) {
            int i, k;
            dma_unit(wave, n, threadIdx.x & 63, i, k);
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

// Workgroups go to the eight XCDs in turn.  Each XCD takes a contiguous run of the tiles, its workgroups
// neighbours of it, so that tiles that read the same rows are read into one L2; or (tiles of unequal length) the
// XCDs take turns at chunks of 32, an XCD's workgroups (gradients of 8 experts' 28672 x 4096 matrices, one
// expert a run: as long as the one with the most tokens, 444 of 2048, 1036 us, 800 to 880 in turn), first to last and
// last to first, as the experts with the most rows may come first.  A workgroup's places are at, at + step, ... below
// end.
struct RowsRun {
    int at, step, end, beg, xcd;
    bool chunked;
    __device__ __forceinline__ RowsRun(int total, bool unequal) {
        xcd = blockIdx.x % 8;
        at = blockIdx.x / 8;
        step = ((int)gridDim.x - xcd + 7) / 8;
        chunked = unequal && total >= 1024;
        if (chunked) {
            const int chunks = (total + 31) / 32, mine = chunks / 8 + (turn(chunks / 8) < chunks % 8);
            const bool last = turn((chunks - 1) / 8) == (chunks - 1) % 8;
            beg = 0, end = 32 * mine - (last ? 32 * chunks - total : 0);
        } else {
            const int per = total / 8, rest = total % 8;
            beg = xcd * per + min(xcd, rest), end = per + (xcd < rest);
        }
    }
    __device__ __forceinline__ int tile(int place) const {
        return chunked ? (place / 32 * 8 + turn(place / 32)) * 32 + place % 32 : beg + place;
    }
    __device__ __forceinline__ int turn(int round) const { return round % 2 == 0 ? xcd : 7 - xcd; }
};

// A tile of the output: columns p0.., rows q0.. (rows_q of them; of weight in half `half` of expert's matrix),
// its sums over stages s_beg..s_end of `length` elements from row `first` on (weight).
struct RowsPlace {
    int p0, q0, rows_q, expert, half, first, length, slice, s_beg, s_end;
    int turn;  // the stage behind which the sums are scaled (weight: the last of the first term), -1 for none
};

// The tiles of a launch, of Tile::kQ rows and kOutP columns.  Lane l of a wave holds the range of expert
// l's rows and its row tiles added to those before; of more than 64 experts they are read again for
// every tile.  Ranges are clamped to [0, M], so a malformed table drops rows instead of leaving the
// buffers.  All lanes of a wave call these together.
template <RowsMode MODE, class Tile, int STEP>
struct RowsTiles {
    static constexpr int kOutP = MODE == kRowsSwiglu ? Tile::kP / 2 : Tile::kP;
    int beg = 0, fin = 0, incl = 0;
    int per_slice;

    __device__ __forceinline__ void count(const RowsMm &p, int e0) {
        const int e = e0 + (threadIdx.x & 63);
        beg = fin = 0;
        if (e < p.n_experts) {
            beg = min(max(p.offsets[e], 0), p.M);
            fin = min(max(p.offsets[e + 1], beg), p.M);
        }
        incl = mx_scan((fin - beg + Tile::kQ - 1) / Tile::kQ);
    }
    // Weights' gradients: the experts with the most rows first, lane l the l-th of them.  Its number is in the three
    // bits above the 2^28 of each end, a register less.  Sorted where an expert has less than a tile for each CU, whose
    // sums differ then (64 experts' 2048 x 1408, 3 to 730 rows each, rows' gradients included, 342 us, 371 unsorted);
    // CUs that work on one expert at a time are even, and experts of few rows, bound by their outputs, are better
    // spread (8 of 28672 x 4096, 256 rows on average: 1540 to 1570 sorted, 1524 not).
    __device__ __forceinline__ void sort(bool by_rows) {
        const int rows = fin - beg;
        const uint32_t lane = threadIdx.x & 63;
        int at = by_rows ? 0 : lane;
#pragma unroll 8
        for (int j = 0; by_rows && j < 64; ++j) {
            const int other = __builtin_amdgcn_readlane(rows, j);
            at += other > rows || (other == rows && j < (int)lane);
        }
        beg = __builtin_amdgcn_ds_permute(4 * at, beg | lane << 29);
        fin = __builtin_amdgcn_ds_permute(4 * at, fin | lane >> 3 << 29);
    }
    // The tiles in all; `most`: those the launch was made for (more only by a malformed table: none then).
    __device__ __forceinline__ int total(const RowsMm &p, int64_t most) {
        int64_t tiles = (int64_t)p.tiles_p * p.tiles_q;
        if (p.offsets != nullptr) {
            int rows = 0;
            for (int e0 = 0; e0 < p.n_experts; e0 += 64) {
                count(p, e0);
                rows += __builtin_amdgcn_readlane(incl, 63);
            }
            if (MODE == kRowsWeight && p.n_experts <= 64) sort(tiles < 256);
            tiles = MODE == kRowsWeight ? tiles * p.n_experts : (int64_t)p.tiles_p * rows;
        }
        per_slice = tiles * p.slices > most || tiles < 0 ? 0 : (int)tiles;
        return per_slice * p.slices;
    }
    // The order of an output's tiles: eight rows of tiles at a time, these fastest, so that the 32 that an XCD
    // works on at once read few rows of either operand (gradients of 8 experts' 28672 x 4096 matrices, 256 tokens
    // each: 795 us, 990 with all row tiles fastest; 8192 cubed 853 and 943).
    static __device__ __forceinline__ void blocked(int tile, int tiles_q, int tiles_p, int &tile_q, int &tile_p) {
        const int group = tile / (8 * tiles_p), rows = min(tiles_q - 8 * group, 8), at = tile - group * 8 * tiles_p;
        tile_q = 8 * group + at % rows;
        tile_p = at / rows;
    }
    __device__ __forceinline__ RowsPlace place(const RowsMm &p, int id) {
        RowsPlace c{};
        c.slice = p.slices == 1 ? 0 : id / per_slice;
        int tile = id - c.slice * per_slice, tile_p;
        c.length = p.K;
        if constexpr (MODE == kRowsWeight) {
            const int each = p.tiles_p * p.tiles_q;
            if (p.offsets != nullptr) {
                c.expert = tile / each, tile %= each;
                int end;
                if (p.n_experts <= 64) {
                    const uint32_t a = __builtin_amdgcn_readlane(beg, c.expert);
                    const uint32_t b = __builtin_amdgcn_readlane(fin, c.expert);
                    c.expert = a >> 29 | b >> 29 << 3;
                    c.first = a & 0x1fffffff, end = b & 0x1fffffff;
                } else {
                    c.first = __builtin_amdgcn_readfirstlane(min(max(p.offsets[c.expert], 0), p.M));
                    end = __builtin_amdgcn_readfirstlane(min(max(p.offsets[c.expert + 1], c.first), p.M));
                }
                c.length = end - c.first;
            }
            int tile_q;
            blocked(tile, p.tiles_q, p.tiles_p, tile_q, tile_p);
            const int tiles_half = p.tiles_q / p.halves;
            c.half = tile_q / tiles_half;
            c.q0 = tile_q % tiles_half * Tile::kQ;
            c.rows_q = min(p.Q - c.q0, Tile::kQ);
        } else if (p.offsets == nullptr) {
            int tile_q;
            blocked(tile, p.tiles_q, p.tiles_p, tile_q, tile_p);
            c.q0 = tile_q * Tile::kQ;
            c.rows_q = min(p.Q - c.q0, Tile::kQ);
        } else {  // expert by expert
            int base = 0, tiles = 1, row = 0, end = 0;
            tile_p = 0;
            for (int e0 = 0; e0 < p.n_experts; e0 += 64) {
                if (p.n_experts > 64) count(p, e0);
                const uint64_t past = __ballot((int64_t)(base + incl) * p.tiles_p > tile);
                if (past != 0) {
                    const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
                    row = __builtin_amdgcn_readlane(beg, l);
                    end = __builtin_amdgcn_readlane(fin, l);
                    tiles = max((end - row + Tile::kQ - 1) / Tile::kQ, 1);
                    const int local = tile - (base + __builtin_amdgcn_readlane(incl, l) - tiles) * p.tiles_p;
                    c.expert = e0 + l;
                    int tile_q;
                    blocked(local, tiles, p.tiles_p, tile_q, tile_p);
                    row += tile_q * Tile::kQ;
                    break;
                }
                base += __builtin_amdgcn_readlane(incl, 63);
            }
            c.q0 = row;
            c.rows_q = min(end - row, Tile::kQ);
        }
        c.p0 = tile_p * kOutP;
        const int half_stages = (c.length + STEP - 1) / STEP;
        const int stages = half_stages * (MODE == kRowsInput ? p.halves : MODE == kRowsWeight ? p.terms : 1);
        c.s_beg = p.slices == 1 ? 0 : (int)((int64_t)stages * c.slice / p.slices);
        c.s_end = p.slices == 1 ? stages : (int)((int64_t)stages * (c.slice + 1) / p.slices);
        if (c.s_beg == c.s_end) c.s_beg = c.s_end = stages;  // a slice without stages: behind the sums' end
        c.turn = MODE == kRowsWeight && p.terms == 2 && c.s_beg < half_stages ? min(half_stages, c.s_end) - 1 : -1;
        return c;
    }
};

// Four of them, to places 1 KB apart.  What a stage's requests cost a wave in instructions is a slot of
// rows_stream_kernel that is longer than the other's products: 8192 cubed 849 us for 861 to 874 with the addresses
// computed anew for each, gradients of the weights and rows 820 and 842 for 890.
__device__ __forceinline__ void rows_dma4(const uint32_t *off, uint64_t from, uint32_t lds) {
    uint32_t m0v = __builtin_amdgcn_readfirstlane(lds);
    from = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(from >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)from);
    asm volatile(
        "s_nop 4\n\t"
        "global_load_lds_dwordx4 %1, %5\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %2, %5\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %5\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %4, %5"
        : "+{m0}"(m0v)
        : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(from)
        : "memory", "scc");
}

// ... of words, to places 256 bytes apart.
__device__ __forceinline__ void rows_dma4_words(const uint32_t *off, uint64_t from, uint32_t lds) {
    uint32_t m0v = __builtin_amdgcn_readfirstlane(lds);
    from = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(from >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)from);
    asm volatile(
        "s_nop 4\n\t"
        "global_load_lds_dword %1, %5\n\t"
        "s_add_u32 m0, m0, 0x100\n\ts_nop 0\n\t"
        "global_load_lds_dword %2, %5\n\t"
        "s_add_u32 m0, m0, 0x100\n\ts_nop 0\n\t"
        "global_load_lds_dword %3, %5\n\t"
        "s_add_u32 m0, m0, 0x100\n\ts_nop 0\n\t"
        "global_load_lds_dword %4, %5"
        : "+{m0}"(m0v)
        : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(from)
        : "memory", "scc");
}

// One unit a lane from an address of each lane's own.
template <int UNIT>
__device__ __forceinline__ void rows_dma(const void *from, uint32_t lds) {
    const uint32_t m0v = __builtin_amdgcn_readfirstlane(lds);
    if constexpr (UNIT == 16)
        asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "{m0}"(m0v) : "memory");
    else
        asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, off" : : "v"(from), "{m0}"(m0v) : "memory");
}

__device__ const __align__(16) uint32_t rows_zeros[4] = {0u, 0u, 0u, 0u};  // the pieces behind the sums' end

// The operands of a tile and the way of their stages into LDS.
//
// DMA: the operands' memory rows are 16-byte aligned, the sums' elements whole pieces, and a tile's offsets
// fit 32 bits.  Where they are not aligned: fp32 by DMA of words.  16 bits staged, sizes of a piece at least: a stage
// is loaded to registers some stages ahead, and written to LDS behind the products of the one before.  Copied:
// anything else, a stage at a time.
enum RowsWay { kRowsDma, kRowsWords, kRowsStaged, kRowsCopied };
template <class T, RowsMode MODE, class Tile, RowsWay WAY>
struct RowsSource {
    static constexpr bool DMA = WAY == kRowsDma || WAY == kRowsWords;
    static constexpr int kUnit = WAY == kRowsWords ? 4 : 16;
    static_assert(WAY == kRowsWords ? sizeof(T) == 4 : WAY != kRowsStaged || sizeof(T) == 2, "the ways");
    static constexpr int kStep = 128 / sizeof(T);
    static constexpr bool PT = MODE == kRowsInput || MODE == kRowsWeight, QT = MODE == kRowsWeight;
    using OpP = RowsOperand<T, PT, Tile::kP, Tile::kThreads, kUnit>;
    using OpQ = RowsOperand<T, QT, Tile::kQ, Tile::kThreads, kUnit>;
    static constexpr int kDma = OpP::kDmaMine + OpQ::kDmaMine;  // of a wave and stage

    // From the tile's first row and the sums' first element on; the second ones: up's rows (SwiGLU), the sums'
    // second half (input), and q's other terms (weight).
    const T *pm, *pm2, *qm, *qm2;
    int rows_p, rows_q, length, stages_half, lead_p, lead_q;
    static constexpr bool kOffsets = WAY != kRowsCopied;
    uint32_t off_p[kOffsets ? OpP::kDmaMine : 1], off_q[kOffsets ? OpQ::kDmaMine : 1];

    // Row i of the P operand's part of a stage: of SwiGLU a wave's first 8 * RT are gate's, the others up's.
    static __device__ __forceinline__ bool is_up(int i) {
        return MODE == kRowsSwiglu && i % (16 * Tile::RT) >= 8 * Tile::RT;
    }
    static __device__ __forceinline__ int row_p(int i) {
        return MODE == kRowsSwiglu ? i / (16 * Tile::RT) * (8 * Tile::RT) + i % (8 * Tile::RT) : i;
    }

    __device__ __forceinline__ void open(const RowsMm &p, const RowsPlace &c, int wave) {
        rows_p = min(p.P - c.p0, MODE == kRowsSwiglu ? Tile::kP / 2 : Tile::kP);
        rows_q = c.rows_q, length = c.length;
        stages_half = (length + kStep - 1) / kStep;
        lead_p = PT && WAY == kRowsStaged ? max(OpP::kPiece - rows_p, 0) : 0;
        lead_q = QT && WAY == kRowsStaged ? max(OpQ::kPiece - rows_q, 0) : 0;
        const int64_t at_p = MODE == kRowsWeight ? c.first * p.ldp + c.p0 - lead_p
                                                 : c.expert * p.expert_stride + (PT ? c.p0 - lead_p : c.p0 * p.ldp);
        const int64_t at_q = QT ? c.first * p.ldq + (int64_t)c.half * p.Q + c.q0 - lead_q : c.q0 * p.ldq;
        pm = (const T *)p.p + at_p, pm2 = MODE == kRowsWeight ? pm : (const T *)p.p2 + at_p;
        qm = (const T *)p.q + at_q, qm2 = MODE == kRowsWeight ? (const T *)p.rest + at_q : qm;
        if constexpr (kOffsets) {
            OpP::dma_offsets(off_p, wave, p.ldp, [&](int i) { return from_row_p(i); });
            OpQ::dma_offsets(off_q, wave, p.ldq, [&](int i) { return from_row_q(i); });
        }
    }
    // The memory row (TRANS: column) that row i is loaded from.
    static constexpr int kUnitElements = kUnit / sizeof(T);
    __device__ __forceinline__ int from_row_p(int i) const {
        return PT ? min(i, rows_p - kUnitElements) + lead_p : min(row_p(i), rows_p - 1);
    }
    __device__ __forceinline__ int from_row_q(int i) const {
        return QT ? min(i, rows_q - kUnitElements) + lead_q : min(i, rows_q - 1);
    }

    // ---- whole stages one after the other: aim at stage st (of those below end), then `whole` of them.
    uint64_t at_p, at_q;
    int whole;
    __device__ __forceinline__ void aim(const RowsMm &p, int st, int end, int wave) {
        const int parts = MODE == kRowsInput ? p.halves : MODE == kRowsWeight ? p.terms : 1;
        const int part = min((st >= stages_half) + (st >= 2 * stages_half), parts - 1);
        const int k0 = (st - part * stages_half) * kStep;
        // Of SwiGLU a wave's runs are all of one matrix.
        static_assert(MODE != kRowsSwiglu || Tile::kWaves != 8 || OpP::kMine * 8 == 8 * Tile::RT, "32 rows a wave");
        at_p = (uint64_t)((part > 0 || is_up(8 * OpP::run(wave, 0)) ? pm2 : pm) + (PT ? k0 * p.ldp : k0));
        at_q = (uint64_t)((MODE == kRowsWeight && part > 0 ? qm2 + (part - 1) * p.rest_plane : qm) +
                          (QT ? k0 * p.ldq : (part > 0 ? p.K : 0) + (int64_t)k0));
        whole = min(max(length - k0, 0) / kStep, end - st);
    }
    __device__ __forceinline__ void bring_whole_p(const RowsMm &p, uint8_t *to, int wave) {
        const uint32_t at = (uint32_t)(uintptr_t)to;
        if constexpr (OpP::kMine == 4) {
            rows_dma4(off_p, at_p, at + 1024 * OpP::run(wave, 0));
        } else {
#pragma unroll
            for (int n = 0; n < OpP::kMine; ++n) rows_dma(off_p[n], at_p, at + 1024 * OpP::run(wave, n));
        }
        at_p += PT ? 128 * p.ldp : 128;
        --whole;
    }
    __device__ __forceinline__ void bring_whole_q(const RowsMm &p, uint8_t *to, int wave) {
        const uint32_t at = (uint32_t)(uintptr_t)to;
        if constexpr (OpQ::kMine == 4 && OpQ::kRuns % OpQ::kWaves == 0) {
            rows_dma4(off_q, at_q, at + Tile::kStageP + 1024 * OpQ::run(wave, 0));
        } else {
#pragma unroll
            for (int n = 0; n < OpQ::kMine; ++n)
                rows_dma(off_q[n], at_q, at + Tile::kStageP + 1024 * OpQ::run(wave, n));
        }
        at_q += QT ? 128 * p.ldq : 128;
    }

    // Where stage st begins, and how many of the sums' elements are left there.
    struct Stage {
        const T *from_p, *from_up, *from_q;
        int left;
    };
    __device__ __forceinline__ Stage stage(const RowsMm &p, int st) const {
        // The half or term of the sums that stage st belongs to: the last one's, past its end, behind them.
        const int parts = MODE == kRowsInput ? p.halves : MODE == kRowsWeight ? p.terms : 1;
        const int part = min((st >= stages_half) + (st >= 2 * stages_half), parts - 1);
        const bool second = part > 0;
        const int k0 = (st - part * stages_half) * kStep;
        Stage s;
        s.left = length - k0;
        s.from_p = (second ? pm2 : pm) + (PT ? k0 * p.ldp : k0);
        s.from_up = MODE == kRowsSwiglu ? pm2 + k0 : s.from_p;
        s.from_q = (MODE == kRowsWeight && second ? qm2 + (part - 1) * p.rest_plane : qm) +
                   (QT ? k0 * p.ldq : (second ? p.K : 0) + (int64_t)k0);
        return s;
    }

    // ---- through registers: stage st (one with elements) to these, and these to LDS.
    struct Held {
        u32x4v in_p[OpP::kMine], in_q[OpQ::kMine];
    };
    __device__ __forceinline__ void fetch(Held &h, const RowsMm &p, int st, int wave) const {
        auto &in_p = h.in_p;
        auto &in_q = h.in_q;
        const Stage s = stage(p, st);
        if (s.left >= kStep) {
            if constexpr (MODE == kRowsSwiglu) {
#pragma unroll
                for (int n = 0; n < OpP::kMine; ++n) {
                    const T *const from = is_up(8 * OpP::run(wave, n)) ? s.from_up : s.from_p;
                    in_p[n] = load_any<u32x4v>((const uint8_t *)from + off_p[n]);
                }
            } else {
                OpP::fetch(in_p, s.from_p, off_p);
            }
            OpQ::fetch(in_q, s.from_q, off_q);
        } else {
#pragma unroll
            for (int n = 0; n < OpP::kMine; ++n)
                OpP::fetch_last(in_p, n, is_up(8 * OpP::run(wave, n)) ? s.from_up : s.from_p, p.ldp, s.left, wave,
                                [&](int i) { return from_row_p(i); });
#pragma unroll
            for (int n = 0; n < OpQ::kMine; ++n)
                OpQ::fetch_last(in_q, n, s.from_q, p.ldq, s.left, wave, [&](int i) { return from_row_q(i); });
        }
    }
    __device__ __forceinline__ void put(Held &h, const RowsMm &p, int st, uint8_t *to, int wave) const {
        const int left = stage(p, st).left;
        OpP::put(h.in_p, to, left, rows_p, wave);
        OpQ::put(h.in_q, to + Tile::kStageP, left, rows_q, wave);
    }

    // ---- by DMA, or piece by piece: stage st to `to`; a stage without elements is zeros.
    __device__ __forceinline__ void bring(const RowsMm &p, int st, uint8_t *to, int wave) const {
        const Stage s = stage(p, st);
        const T *const from_p = s.from_p, *const from_up = s.from_up, *const from_q = s.from_q;
        const int left = s.left;
        if constexpr (DMA) {
            const uint32_t at = (uint32_t)(uintptr_t)to;
            // The matrix of a wave's n-th instruction: of SwiGLU a run is 8 rows of one.
            auto base_p = [&](int n) { return is_up(8 * OpP::run(wave, n / OpP::kUnits)) ? from_up : from_p; };
            if (left >= kStep) {
                if constexpr (WAY == kRowsWords) {
#pragma unroll
                    for (int n = 0; n < OpP::kDmaMine; n += 4)
                        rows_dma4_words(off_p + n, (uint64_t)base_p(n), at + OpP::dma_to(wave, n));
#pragma unroll
                    for (int n = 0; n < OpQ::kDmaMine; n += 4)
                        rows_dma4_words(off_q + n, (uint64_t)from_q, at + Tile::kStageP + OpQ::dma_to(wave, n));
                } else {
#pragma unroll
                    for (int n = 0; n < OpP::kDmaMine; ++n)
                        rows_dma(off_p[n], (uint64_t)base_p(n), at + OpP::dma_to(wave, n));
#pragma unroll
                    for (int n = 0; n < OpQ::kDmaMine; ++n)
                        rows_dma(off_q[n], (uint64_t)from_q, at + Tile::kStageP + OpQ::dma_to(wave, n));
                }
            } else {  // the sums end inside the stage
                int in_run = threadIdx.x & 63;
                asm volatile("" : "+v"(in_run));  // one stage of many: nothing kept in registers for it
#pragma unroll
                for (int n = 0; n < OpP::kDmaMine; ++n) {
                    int i, k;
                    OpP::dma_unit(wave, n, in_run, i, k);
                    rows_dma<kUnit>(k < left ? (const void *)(base_p(n) + off_p[n] / sizeof(T)) : rows_zeros,
                                    at + OpP::dma_to(wave, n));
                }
#pragma unroll
                for (int n = 0; n < OpQ::kDmaMine; ++n) {
                    int i, k;
                    OpQ::dma_unit(wave, n, in_run, i, k);
                    rows_dma<kUnit>(k < left ? (const void *)(from_q + off_q[n] / sizeof(T)) : rows_zeros,
                                    at + Tile::kStageP + OpQ::dma_to(wave, n));
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
    }
};

// A tile's sums to the output, straight from the registers: of two tiles side by side lanes exchange halves, so
// that each holds eight columns of a row and a row's four lanes 64 contiguous bytes (of 16 bits).
//
// The code of every epilogue unrolled over a wave's sums would be 150 KB, more than the instruction cache, and
// cost a tile of 256 x 256 some 8 us.  So plain outputs (whole groups of eight columns) have a path of
// their own.  kRowsFull has one for each activation, for whole groups too; kRowsAny takes one row of tiles at a time,
// in a loop that moves the next one's sums into the same registers (which costs registers that the large tiles do not
// have).  Of weights' gradients kRowsPlain has rows at multiples of 64 bytes, kRowsFull others.
enum RowsOutput { kRowsPlain, kRowsFull, kRowsAny };

// 16 bytes of a row, values col.. of P, through the caches.
template <class Out>
__device__ __forceinline__ void rows_store_line(Out *to, u32x4v v, int col, int P) {
    constexpr int kN = 16 / sizeof(Out);
    const MxVec<Out, kN> e = __builtin_bit_cast(MxVec<Out, kN>, v);
    if (col + kN <= P) return store_any(to, v);
#pragma unroll
    for (int i = 0; i < kN - 1; ++i)
        if (col + i < P) to[i] = e.v[i];
}
// The same of 16 bits where some rows are at odd places, those in whole words from the second value on: `next` holds the
// first of the lane with the columns behind, which lanes 56 and up have not.
template <class Out>
__device__ __forceinline__ void rows_store_words(Out *to, u32x4v v, uint32_t next, int col, int P) {
    if ((uintptr_t)to % 4 == 0 || col + 8 > P) return rows_store_line(to, v, col, P);
    typedef uint32_t Words3 __attribute__((ext_vector_type(3), aligned(4)));
    typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(4)));
    const int lane = threadIdx.x & 63;
    const MxVec<Out, 8> e = __builtin_bit_cast(MxVec<Out, 8>, v);
    const uint32_t w[4] = {v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16,
                           v[3] >> 16 | next << 16};
    if (lane < 56 && col + 8 < P) {
        *(Words4 *)(to + 1) = Words4{w[0], w[1], w[2], w[3]};
    } else {
        *(Words3 *)(to + 1) = Words3{w[0], w[1], w[2]};
        to[7] = e.v[7];
    }
    if (lane < 8) to[0] = e.v[0];
}

template <class T, RowsMode MODE, RowsOutput KIND, class Tile>
__device__ __forceinline__ void rows_output(const RowsMm &p, const RowsPlace &c, f32x4v (&acc)[Tile::RT][Tile::TT],
                                            int wp, int wq) {
    constexpr int RT = Tile::RT, TT = Tile::TT;
    constexpr int kWaveP = MODE == kRowsSwiglu ? 8 * RT : 16 * RT;  // columns of a wave
    // Pairs of tiles side by side, or (the small tile's gate and up) of two rows of tiles.
    constexpr bool kBeside = kWaveP % 32 == 0;
    static_assert(kBeside || (TT % 2 == 0 && RT == 2 && MODE == kRowsSwiglu), "pairs of tiles");
    constexpr int kRows = kBeside ? 1 : 2, kPairs = kBeside ? kWaveP / 32 : 1;
    const int lane = threadIdx.x & 63, r16 = lane & 15, odd = (lane >> 4) & 1, upper = lane >> 5;
    const bool parts = p.slices > 1, wide = MODE == kRowsWeight && p.wide, to32 = parts || wide;
    // The output's (or the slice's sums') matrix, and its rows' length.
    const int64_t cols = MODE == kRowsSwiglu ? 2 * (int64_t)p.P : p.P, matrices = max(p.n_experts, 1);
    int64_t ld = p.ldy;
    uint8_t *y;
    if (parts) {
        ld = cols;
        const int64_t all = MODE == kRowsWeight ? p.Q * p.halves * matrices : p.Q;
        const int64_t mine = MODE == kRowsWeight ? (c.half * matrices + c.expert) * p.Q : 0;
        y = (uint8_t *)(p.part + (c.slice * all + mine) * cols);
    } else {
        y = (uint8_t *)(MODE == kRowsWeight && c.half != 0 ? p.y2 : p.y);
        if constexpr (MODE == kRowsWeight) y += c.expert * p.expert_stride * (wide ? 4 : sizeof(T));
    }
    // Row and column of the lane's eight of pair `pair` in row tt of tiles.
    auto row_of = [&](int tt) { return 16 * (TT * wq + tt + (kBeside ? 0 : odd)) + r16; };
    auto col_of = [&](int pair) { return c.p0 + kWaveP * wp + (kBeside ? 32 * pair + 16 * odd : 0) + 8 * upper; };
    auto take = [&](int tt, int pair, float *v, float *up) {
        if constexpr (kBeside) {
            rows_exchange(acc[2 * pair][tt], acc[2 * pair + 1][tt], v);
            if constexpr (MODE == kRowsSwiglu)
                rows_exchange(acc[RT / 2 + 2 * pair][tt], acc[RT / 2 + 2 * pair + 1][tt], up);
        } else {
            rows_exchange(acc[0][tt], acc[0][tt + 1], v);
            rows_exchange(acc[1][tt], acc[1][tt + 1], up);
        }
    };
    const RowsEpilogue &e = p.epi;
    if constexpr (KIND == kRowsFull && MODE == kRowsForward) {
        auto all = [&](auto act) {
#pragma unroll
            for (int pair = 0; pair < kPairs; ++pair) {
                const int col = col_of(pair);
                float bias[8];
                rows_load8((const T *)e.bias + col, e.bias != nullptr && col < p.P ? 8 : 0, bias);
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    float v[8];
                    take(tt, pair, v, v);
                    const int in_tile = row_of(tt);
                    if (in_tile < c.rows_q && col < p.P) {
                        const int64_t row = c.q0 + in_tile;
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] += bias[i];
                        if (e.pre != nullptr) rows_store8((T *)e.pre + row * p.P + col, 8, v);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = rows_act<T>(v[i], decltype(act)::value);
                        if (e.residual != nullptr) {
                            float r[8];
                            rows_load8((const T *)e.residual + row * e.residual_stride + col, 8, r);
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[i] += r[i];
                        }
                        rows_store8((T *)y + row * ld + col, 8, v);
                    }
                }
            }
        };
        switch (e.act) {
            case JJO_ACT_RELU: return all(std::integral_constant<int, JJO_ACT_RELU>{});
            case JJO_ACT_GELU: return all(std::integral_constant<int, JJO_ACT_GELU>{});
            case JJO_ACT_GELU_TANH: return all(std::integral_constant<int, JJO_ACT_GELU_TANH>{});
            case JJO_ACT_SILU: return all(std::integral_constant<int, JJO_ACT_SILU>{});
        }
        return all(std::integral_constant<int, JJO_ACT_NONE>{});
    }
    // Weights' gradients go past the caches, in whole lines: nothing near reads them, and they would push out what
    // the tiles beside read (64 experts of 2048 x 1408, 244 tokens each: 160 us, 195 through the caches).  Stores of 64
    // bytes a row reach 3.0 to 4.0 TB/s that way, of 128 bytes 5.6 to 6.3, as through the caches.  So lanes 8..15 of
    // each 16 exchange with 0..7: an instruction writes 128 bytes of eight rows.  Rows that do not begin at multiples
    // of 64 bytes go through the caches, which join the lines that two stores share (64 experts of 2048 x 1408 with 25
    // rows each, 4 bytes beside: 128 us, past the caches 188; at a multiple 110).  Rows of 16 bits at odd places are
    // written in whole words but for their ends, each lane taking the next one's first value (2 bytes beside: 172 us,
    // 217 otherwise).
    if constexpr (MODE == kRowsWeight && RT == 4) {
        const bool high = (lane & 8) != 0;
        auto all = [&](auto past_tag) {
            constexpr bool PAST = decltype(past_tag)::value;
            auto lines = [&](u32x4v a, u32x4v b, int tt, int col, auto out) {
                using Out = decltype(out);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t mine = high ? a[i] : b[i];
                    const uint32_t x = __builtin_amdgcn_update_dpp(0, mine, 0x128, 0xf, 0xf, false);  // row_ror:8
                    a[i] = high ? x : a[i], b[i] = high ? b[i] : x;
                }
                const int in_tile = 16 * (TT * wq + tt) + (r16 & 7);
                Out *const to = (Out *)y + (c.q0 + in_tile) * ld + col;
                if constexpr (PAST) {
                    if (col >= p.P) return;
                    if (in_tile < c.rows_q) rows_store_past(to, a);
                    if (in_tile + 8 < c.rows_q) rows_store_past(to + 8 * ld, b);
                } else {
                    if constexpr (sizeof(Out) == 2) {
                        if (((uintptr_t)y | (uint64_t)ld * 2) % 4 != 0) {
                            // The next eight columns are those of the lane + 32, then + 16, then + 8.
                            const int next = 4 * (upper == 0 ? lane ^ 32 : odd == 0 ? lane ^ 48 : lane ^ 56);
                            const uint32_t next_a = __builtin_amdgcn_ds_bpermute(next, a[0]);
                            const uint32_t next_b = __builtin_amdgcn_ds_bpermute(next, b[0]);
                            if (in_tile < c.rows_q) rows_store_words(to, a, next_a, col, p.P);
                            if (in_tile + 8 < c.rows_q) rows_store_words(to + 8 * ld, b, next_b, col, p.P);
                            return;
                        }
                    }
                    if (in_tile < c.rows_q) rows_store_line(to, a, col, p.P);
                    if (in_tile + 8 < c.rows_q) rows_store_line(to + 8 * ld, b, col, p.P);
                }
            };
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                if (sizeof(T) == 4 || to32) {
#pragma unroll
                    for (int rt = 0; rt < RT; rt += 2)
                        lines(__builtin_bit_cast(u32x4v, acc[rt][tt]), __builtin_bit_cast(u32x4v, acc[rt + 1][tt]), tt,
                              c.p0 + kWaveP * wp + 16 * (rt + high) + 4 * (lane >> 4), 0.0f);
                } else if constexpr (sizeof(T) == 2) {
                    float v[8], w[8];
                    take(tt, 0, v, v);
                    take(tt, 1, w, w);
                    lines(rows_pack8<T>(v), rows_pack8<T>(w), tt, col_of(high), (T)0.0f);
                }
            }
        };
        if (KIND == kRowsPlain) return all(std::true_type{});
        if (KIND == kRowsFull) return all(std::false_type{});
        if (((uintptr_t)y | (uint64_t)ld * (to32 ? 4 : sizeof(T))) % 64 == 0) return all(std::true_type{});
        return all(std::false_type{});
    }
    const bool bare = e.bias == nullptr && e.residual == nullptr && e.pre == nullptr && e.act == JJO_ACT_NONE;
    if (KIND != kRowsAny || (p.P % 8 == 0 && (parts || bare))) {
        auto all = [&](auto wide_tag) {
            constexpr bool WIDE = decltype(wide_tag)::value;
            using Out = std::conditional_t<WIDE, float, T>;
#pragma unroll
            for (int tt = 0; tt < TT; tt += kRows)
#pragma unroll
                for (int pair = 0; pair < kPairs; ++pair) {
                    float v[8], up[8];
                    take(tt, pair, v, up);
                    const int in_tile = row_of(tt), col = col_of(pair);
                    if (in_tile < c.rows_q && col < p.P) {
                        Out *const to = (Out *)y + (c.q0 + in_tile) * ld + col;
                        if constexpr (MODE == kRowsSwiglu && WIDE) {
                            rows_store8(to, 8, v);
                            rows_store8(to + p.P, 8, up);
                        } else {
                            if constexpr (MODE == kRowsSwiglu) {
                                if (KIND == kRowsFull) {
                                    T *const pre = (T *)e.pre + (int64_t)(c.q0 + in_tile) * 2 * p.P + col;
                                    rows_store8(pre, 8, v);
                                    rows_store8(pre + p.P, 8, up);
                                }
                                rows_swiglu(v, up);
                            }
                            rows_store8(to, 8, v);
                        }
                    }
                }
        };
        if (to32) all(std::true_type{});
        else all(std::false_type{});
        return;
    }
    if constexpr (KIND == kRowsAny)
#pragma unroll 1
    for (int tt = 0; tt < TT; tt += kRows) {
#pragma unroll
        for (int pair = 0; pair < kPairs; ++pair) {
            float v[8], up[8];
            take(0, pair, v, up);
            const int in_tile = row_of(tt), col = col_of(pair), n = min(8, p.P - col);
            const int64_t row = c.q0 + in_tile;
            if (in_tile < c.rows_q && n > 0) {
                if (parts) {
                    rows_store8((float *)y + row * ld + col, n, v);
                    if constexpr (MODE == kRowsSwiglu) rows_store8((float *)y + row * ld + p.P + col, n, up);
                } else if constexpr (MODE == kRowsSwiglu) {
                    rows_finish_swiglu<T>(e, v, up, row, col, n, p.P, y);
                } else {
                    rows_finish<T>(e, v, row, col, n, p.P, y, ld, wide);
                }
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t + kRows < TT; ++t) acc[rt][t] = acc[rt][t + kRows];
    }
}

// Behind stage st, the last one of fp16's first term: the scale that its values were kept with leaves the sums.
template <class T, RowsMode MODE, class Tile>
__device__ __forceinline__ void rows_turn(const RowsMm &p, const RowsPlace &c, int st,
                                          f32x4v (&acc)[Tile::RT][Tile::TT]) {
    if constexpr (MODE == kRowsWeight && std::is_same_v<T, _Float16>) {
        if (st == c.turn)
#pragma unroll
            for (int rt = 0; rt < Tile::RT; ++rt)
#pragma unroll
                for (int tt = 0; tt < Tile::TT; ++tt) acc[rt][tt] *= p.first_scale;
    }
}

// ---- four waves, a tile a workgroup, two or more workgroups a CU: one stages while another multiplies.
// Stages that the staged way holds in registers.  bf16, odd K and N, us: tiles of 64, 64 x 4095 over 4095 with one
// 18.0, with three 15.9 (of four waves their loads are most of what a CU waits for); tiles of 128, 2047 rows, forward
// 98 with one and 109 with two, rows' gradients 128 and 123, weights' 136 and 136.
template <RowsMode MODE, int RT>
constexpr int kRowsHeld = RT == 2 ? 3 : MODE == kRowsInput ? 2 : 1;
template <class E, RowsMode MODE, class Tile, RowsWay WAY>
__global__ __launch_bounds__(Tile::kThreads) void rows_mm_kernel(RowsMm p, int most) {
    typedef typename E::type T;
    constexpr int RT = Tile::RT, TT = Tile::TT;
    using Source = RowsSource<T, MODE, Tile, WAY>;
    extern __shared__ __align__(16) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % Tile::WP, wq = wave / Tile::WP;
    RowsTiles<MODE, Tile, Source::kStep> tiles;
    const RowsRun run(tiles.total(p, most), MODE == kRowsWeight);
    if (run.at >= run.end) return;
    const RowsPlace c = tiles.place(p, run.tile(run.at));
    Source source;
    source.open(p, c, wave);

    f32x4v acc[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = f32x4v{0.f, 0.f, 0.f, 0.f};
    const typename Source::OpP::Reader read_p(16 * RT * wp);
    const typename Source::OpQ::Reader read_q(16 * TT * wq);
    auto step = [&](auto u_tag, const uint8_t *in_p) {
        constexpr int U = decltype(u_tag)::value;
        const uint8_t *const in_q = in_p + Tile::kStageP;
        u32x4v a[RT], b[TT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) a[rt] = read_p.template read<U>(in_p, rt);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) b[tt] = read_q.template read<U>(in_q, tt);
        if constexpr (sizeof(T) == 4) {  // in turn: the next sum of a tile does not wait for its last
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                            __uint_as_float(a[rt][j]), __uint_as_float(b[tt][j]), acc[rt][tt], 0, 0, 0);
        } else {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt][tt] = rows_mfma<T>(a[rt], b[tt], acc[rt][tt]);
        }
    };
    auto multiply = [&](int st, const uint8_t *in) {
        step(std::integral_constant<int, 0>{}, in);
        step(std::integral_constant<int, 1>{}, in);
        rows_turn<T, MODE, Tile>(p, c, st, acc);
    };
    if constexpr (WAY == kRowsStaged) {
        static_assert(Tile::NB == 2, "the buffer of the stage before is the next one's");
        // kAhead stages on their way to registers while one is multiplied.  Behind the last stage it is loaded again:
        // every wait then counts the same loads behind those that it is for.
        constexpr int kAhead = kRowsHeld<MODE, RT>;
        auto all = [&]() {
            typename Source::Held held[kAhead];
            const int last = c.s_end - 1;
            int st = c.s_beg;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) source.fetch(held[i], p, min(st + i, last), wave);
            uint8_t *in = lds, *next = lds + Tile::kStage;
            source.put(held[0], p, st, in, wave);
            for (;;) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    source.fetch(held[i], p, min(st + kAhead, last), wave);
                    // Stage st is in LDS, and no wave reads the buffer of stage st - 1 any more.
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    multiply(st, in);
                    if (++st > last) return;
                    source.put(held[(i + 1) % kAhead], p, st, next, wave);
                    uint8_t *const was = in;
                    in = next, next = was;
                }
            }
        };
        if (c.s_beg < c.s_end) all();
    } else {
        constexpr int kAhead = Tile::NB - 1;  // stages on their way while one is multiplied
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (c.s_beg + i < c.s_end) source.bring(p, c.s_beg + i, lds + i * Tile::kStage, wave);
        int buffer = 0;
        for (int st = c.s_beg; st < c.s_end; ++st) {
            // Stage st has landed, and no wave reads the buffer of stage st - 1 any more.
            if (st + kAhead - 1 < c.s_end)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((kAhead - 1) * Source::kDma)
                             : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (st + kAhead < c.s_end)
                source.bring(p, st + kAhead, lds + (buffer == 0 ? Tile::NB - 1 : buffer - 1) * Tile::kStage, wave);
            multiply(st, lds + buffer * Tile::kStage);
            buffer = buffer == Tile::NB - 1 ? 0 : buffer + 1;
        }
    }
    rows_output<T, MODE, kRowsAny, Tile>(p, c, acc, wp, wq);
}

// ---- eight waves, a workgroup a CU that goes from tile to tile.
//
// Two waves a SIMD, one half of the waves a slot behind the other: while one reads its operands of a step from
// LDS, the other multiplies.  A barrier ends each slot, four of them a stage.  The stages of a workgroup's
// tiles are one stream: the next tile's first ones are on their way during a tile's last, and one half of the
// waves writes its outputs while the other multiplies.  Against a tile a workgroup: sums of 64 tokens for 8 experts'
// 28672 x 4096 482 us, 644 before.  Slower, and not kept: both steps of a stage in one slot (2047 x 14336 over 4096
// 260 against 246 us on 128 rows; no registers for it on 256), stages of 64 bytes five deep (235 against 196), the
// next stage requested before the outputs and these left in flight (806 against 795 for 256 tokens).
template <class E, RowsMode MODE, RowsOutput KIND, class Tile>
__global__ __launch_bounds__(Tile::kThreads) void rows_stream_kernel(RowsMm p, int most) {
    typedef typename E::type T;
    constexpr int RT = Tile::RT, TT = Tile::TT;
    using Source = RowsSource<T, MODE, Tile, kRowsDma>;
    extern __shared__ __align__(16) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % Tile::WP, wq = wave / Tile::WP;
    RowsTiles<MODE, Tile, Source::kStep> tiles;
    RowsRun run(tiles.total(p, most), MODE == kRowsWeight);
    if (run.at >= run.end) return;
    constexpr int kAhead = Tile::NB - 1;
    static_assert(kAhead == 1 || kAhead == 2, "the waits below");
    // The stream's next stage, of the tile `brought`.  A tile without stages has one of zeros.
    Source source;
    int brought = run.at, st, st_end, pending = 0;  // pending: stages brought and not multiplied yet
    auto open = [&]() {
        const RowsPlace c = tiles.place(p, run.tile(brought));
        source.open(p, c, wave);
        st = c.s_beg, st_end = max(c.s_end, c.s_beg + 1);
        source.aim(p, st, c.s_end, wave);
    };
    open();
    // Forward: a stage's rows are asked for between the products of the slot behind the columns' requests, and these
    // behind the reads (2047 x 14336 over 4096 198 us, 213 otherwise; the other forms lose, SwiGLU of 8 experts 733
    // against 703, as less of the stage's way to memory is hidden).
    constexpr bool kBetween = MODE == kRowsForward;
    uint8_t *rows_due = nullptr;
    auto bring = [&](int buffer) {
        if (st == st_end) {
            if (brought + run.step >= run.end) return;
            brought += run.step;
            open();
        }
        uint8_t *const to = lds + buffer * Tile::kStage;
        if (source.whole > 0) {
            source.bring_whole_p(p, to, wave);
            if (kBetween) rows_due = to;
            else source.bring_whole_q(p, to, wave);
        } else {  // the sums, or their half, end inside the stage (or begin anew with the next)
            source.bring(p, st, to, wave);
            source.aim(p, st + 1, st_end, wave);
        }
        ++st;
        ++pending;
    };

    f32x4v acc[RT][TT];
    const typename Source::OpP::Reader read_p(16 * RT * wp);
    const typename Source::OpQ::Reader read_q(16 * TT * wq);
    u32x4v a[RT], b[TT];
    // SwiGLU: the waves behind the tile's rows leave the operands and products out (1023 tokens of 8 experts, three
    // routers: 628, 689 and 613 us, 643, 700 and 624 with them; a forward product loses by the branches, 204 against
    // 199, tiles of 160 rows 650 against 635).
    constexpr bool kIdle = MODE == kRowsSwiglu && TT == 8;
    bool idle = false;
    auto read = [&](auto u_tag, int buffer) {
        constexpr int U = decltype(u_tag)::value;
        const uint8_t *const in_p = lds + buffer * Tile::kStage, *const in_q = in_p + Tile::kStageP;
        if (kIdle && idle) return;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) a[rt] = read_p.template read<U>(in_p, rt);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) b[tt] = read_q.template read<U>(in_q, tt);
    };
    auto products = [&](bool between) {
        if (kIdle && idle) return;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            if (kBetween && tt == 1 && between) {
                __builtin_amdgcn_sched_barrier(0);
                if (rows_due != nullptr) source.bring_whole_q(p, rows_due, wave), rows_due = nullptr;
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][tt] = rows_mfma<T>(a[rt], b[tt], acc[rt][tt]);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    auto slot_end = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // The stage behind the current one has landed; the one behind that may be on its way (loads return in order).
    auto landed = [&](int behind) {
        if (kAhead == 2 && pending - behind == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(Source::kDma) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    constexpr std::integral_constant<int, 0> kU0{};
    constexpr std::integral_constant<int, 1> kU1{};

#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        bring(i);
        if (rows_due != nullptr) source.bring_whole_q(p, rows_due, wave), rows_due = nullptr;
    }
    landed(0);
    slot_end();
    if (wave >= 4) slot_end();
    int buffer = 0;
    for (; run.at < run.end; run.at += run.step) {
        const RowsPlace c = tiles.place(p, run.tile(run.at));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = f32x4v{0.f, 0.f, 0.f, 0.f};
        if (kIdle) idle = c.rows_q <= 16 * TT * wq;
        for (int left = max(c.s_end - c.s_beg, 1); left > 0; --left) {
            // Into the buffer of the stage before, whose last readers' slot has ended.
            const int before = buffer == 0 ? Tile::NB - 1 : buffer - 1;
            if (!kBetween) bring(before);
            read(kU0, buffer);
            if (kBetween) bring(before);
            slot_end();
            products(true);
            slot_end();
            read(kU1, buffer);
            if (wave >= 4) landed(1);
            slot_end();
            products(false);
            if (wave < 4) landed(1);
            slot_end();
            rows_turn<T, MODE, Tile>(p, c, c.s_end - left, acc);
            --pending;
            buffer = buffer == Tile::NB - 1 ? 0 : buffer + 1;
        }
        rows_output<T, MODE, KIND, Tile>(p, c, acc, wp, wq);
    }
    if (wave < 4) slot_end();
}

template <class E, RowsMode MODE, class Tile, RowsWay WAY>
hipError_t run_rows(RowsMm p, hipStream_t stream) {
    constexpr int kOutP = MODE == kRowsSwiglu ? Tile::kP / 2 : Tile::kP;
    p.tiles_p = (p.P + kOutP - 1) / kOutP;
    p.tiles_q = (p.Q + Tile::kQ - 1) / Tile::kQ;
    if (MODE == kRowsWeight) p.tiles_q *= p.halves;
    else if (p.offsets != nullptr) p.tiles_q += std::min(p.n_experts, p.M);
    if ((int64_t)p.tiles_p * p.tiles_q > INT32_MAX / 64) return hipErrorInvalidConfiguration;
    const int64_t most = (int64_t)p.tiles_p * p.tiles_q * p.slices *
                         (MODE == kRowsWeight && p.offsets != nullptr ? p.n_experts : 1);
    // Whole chunks of every XCD.
    const int64_t blocks = MODE == kRowsWeight ? (most + 255) / 256 * 256 : most;
    if (most >= INT32_MAX / 64 || blocks * Tile::kThreads >= 1LL << 32) return hipErrorInvalidConfiguration;
    auto go = [&](auto kernel, int wgs) {
        const hipError_t e = ensure_dynamic_lds((const void *)kernel, Tile::kLds);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(Tile::kThreads), Tile::kLds, stream, p, (int)most);
        return hipGetLastError();
    };
    if constexpr (Tile::kWaves == 8) {
        const int wgs = (int)std::min<int64_t>(blocks, device_cu_count());
        const RowsEpilogue &e = p.epi;
        if constexpr (MODE == kRowsForward || MODE == kRowsSwiglu)
            if (p.slices == 1 &&
                (e.bias != nullptr || e.residual != nullptr || e.pre != nullptr || e.act != JJO_ACT_NONE))
                return go(rows_stream_kernel<E, MODE, kRowsFull, Tile>, wgs);
        if constexpr (MODE == kRowsWeight) {
            const int es = p.wide ? 4 : (int)sizeof(typename E::type);
            const bool lines = p.slices > 1 ? (uintptr_t)p.part % 64 == 0 && p.P % 16 == 0
                                            : ((uintptr_t)p.y | (uintptr_t)p.y2 | (uintptr_t)(p.ldy * es)) % 64 == 0;
            if (!lines) return go(rows_stream_kernel<E, MODE, kRowsFull, Tile>, wgs);
        }
        return go(rows_stream_kernel<E, MODE, kRowsPlain, Tile>, wgs);
    } else
        return go(rows_mm_kernel<E, MODE, Tile, WAY>, (int)blocks);
}

// DMA where every memory row of both operands is 16-byte aligned, a tile's rows and a stage's elements
// are within 4 GiB of its first, and rows come in whole pieces.
inline RowsWay rows_way(RowsMode mode, int es, const RowsMm &p) {
    const int piece = 16 / es;
    // The contiguous directions: of both operands the sums' (forward), P's and the sums' (input), P's and Q's (weight).
    const int a = mode == kRowsForward || mode == kRowsSwiglu ? p.K : p.P, b = mode == kRowsWeight ? p.Q : p.K;
    if (p.ldp * es >= (1LL << 32) / 512 || p.ldq * es >= (1LL << 32) / 512) return kRowsCopied;
    auto aligned = [&](const void *m, int64_t ld) { return (uintptr_t)m % 16 == 0 && ld % piece == 0; };
    const bool all = aligned(p.p, p.ldp) && aligned(p.q, p.ldq) && aligned(p.p2, p.ldp) && aligned(p.rest, p.ldq) &&
                     p.rest_plane % piece == 0 && a % piece == 0 && b % piece == 0;
    return all ? kRowsDma : es == 4 ? kRowsWords : a < piece || b < piece ? kRowsCopied : kRowsStaged;
}

template <class E, RowsMode MODE>
hipError_t rows_by_tile(const RowsMm &p, int tile, hipStream_t stream) {
    const RowsWay way = rows_way(MODE, (int)sizeof(typename E::type), p);
    if (way == kRowsCopied) return run_rows<E, MODE, RowsTile<4, 4, 2, 2>, kRowsCopied>(p, stream);
    if (way != kRowsDma) {
        constexpr bool kWords = sizeof(typename E::type) == 4;
        constexpr RowsWay kWay = kWords ? kRowsWords : kRowsStaged;
        if (tile == kRowsTile64) return run_rows<E, MODE, RowsTile<2, 2, 2, 2, kWords ? 4 : 2>, kWay>(p, stream);
        return run_rows<E, MODE, RowsTile<4, 4, 2, 2>, kWay>(p, stream);
    }
    if (tile == kRowsTile64) return run_rows<E, MODE, RowsTile<2, 2, 2, 2, 4>, kRowsDma>(p, stream);
    if constexpr (sizeof(typename E::type) == 2) {
        // The large tiles write whole groups of eight columns.
        if (tile == kRowsTile256 && p.P % 8 == 0) return run_rows<E, MODE, RowsTile<4, 8, 4, 2>, kRowsDma>(p, stream);
        if constexpr (MODE == kRowsForward || MODE == kRowsInput)
            if (tile == kRowsTile160 && p.P % 8 == 0)
                return run_rows<E, MODE, RowsTile<4, 5, 4, 2, 3>, kRowsDma>(p, stream);
    }
    return run_rows<E, MODE, RowsTile<4, 4, 2, 2>, kRowsDma>(p, stream);
}

}  // namespace
}  // namespace jjo
