// MXFP4 weights x MXFP4 activations for few tokens (a decode batch, an expert's handful of
// rows) on gfx950's scaled matrix instruction, operands straight from memory to registers.
//
//     y[t][n] = sum over blocks b of 2^(sw[n,b] + sx[t,b] - 254) * sum_j cw[n,b,j] * cx[t,b,j]
//
// Bound by reading the weights (17/32 byte a value).  What that takes:
//   * Addresses.  The instruction's operand has 16 rows in neighbouring lanes, so loading it as it is
//     touches four rows in every four lanes, 64 cache tags a load instead of 16; with the
//     activation's loads beside the weights' that was what the kernel waited for (114688 x 4096, 4
//     tokens: 54 us, of which 13 the activation's loads and 10 the scales').  Here the 16 rows of an operand
//     are 4 weight rows x 4 neighbouring blocks: lane 16 j + 4 a + b has row a, block 4 j + b of a chunk of 16
//     blocks, so a load is 4 rows x 256 contiguous bytes.  The activation is held alike (4
//     tokens x 4 blocks), and of the 16 x 16 products the ones wanted are those whose weight and
//     activation blocks agree, a quarter: sum over b of acc[(a, b)][(t, b)].  The matrix cores idle
//     anyway; the diagonal is summed once, at the end.
//   * Loads in flight: a wave asks for all chunks of its slice (NC) before it multiplies the first; KW
//     waves cut K between them, so that a small output still fills the chip.  Sums are fp32, the
//     slices' added through LDS in slice order.
//   * Scales: 16 bytes a lane, once per NC chunks, through the wave's own LDS.
#include <hip/hip_runtime.h>

#include "mxfp4_mm.hpp"

namespace jjo {
namespace {

struct MxProblem {
    const uint8_t *w, *w2, *x;  // w2: the up matrix (SwiGLU)
    void *y;                    // outputs, or the MXFP4 rows of the SwiGLU form
    int dtype;
    int K, N, M;
    int tiles_n;           // row tiles of the launch
    int first_t, first_n;  // its first token tile and row tile
    MxGroups g;
};

// 16 consecutive values of the fused activation.
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

__device__ __forceinline__ float quad_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, true));  // lane ^ 1
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, true));  // lane ^ 2
    return v;
}

// Chunks of 512 values that a wave asks for at once: 3 and 4 cost registers and gain nothing on average
// (one token, K = 4096, N = 11008: 6.6 us with 2, 6.5 with 4; K = 11008, N = 4096: 7.4 and 7.0).
constexpr int kMxChunks = 2;

// A wave has 16 weight rows (4 operands of 4 rows) x TG operands of 4 tokens and NC chunks of 512 values at
// once; KW waves cut K between them, RW have rows of their own.  SWIGLU: RW = 4, two times 16 gate
// rows and the two times 16 up rows beside them.  XT: void (x is MXFP4), or the type of the one
// token's row, which every wave quantizes for its own slice of K.
template <int TG, int KW, int RW, bool GROUPED, bool SWIGLU, class XT>
__global__ __launch_bounds__(64 * KW * RW) void mxfp4_direct_kernel(MxProblem p) {
    constexpr bool kFused = !std::is_void_v<XT>;
    constexpr int W = KW * RW, kTokens = 4 * TG;
    constexpr int NC = kMxChunks, kPieces = NC;  // of 16 scale bytes a row
    constexpr int kScaleRows = kFused ? 16 : 16 + kTokens, kAtOnce = 64 / kPieces;  // rows a load instruction
    constexpr int kScaleLoads = (kScaleRows + kAtOnce - 1) / kAtOnce;
    __shared__ __align__(16) uint8_t s_scales[W][kScaleLoads * kAtOnce][16 * kPieces];
    __shared__ __align__(16) uint8_t x_codes[kFused ? W : 1][kFused ? 256 * NC : 16];
    __shared__ uint8_t x_scales[kFused ? W : 1][kFused ? 16 * NC : 1];
    __shared__ float part[W][TG][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave % KW, rw = wave / KW;
    const int la = lane >> 2 & 3, lb = lane & 3, lj = lane >> 4, blk0 = 4 * lj + lb;
    // Row tiles vary fastest: the eight XCDs, which take workgroups in turn, then have the same
    // share of the token tiles that exist.
    const int tile_t = p.first_t + (int)(blockIdx.x / (unsigned)p.tiles_n);
    const int tile_n = p.first_n + (int)(blockIdx.x % (unsigned)p.tiles_n);
    int expert = 0, first = tile_t * kTokens, end = p.M;
    if constexpr (GROUPED) {
        if (!mx_expert_tile(p.g.offsets, p.g.n_experts, p.M, kTokens, tile_t, expert, first, end)) return;
    }
    static_assert(!SWIGLU || RW == 4, "32 gate rows and the same 32 up rows");
    const int n0 = SWIGLU ? 32 * tile_n + 16 * (rw & 1) : 16 * (tile_n * RW + rw);
    const int nb = p.K / kQK, chunks = (nb + 15) / 16;
    const int c_beg = chunks * kw / KW, c_end = chunks * (kw + 1) / KW;
    const size_t half = (size_t)p.K / 2;

    const uint8_t *const w = SWIGLU && rw >= 2 ? p.w2 : p.w;
    const size_t w_first = (size_t)expert * p.N, w_all = (size_t)(GROUPED ? p.g.n_experts : 1) * p.N;
    const uint8_t *w_row[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) w_row[g] = w + (w_first + min(n0 + 4 * g + la, p.N - 1)) * half;
    // The token of row `r` of the tile, and x's rows.
    const bool routed = GROUPED && p.g.src_route != nullptr;
    const size_t x_all = routed ? p.g.x_rows : p.M;
    auto token = [&](int r) {
        const int t = min(first + r, end - 1);
        return routed ? min(max(p.g.src_route[t] / p.g.top_k, 0), p.g.x_rows - 1) : t;
    };
    const uint8_t *x_row[TG], *s_row[kScaleLoads];
    if constexpr (!kFused) {
#pragma unroll
        for (int t = 0; t < TG; ++t) x_row[t] = p.x + (size_t)token(4 * t + la) * half;
    }
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
        const int r = i * kAtOnce + lane / kPieces;
        if (kFused || r < 16) s_row[i] = w + w_all * half + (w_first + min(n0 + min(r, 15), p.N - 1)) * nb;
        else s_row[i] = p.x + x_all * half + (size_t)token(min(r - 16, kTokens - 1)) * nb;
    }

    f32x4v acc[4][TG];
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int t = 0; t < TG; ++t) acc[g][t] = f32x4v{0.f, 0.f, 0.f, 0.f};

    for (int c0 = c_beg; c0 < c_end; c0 += NC) {
        // ---- everything of NC chunks is asked for, in the order of its use (loads return in order);
        // chunks behind the slice are its last one again
        float v[16];
        if constexpr (kFused) {  // 16 values a lane; behind the row's end its last ones (they meet zero weights)
            typedef std::conditional_t<kFused, XT, float> T;
            load16((const T *)p.x + min(512 * c0 + 16 * lane, p.K - 32 + 16 * (lane & 1)), v);
        }
        u32x4v sv[kScaleLoads], a[NC][4], b[NC][TG];
        const int piece = lane % kPieces, s_at = min(16 * (c0 + piece), nb - 16);
        // The last 16 bytes of a row where it ends earlier: behind codes, so also before a short row's start.
#pragma unroll
        for (int i = 0; i < kScaleLoads; ++i) __builtin_memcpy(&sv[i], s_row[i] + s_at, 16);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const size_t at = 16 * (size_t)min(16 * min(c0 + c, c_end - 1) + blk0, nb - 1);
#pragma unroll
            for (int g = 0; g < 4; ++g) a[c][g] = *reinterpret_cast<const u32x4v *>(w_row[g] + at);
            if constexpr (!kFused) {
#pragma unroll
                for (int t = 0; t < TG; ++t) b[c][t] = *reinterpret_cast<const u32x4v *>(x_row[t] + at);
            }
        }
        // ---- scales, and the fused activation, to the wave's LDS
        if constexpr (kFused) {
            uint32_t m = mx_amax8(v), o = mx_amax8(v + 8);
            m = o > m ? o : m;
            o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true);  // lane ^ 1
            m = o > m ? o : m;
            const uint32_t s = mx_scale_byte(m);
            *reinterpret_cast<uint2 *>(&x_codes[wave][8 * lane]) = make_uint2(mx_codes8(v, s), mx_codes8(v + 8, s));
            if ((lane & 1) == 0) x_scales[wave][lane >> 1] = (uint8_t)s;
        }
        const int over = 16 * (c0 + piece) + 16 - nb;  // zeros behind the row's end
#pragma unroll
        for (int i = 0; i < kScaleLoads; ++i) {
            if (16 * (c0 + kPieces) > nb) {
                unsigned __int128 s;
                __builtin_memcpy(&s, &sv[i], 16);
                s = over >= 16 ? 0 : s >> (8 * max(over, 0));
                __builtin_memcpy(&sv[i], &s, 16);
            }
            *reinterpret_cast<u32x4v *>(&s_scales[wave][i * kAtOnce + lane / kPieces][16 * piece]) = sv[i];
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c0 + c >= c_end) break;
            if (16 * (c0 + c) + 16 > nb) {  // the row ends inside the chunk: zero weights behind it
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    if (16 * (c0 + c) + blk0 >= nb) a[c][g] = u32x4v{0u, 0u, 0u, 0u};
            }
            uint32_t sw[4], sx[TG];
#pragma unroll
            for (int g = 0; g < 4; ++g) sw[g] = s_scales[wave][4 * g + la][16 * c + blk0];
#pragma unroll
            for (int t = 0; t < TG; ++t) {
                if constexpr (kFused) {
                    b[c][t] = *reinterpret_cast<const u32x4v *>(&x_codes[wave][16 * (16 * c + blk0)]);
                    sx[t] = x_scales[wave][16 * c + blk0];
                } else {
                    sx[t] = s_scales[wave][16 + 4 * t + la][16 * c + blk0];
                }
            }
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int t = 0; t < TG; ++t) acc[g][t] = mx_mfma<0, 0>(a[c][g], b[c][t], acc[g][t], sw[g], sx[t]);
        }
        __builtin_amdgcn_wave_barrier();
    }

    // ---- acc[g][t] of lane 16 q + 4 t' + b' has (row 4 g + q, block group i) in register i for token 4 t + t',
    // block group b': register b' of it, summed over the four lanes of b', is the output.  Lane 16 q + 4 t' + b' keeps
    // row 4 b' + q.
    float r[TG];
#pragma unroll
    for (int t = 0; t < TG; ++t) {
        float s[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4v d = acc[g][t];
            s[g] = quad_sum(lb == 0 ? d[0] : lb == 1 ? d[1] : lb == 2 ? d[2] : d[3]);
        }
        r[t] = lb == 0 ? s[0] : lb == 1 ? s[1] : lb == 2 ? s[2] : s[3];
    }
#pragma unroll
    for (int t = 0; t < TG; ++t) part[wave][t][lane] = r[t];
    __syncthreads();
    auto total = [&](int row_wave, int t) {
        float s = part[row_wave * KW][t][lane];
#pragma unroll
        for (int k = 1; k < KW; ++k) s += part[row_wave * KW + k][t][lane];
        return s;
    };
    const int row = 4 * lb + lj;
    if constexpr (SWIGLU) {
        // A block of 32 values of a token is two values each of 16 lanes (all but bits 2, 3 of the lane).
        uint8_t *codes = (uint8_t *)p.y, *scales = codes + (size_t)p.M * (p.N / 2);
        const int n = 32 * tile_n;
        for (int t = wave; t < TG; t += W) {
            const int tok = first + 4 * t + la;
            float h[8] = {mx_silu_mul(total(0, t), total(2, t)), mx_silu_mul(total(1, t), total(3, t)), 0, 0, 0, 0, 0, 0};
            uint32_t m = mx_amax8(h);
#pragma unroll
            for (int d : {1, 2, 16, 32}) {
                const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
                m = o > m ? o : m;
            }
            const uint32_t s = mx_scale_byte(m);
            uint32_t c = mx_codes8(h, s);
            c |= (uint32_t)__shfl_xor((int)c, 16) << 8;  // of row ^ 1: bits 8..15
            if (tok >= end || (lj & 1) != 0) continue;
            uint8_t *to = codes + (size_t)tok * (p.N / 2) + n / 2 + row / 2;
            to[0] = (uint8_t)((c & 15u) | (c >> 8 & 15u) << 4);
            to[8] = (uint8_t)((c >> 4 & 15u) | (c >> 12 & 15u) << 4);
            if (row == 0) scales[(size_t)tok * (p.N / kQK) + n / kQK] = (uint8_t)s;
        }
    } else {
#pragma unroll
        for (int t = 0; t < TG; ++t) {
            if (t % KW != kw) continue;
            const float out = total(rw, t);
            const int tok = first + 4 * t + la, n = n0 + row;
            if (tok >= end || n >= p.N) continue;
            const size_t to = (size_t)(GROUPED && p.g.route_dst != nullptr ? p.g.route_dst[tok] : tok) * p.N + n;
            if (p.dtype == JJO_DTYPE_F32) ((float *)p.y)[to] = out;
            else if (p.dtype == JJO_DTYPE_F16) ((_Float16 *)p.y)[to] = (_Float16)out;
            else ((__bf16 *)p.y)[to] = (__bf16)out;
        }
    }
}

template <int TG, int KW, int RW, bool SWIGLU, class XT = void>
hipError_t run_direct(MxProblem p, hipStream_t stream) {
    constexpr int rows = SWIGLU ? 32 : 16 * RW, threads = 64 * KW * RW;
    // token tiles of M rows, and one more for each expert that can have a rest
    const int64_t rests = p.g.offsets != nullptr ? std::min(p.g.n_experts, p.M) : 0;
    const int64_t token_tiles = (p.M + 4 * TG - 1) / (4 * TG) + rests;
    const int64_t row_tiles = (p.N + rows - 1) / rows;
    // A grid has fewer than 2^32 threads: more (2^33 outputs of short rows, 2^28 weight rows) are several launches.
    constexpr int64_t kMost = ((1LL << 32) - 1) / threads;
    for (int64_t n = 0; n < row_tiles; n += kMost) {
        p.first_n = (int)n, p.tiles_n = (int)std::min(kMost, row_tiles - n);
        const int64_t at_once = kMost / p.tiles_n;
        for (int64_t t = 0; t < token_tiles; t += at_once) {
            p.first_t = (int)t;
            const dim3 grid((unsigned)(p.tiles_n * std::min(at_once, token_tiles - t))), block(threads);
            if constexpr (!std::is_void_v<XT>)
                hipLaunchKernelGGL((mxfp4_direct_kernel<TG, KW, RW, false, false, XT>), grid, block, 0, stream, p);
            else if (p.g.offsets != nullptr)
                hipLaunchKernelGGL((mxfp4_direct_kernel<TG, KW, RW, true, SWIGLU, void>), grid, block, 0, stream, p);
            else if constexpr (!SWIGLU)
                hipLaunchKernelGGL((mxfp4_direct_kernel<TG, KW, RW, false, false, void>), grid, block, 0, stream, p);
            else
                return hipErrorInvalidValue;
            if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace

// Tokens at once, of the mean rows of an expert: an uneven share of 3 rows is mostly up to 4 for one expert, and
// more operands than tokens cost what they would with tokens (K = 4096, N = 14336: 7.4 us for 4 tokens on one
// operand, 7.9 for 7 on two, 9.6 for 16 on four).  More than 16 tokens are more tiles of 16: operands for 24
// and 32 took longer at every size (4096 x 4096, 32 tokens: 7.6 against 5.9 us).
hipError_t launch_mxfp4_direct(const void *w, const void *xq, void *y, int dtype, int K, int N, int M,
                               const MxGroups &groups, hipStream_t stream) {
    const MxProblem p{(const uint8_t *)w, nullptr, (const uint8_t *)xq, y, dtype, K, N, M, 0, 0, 0, groups};
    const bool grouped = groups.offsets != nullptr;
    const int64_t experts = mx_experts(M, groups), rows = mx_rows(M, groups), mean = (M + experts - 1) / experts;
    if (mean <= (grouped ? 3 : 4)) return run_direct<1, 4, 1, false>(p, stream);
    if (rows <= 8) return run_direct<2, 4, 1, false>(p, stream);
    // Two row tiles a workgroup and half as many slices of K once there are three workgroups a CU
    // (4096 x 4096: 32 tokens 5.9 us on four slices, 6.5 on two; 96 tokens 10.6 and 9.2).
    if (experts * ((N + 15) / 16) * ((rows + 15) / 16) > 3 * device_cu_count())
        return run_direct<4, 2, 2, false>(p, stream);
    return run_direct<4, 4, 1, false>(p, stream);
}

hipError_t launch_mxfp4_direct_swiglu(const void *w_gate, const void *w_up, const void *xq, void *mid, int K, int I,
                                      int M, const MxGroups &groups, hipStream_t stream) {
    const MxProblem p{(const uint8_t *)w_gate, (const uint8_t *)w_up, (const uint8_t *)xq, mid, JJO_DTYPE_F32, K, I, M,
                      0, 0, 0, groups};
    const int experts = mx_experts(M, groups), mean = (M + experts - 1) / experts;
    if (mean <= 3) return run_direct<1, 1, 4, true>(p, stream);
    return run_direct<4, 1, 4, true>(p, stream);
}

hipError_t launch_mxfp4_gemv(const void *w, const void *x, int x_dtype, void *y, int y_dtype, int K, int N,
                             hipStream_t stream) {
    const MxProblem p{(const uint8_t *)w, nullptr, (const uint8_t *)x, y, y_dtype, K, N, 1, 0, 0, 0, MxGroups{}};
    return mx_by_dtype(x_dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        return run_direct<1, 4, 1, false, T>(p, stream);
    });
}

}  // namespace jjo
