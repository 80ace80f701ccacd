// Device pieces that the MXFP4 matrix kernels share: the scaled matrix instruction, an expert's tile
// of sorted rows, and the SwiGLU epilogue.
#pragma once

#include "mxfp4_common.hpp"

namespace jjo {

// acc[16 weights][16 tokens] += W[16][128] . X[16][128]^T.  Lane l holds row l % 16 of either
// operand and of it the block l / 16 (32 values, 16 bytes) with that block's scale byte, byte BW (BX)
// of its scale register; of acc it holds weights 4 * (l / 16) + 0..3 of token l % 16.
template <int BW, int BX>
__device__ __forceinline__ f32x4v mx_mfma(u32x4v w, u32x4v x, f32x4v acc, uint32_t sw, uint32_t sx) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, BW, (int)sw, BX, (int)sx);
}

// Inclusive sums over the wave's lanes: row shifts inside the rows of 16, then row_bcast15 and
// row_bcast31; a lane without a source takes 0.
__device__ __forceinline__ int mx_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// The tile-th tile of `rows` sorted rows, counted over the experts in order: its expert, its
// first row and the end of its expert's rows; false behind the last.  Ranges are clamped to
// [0, M], so a malformed table drops rows instead of leaving the buffers.  All lanes of a
// wave call it together.
__device__ __forceinline__ bool mx_expert_tile(const int32_t *__restrict__ offsets, int n_experts, int M, int rows,
                                               int tile, int &expert, int &first, int &end) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int e0 = 0; e0 < n_experts; e0 += 64) {
        const int e = e0 + lane;
        int beg = 0, fin = 0;
        if (e < n_experts) {
            beg = min(max(offsets[e], 0), M);
            fin = min(max(offsets[e + 1], beg), M);
        }
        const int mine = (fin - beg + rows - 1) / rows;
        const int incl = mx_scan(mine);
        const uint64_t past = __ballot(base + incl > tile);
        if (past != 0) {
            const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
            const int t0 = base + __builtin_amdgcn_readlane(incl - mine, l);
            const int begin = __builtin_amdgcn_readlane(beg, l);
            expert = e0 + l;  // scalars: the row addresses below are
            first = begin + (tile - t0) * rows;
            end = __builtin_amdgcn_readlane(fin, l);
            return first >= begin && first < end;  // only sums of a malformed table that overflowed fail it
        }
        base += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

__device__ __forceinline__ float mx_silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// One block of 32 intermediate values of one token: the lane holds values 16 * h + 4 * q + i
// (h = 0, 1; q = lane / 16) as silu(gate[h][i]) * up[h][i].  Writes the codes and the scale.
__device__ __forceinline__ void mx_swiglu_store(const f32x4v (&gate)[2], const f32x4v (&up)[2], uint8_t *codes,
                                                uint8_t *scale, bool live) {
    const int q = (threadIdx.x & 63) >> 4;
    float v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = mx_silu_mul(gate[h][i], up[h][i]);
    uint32_t m = mx_amax8(v);
    uint32_t o = (uint32_t)__shfl_xor((int)m, 16);
    m = o > m ? o : m;
    o = (uint32_t)__shfl_xor((int)m, 32);
    m = o > m ? o : m;
    const uint32_t s = mx_scale_byte(m);
    const uint32_t c = mx_codes8(v, s);
    if (!live) return;
    *reinterpret_cast<uint16_t *>(codes + 2 * q) = (uint16_t)c;
    *reinterpret_cast<uint16_t *>(codes + 8 + 2 * q) = (uint16_t)(c >> 16);
    if (q == 0) *scale = (uint8_t)s;
}

}  // namespace jjo
