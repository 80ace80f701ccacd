// Top-k gating of one token by one wave, for the routing kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace jjo {
namespace {

// ---------------------------------------------------------------- top-k
// One wave per token (num_experts <= 1024, top_k <= 32).
// Selection: moe_top_k.cu:120-176 -- top_k rounds; round k scans e = 0..E-1 with
// v(e) = -inf for an expert taken in an earlier round, else the logit, keeps e = 0's
// value first and takes a later e only when strictly greater; ids[k] in selection
// order.  That keeps the smallest id of the largest non-NaN value, or expert 0 when
// v(0) is NaN (nothing compares greater than NaN), and it re-selects a taken expert
// once only -inf values are left; the wave computes exactly that.  Each lane holds
// experts lane + 64j as unsigned keys in the order of the values (-0 as +0; NaN and
// experts past the end 0, below the key of -inf; a taken expert becomes -inf): a
// round is a lane-local maximum, a DPP maximum over the wave and one ballot of the
// lanes that hold it, whose smallest (j, lane) is the smallest id.  The rounds are a
// serial chain, so their latency is the kernel's time: shuffles of (value, id, valid)
// over 16 registers a lane took 11.9 us for 100 tokens, 64 experts, top-6; PER =
// ceil(num_experts / 64) keys and DPP take 4.8 us.
// Weights: softmax over the selected logits (delayed_softmax, moe_top_k.cu:12-55,
// 190-195): max = the first selected value, e_i = expf(v_i - max), and the sum is
// the 32-lane xor butterfly of warp_reduce_xor_sum (include/cuda_utils.cuh:37-43)
// over e_0..e_{top_k-1} held by lanes 0..top_k-1 (zeros elsewhere), run on the
// lanes themselves, so the association order is the reference's; w_i = e_i * (1 / sum).
__device__ __forceinline__ uint64_t ballot64(bool p) { return __ballot(p); }

constexpr uint32_t kNegInfKey = 0x007fffffu;  // order_key(-inf)

// Unsigned key in the order of the non-NaN floats, -0 equal to +0; NaN gives 0.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 + 0 = +0
    return x == x ? u ^ (uint32_t)(((int32_t)u >> 31) | (int32_t)0x80000000) : 0u;
}

__device__ __forceinline__ float order_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Maximum / sum of the wave's 64 values, in every lane: row shifts inside the rows of
// 16, then row_bcast15 and row_bcast31; a lane without a source takes 0.
#define JJO_WAVE_FOLD(v, OP)                                                          \
    v = OP(v, (decltype(v))__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false)); \
    v = OP(v, (decltype(v))__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false)); \
    v = OP(v, (decltype(v))__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false)); \
    v = OP(v, (decltype(v))__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false)); \
    v = OP(v, (decltype(v))__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false)); \
    v = OP(v, (decltype(v))__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false))

__device__ __forceinline__ uint32_t umax32(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t uadd32(uint32_t a, uint32_t b) { return a + b; }

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    JJO_WAVE_FOLD(v, umax32);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
    JJO_WAVE_FOLD(v, uadd32);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
#undef JJO_WAVE_FOLD

// All 64 lanes of the wave call this for one token; lanes 0..top_k-1 write
// weights[lane] and ids[lane].  num_experts <= 64 * PER.
template <int PER>
__device__ __forceinline__ void top_k_token(const float *__restrict__ row, int num_experts, int top_k,
                                            float *__restrict__ weights, int *__restrict__ ids, int lane) {
    uint32_t key[PER];
    float v0 = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = lane + 64 * j;
        const float x = e < num_experts ? row[e] : 0.0f;
        if (j == 0) v0 = x;
        key[j] = e < num_experts ? order_key(x) : 0u;
    }
    v0 = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v0)));  // expert 0's logit
    bool nan0 = v0 != v0;  // until expert 0 is taken (and -inf)
    float my_v = 0.0f, mx = 0.0f;
    int my_id = 0;
    for (int k = 0; k < top_k; ++k) {
        uint32_t bk = key[0];
        int bj = 0;
#pragma unroll
        for (int j = 1; j < PER; ++j)
            if (key[j] > bk) {  // ids ascend with j
                bk = key[j];
                bj = j;
            }
        float bv;
        int bid;
        if (nan0) {  // v(0) NaN: the scan never leaves expert 0
            bv = v0;
            bid = 0;
            nan0 = false;
        } else {  // expert 0 is a candidate: the maximum is at least the key of -inf
            const uint32_t m = wave_max(bk);
            uint64_t tied = ballot64(bk == m);
            int j = 0;
            if constexpr (PER > 1) {
                if ((tied & (tied - 1)) == 0) {
                    j = __builtin_amdgcn_readlane(bj, __builtin_ctzll(tied));
                } else {
                    for (j = 0; j < PER - 1; ++j) {
                        const uint64_t at_j = ballot64(bk == m && bj == j);
                        if (at_j != 0) {
                            tied = at_j;
                            break;
                        }
                    }
                }
            }
            bid = 64 * j + __builtin_ctzll(tied);
            bv = order_value(m);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (lane + 64 * j == bid) key[j] = kNegInfKey;
        if (k == 0) mx = bv;
        if (lane == k) {
            my_v = bv;
            my_id = bid;
        }
    }
    const float ex = lane < top_k ? expf(my_v - mx) : 0.0f;
    float t = ex;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) t = t + __shfl_xor(t, off);
    const float inv_sum = 1.0f / __shfl(t, 0);
    if (lane < top_k) {
        weights[lane] = ex * inv_sum;
        ids[lane] = my_id;
    }
}

}  // namespace
}  // namespace jjo
