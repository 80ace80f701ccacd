// Token rows (fp32, fp16, bf16) to their experts and back on gfx950, and the gradients.
//
//   sort      pos(r) = #{live r' : e(r') < e(r)} + #{live r' < r : e(r') = e(r)}, the order of
//             moe_dispatch_kernel; a route whose id is outside [0, E) is dropped (dst -1)
//   dispatch  rows[pos(r)] = x[r / top_k]
//   its gradient          gx[t] = sum over k of g[dst(t, k)]
//   combine   y[t] = sum over k of w(t, k) rows[dst(t, k)]
//   its gradients         grows[dst(t, k)] = w(t, k) gy[t],  gw(t, k) = <gy[t], rows[dst(t, k)]>
//
// All of it is bound by HBM once there are some hundred rows and by latency below: a row is
// moved in 16-byte pieces, sums are fp32 in k order (one rounding, at the store), and only counts
// are added with atomics, so a result does not depend on timing.
#include <hip/hip_runtime.h>

#include "moe_top_k.hpp"
#include "mxfp4_common.hpp"

namespace jjo {
namespace {

constexpr int kSortMax = 4096;  // routes that every workgroup of the dispatch counts by itself

__device__ __forceinline__ bool live_id(int e, int n_experts) { return (unsigned)e < (unsigned)n_experts; }

__device__ __forceinline__ int wave_total(int v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Exclusive bases of the experts' counts in s_cnt[0..1023] (n_experts <= 1024), by 256 threads
// of one workgroup: thread i takes entries 4i..4i+3.  s_part: four ints.
__device__ __forceinline__ void expert_bases(int *s_cnt, int *s_part) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int c[4], tot = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) tot += c[i] = s_cnt[4 * tid + i];
    int incl = tot;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 63) s_part[wave] = incl;
    __syncthreads();
    int base = incl - tot;
    for (int w = 0; w < wave; ++w) base += s_part[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        s_cnt[4 * tid + i] = base;
        base += c[i];
    }
    __syncthreads();
}

// A row of any length in pieces of 16 bytes, whatever its alignment (a load or store of a wave then
// touches a line more): the last piece ends with the row and overlaps the one before, which is
// the same values once more.  Rows shorter than a piece go by single elements.  8192 tokens top-2 of
// 4095 bf16 values: the combine 32 us, 71 by single elements (31 for 4096).

// ---- dispatch of up to kSortMax routes in one launch.  Workgroup (t + 1, c) has its piece of
// token t's row in flight, counts for each of the token's routes the routes that sort before
// it (16 compares a thread and route at most) and stores the piece at each position;
// workgroup 0 counts the experts' offsets.
template <class U>
__global__ __launch_bounds__(256) void dispatch_rows_kernel(const int32_t *__restrict__ ids,
                                                            const uint16_t *__restrict__ x, int R, int top_k,
                                                            int row_len, int n_experts, int32_t *__restrict__ offsets,
                                                            int32_t *__restrict__ src_route,
                                                            int32_t *__restrict__ dst_of_route,
                                                            uint16_t *__restrict__ rows) {
    constexpr int kIds = kSortMax / 256, kUnits = 4, kLen = sizeof(U) / 2;  // row_len: in 2-byte units
    __shared__ int s_cnt[1024];
    __shared__ int s_part[4][32];
    __shared__ int s_pos[32];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (blockIdx.x == 0) {
        if (blockIdx.y != 0) return;
        for (int e = tid; e < 1024; e += 256) s_cnt[e] = 0;
        __syncthreads();
        for (int r = tid; r < R; r += 256) {
            const int e = ids[r];
            if (live_id(e, n_experts)) atomicAdd(&s_cnt[e], 1);
        }
        __syncthreads();
        const int last = s_cnt[n_experts - 1];
        expert_bases(s_cnt, s_part[0]);
        for (int e = tid; e < n_experts; e += 256) offsets[e] = s_cnt[e];
        if (tid == 0) offsets[n_experts] = s_cnt[n_experts - 1] + last;
        return;
    }
    const int t = blockIdx.x - 1, u0 = blockIdx.y * (256 * kUnits);
    const uint16_t *row = x + (size_t)t * row_len;
    U v[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = (u0 + tid + 256 * i) * kLen;
        if (u < row_len) v[i] = load_any<U>(row + min(u, row_len - kLen));
    }
    int key[kIds];  // expert * kSortMax + route; a dropped route sorts behind all
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
        const int r = tid + 256 * i;
        const int e = r < R ? ids[r] : -1;
        key[i] = live_id(e, n_experts) ? e * kSortMax + r : 0x7fffffff;
    }
    const int r_own = t * top_k + min(lane, top_k - 1);  // lane k: route k of the token
    const int e_own = ids[r_own];
    const int own_key = live_id(e_own, n_experts) ? e_own * kSortMax + r_own : -1;
    for (int k = 0; k < top_k; ++k) {
        const int own = __builtin_amdgcn_readlane(own_key, k);
        int n = 0;
#pragma unroll
        for (int i = 0; i < kIds; ++i) n += key[i] < own;
        n = wave_total(n);
        if (lane == 0) s_part[wave][k] = own < 0 ? -1 : n;
    }
    __syncthreads();
    if (tid < top_k) {
        const int a = s_part[0][tid];
        const int pos = a < 0 ? -1 : a + s_part[1][tid] + s_part[2][tid] + s_part[3][tid];
        s_pos[tid] = pos;
        if (blockIdx.y == 0) {
            dst_of_route[t * top_k + tid] = pos;
            if (pos >= 0) src_route[pos] = t * top_k + tid;
        }
    }
    __syncthreads();
    for (int k = 0; k < top_k; ++k) {
        const int pos = s_pos[k];
        if (pos < 0) continue;
        uint16_t *out = rows + (size_t)pos * row_len;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = (u0 + tid + 256 * i) * kLen;
            if (u < row_len) store_any(out + min(u, row_len - kLen), v[i]);
        }
    }
}

// ---- sort of up to kSortOne routes in one launch.  Workgroup c places the routes of chunk c, whose ids it keeps
// in registers; it counts the experts of every other chunk itself (those before its own apart
// from those behind), so there is no scratch and no second launch.  A wave's 64 ids are
// counted by one ballot per bit of the id and one LDS add per distinct id.  Bound by latency: ids
// are asked for four loads at a time (800 routes of 64 experts: 5.0 us, 9.0 with a load at a time and the own chunk
// read three times).
constexpr int kChunk = 1024, kOwn = kChunk / 256;
constexpr int kSortOne = 4096;

// Lanes of the wave with the same live id as this one, of `bits` bits.
__device__ __forceinline__ uint64_t same_id(int e, int n_experts, int bits) {
    uint64_t grp = __ballot(live_id(e, n_experts));
    for (int b = 0; b < bits; ++b) {
        const uint64_t one = __ballot((e >> b) & 1);
        grp &= (e >> b) & 1 ? one : ~one;
    }
    return grp;
}

__device__ __forceinline__ void count_ids(int e, int n_experts, uint64_t grp, int *to) {
    const int lane = threadIdx.x & 63;
    if (live_id(e, n_experts) && lane == 63 - __builtin_clzll(grp)) atomicAdd(&to[e], __builtin_popcountll(grp));
}

// Route r (up to `end`) to its position, `next` of its wave and expert and the lanes before it.
__device__ __forceinline__ void place_id(int e, int n_experts, uint64_t grp, int r, int end, int *next,
                                         int32_t *__restrict__ src_route, int32_t *__restrict__ dst_of_route) {
    const int lane = threadIdx.x & 63;
    const bool live = live_id(e, n_experts);
    int pos = -1;
    if (live) {
        pos = next[e] + __builtin_popcountll(grp & ((1ull << lane) - 1ull));
        src_route[pos] = r;
    }
    if (r < end) dst_of_route[r] = pos;
    if (live && lane == 63 - __builtin_clzll(grp)) next[e] = pos + 1;  // after every lane's read: one wave
}

__device__ __forceinline__ void sort_chunk(int chunk, const int32_t *__restrict__ ids, int R, int n_experts,
                                           int32_t *__restrict__ offsets, int32_t *__restrict__ src_route,
                                           int32_t *__restrict__ dst_of_route) {
    __shared__ int s_all[1024], s_other[2][1024];  // other chunks: before this one, behind it
    __shared__ int s_wave[4][1024];  // the chunk's routes per wave, then each wave's next position
    __shared__ int s_part[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bits = 32 - __builtin_clz(n_experts);
    // 256 routes from r0 on, 64 at a time
    auto load = [&](int r0, int (&e)[kOwn]) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int r = r0 + 64 * i + lane;
            e[i] = r < R ? ids[r] : -1;
        }
    };
    int own[kOwn], *const mine = s_wave[wave];
    const int w0 = chunk * kChunk + 256 * wave;
    load(w0, own);
    for (int e = tid; e < n_experts; e += 256) {
        s_other[0][e] = s_other[1][e] = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) s_wave[w][e] = 0;
    }
    __syncthreads();
    uint64_t grp[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        grp[i] = same_id(own[i], n_experts, bits);
        count_ids(own[i], n_experts, grp[i], mine);
    }
    for (int r0 = 256 * wave; r0 < R; r0 += kChunk) {
        if (r0 == w0) continue;
        int e[kOwn];
        load(r0, e);
#pragma unroll
        for (int i = 0; i < kOwn; ++i) count_ids(e[i], n_experts, same_id(e[i], n_experts, bits), s_other[r0 > w0]);
    }
    __syncthreads();
    for (int e = tid; e < 1024; e += 256) {
        int n = 0;
        if (e < n_experts) {
            n = s_other[0][e] + s_other[1][e];
#pragma unroll
            for (int w = 0; w < 4; ++w) n += s_wave[w][e];
        }
        s_all[e] = n;
    }
    __syncthreads();
    const int last = s_all[n_experts - 1];
    expert_bases(s_all, s_part);
    if (chunk == 0) {
        for (int e = tid; e < n_experts; e += 256) offsets[e] = s_all[e];
        if (tid == 0) offsets[n_experts] = s_all[n_experts - 1] + last;
    }
    for (int e = tid; e < n_experts; e += 256) {
        int base = s_all[e] + s_other[0][e];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int n = s_wave[w][e];
            s_wave[w][e] = base;
            base += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
        place_id(own[i], n_experts, grp[i], w0 + 64 * i + lane, R, mine, src_route, dst_of_route);
}

// ---- sort of many routes, in three launches, linear in their number.  dst_of_route is the scratch: a
// chunk's part of it (at least kChunk entries, as many as there can be experts; the last chunk is up
// to twice as long) holds the chunk's counts, then its first positions, then its results.

__global__ __launch_bounds__(256) void sort_count_kernel(const int32_t *__restrict__ ids, int R, int n_experts,
                                                         int chunks, int32_t *__restrict__ dst_of_route) {
    __shared__ int s_cnt[1024];
    for (int e = threadIdx.x; e < n_experts; e += 256) s_cnt[e] = 0;
    __syncthreads();
    const int beg = blockIdx.x * kChunk, end = (int)blockIdx.x == chunks - 1 ? R : beg + kChunk;
    for (int r0 = beg; r0 < end; r0 += 1024) {
        int e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + 256 * i + threadIdx.x;
            e[i] = r < end ? ids[r] : -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (live_id(e[i], n_experts)) atomicAdd(&s_cnt[e[i]], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_experts; e += 256) dst_of_route[beg + e] = s_cnt[e];
}

// One workgroup: counts to first positions.  Thread (g, e) has expert e in the g-th part of the chunks;
// eight loads in flight.
__global__ __launch_bounds__(1024) void sort_scan_kernel(int n_experts, int wide, int chunks,
                                                         int32_t *__restrict__ dst_of_route,
                                                         int32_t *__restrict__ offsets) {
    constexpr int kAhead = 8;
    __shared__ int s_sum[1024], s_base[1024], s_part[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int e = tid % wide, g = tid / wide, groups = 1024 / wide;  // wide: n_experts up to a power of two, at least 16
    const int beg = (int)((int64_t)chunks * g / groups);
    const int end = e < n_experts ? (int)((int64_t)chunks * (g + 1) / groups) : beg;
    int32_t *const at = dst_of_route + e;
    int sum = 0;
    for (int i = beg; i < end; i += kAhead) {
        int v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = i + k < end ? at[(size_t)(i + k) * kChunk] : 0;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) sum += v[k];
    }
    s_sum[tid] = sum;
    __syncthreads();
    int before = 0, total = 0;  // of expert e: in the groups before this one, in all
    for (int k = 0; k < groups; ++k) {
        const int v = s_sum[k * wide + e];
        if (k < g) before += v;
        total += v;
    }
    // exclusive sum of the totals over the experts: the first `wide` threads
    int incl = tid < wide ? total : 0;
    const int mine = incl;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 63) s_part[wave] = incl;
    __syncthreads();
    int base = incl - mine;
    for (int w = 0; w < wave; ++w) base += s_part[w];
    if (tid < wide) s_base[tid] = base;
    if (tid < n_experts) offsets[tid] = base;
    if (tid == n_experts - 1) offsets[n_experts] = base + mine;
    __syncthreads();
    int pos = s_base[e] + before;
    for (int i = beg; i < end; i += kAhead) {
        int v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = i + k < end ? at[(size_t)(i + k) * kChunk] : 0;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (i + k < end) at[(size_t)(i + k) * kChunk] = pos;
            pos += v[k];
        }
    }
}

__global__ __launch_bounds__(256) void sort_place_kernel(const int32_t *__restrict__ ids, int R, int n_experts,
                                                         int chunks, int32_t *__restrict__ src_route,
                                                         int32_t *__restrict__ dst_of_route) {
    __shared__ int s_base[1024];
    __shared__ int s_wave[4][1024];  // 1024 routes' counts per wave, then each wave's next position
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bits = 32 - __builtin_clz(n_experts);
    const int beg = blockIdx.x * kChunk, end = (int)blockIdx.x == chunks - 1 ? R : beg + kChunk;
    for (int e = tid; e < n_experts; e += 256) s_base[e] = dst_of_route[beg + e];
    for (int r0 = beg; r0 < end; r0 += kChunk) {
        for (int e = tid; e < n_experts; e += 256) {
#pragma unroll
            for (int w = 0; w < 4; ++w) s_wave[w][e] = 0;
        }
        int own[kOwn], *const mine = s_wave[wave];
        uint64_t grp[kOwn];
        const int w0 = r0 + 256 * wave;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int r = w0 + 64 * i + lane;
            own[i] = r < end ? ids[r] : -1;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            grp[i] = same_id(own[i], n_experts, bits);
            count_ids(own[i], n_experts, grp[i], mine);
        }
        __syncthreads();
        for (int e = tid; e < n_experts; e += 256) {
            int base = s_base[e];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int n = s_wave[w][e];
                s_wave[w][e] = base;
                base += n;
            }
            s_base[e] = base;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            place_id(own[i], n_experts, grp[i], w0 + 64 * i + lane, end, mine, src_route, dst_of_route);
        __syncthreads();  // the counts are cleared
    }
}

// The sort and the quantizer of x (n8 groups of eight values) in one launch: neither needs the other.
template <class T>
__global__ __launch_bounds__(256) void sort_quantize_kernel(const int32_t *__restrict__ ids, int R, int n_experts,
                                                            int32_t *__restrict__ offsets,
                                                            int32_t *__restrict__ src_route,
                                                            int32_t *__restrict__ dst_of_route, int chunks,
                                                            const T *__restrict__ x, int64_t n8,
                                                            uint8_t *__restrict__ xq) {
    if ((int)blockIdx.x < chunks) {
        sort_chunk(blockIdx.x, ids, R, n_experts, offsets, src_route, dst_of_route);
        return;
    }
    const int64_t i = (int64_t)(blockIdx.x - chunks) * 256 + threadIdx.x;
    if (i < n8) mx_quantize8(x + 8 * i, i, n8, xq);
}

// Few routes: workgroup 0 selects every token's experts (a wave per token) and places the routes, each
// thread counting those before its own; the other workgroups quantize x meanwhile.
constexpr int kRouteOne = 512;

template <class T, int PER>
__global__ __launch_bounds__(1024) void route_quantize_kernel(const float *__restrict__ logits, int num_tokens,
                                                              int num_experts, int top_k, float *__restrict__ route_w,
                                                              int32_t *__restrict__ ids, int32_t *__restrict__ offsets,
                                                              int32_t *__restrict__ src_route,
                                                              int32_t *__restrict__ dst_of_route,
                                                              const T *__restrict__ x, int64_t n8,
                                                              uint8_t *__restrict__ xq) {
    if (blockIdx.x > 0) {
        const int64_t i = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x;
        if (i < n8) mx_quantize8(x + 8 * i, i, n8, xq);
        return;
    }
    __shared__ int s_ids[kRouteOne];
    __shared__ float s_w[kRouteOne];
    const int R = num_tokens * top_k, tid = threadIdx.x, wave = tid >> 6;
    for (int t = wave; t < num_tokens; t += 16)
        top_k_token<PER>(logits + (size_t)t * num_experts, num_experts, top_k, s_w + t * top_k, s_ids + t * top_k,
                         tid & 63);
    __syncthreads();
    // Threads 0..511: the routes; 512..: the experts' offsets.
    if (tid < R) {
        const int e = s_ids[tid];
        int pos = 0;
        for (int j = 0; j < R; ++j) {
            const int o = s_ids[j];
            pos += (o < e) | ((o == e) & (j < tid));
        }
        dst_of_route[tid] = pos;
        src_route[pos] = tid;
        route_w[tid] = s_w[tid];
        ids[tid] = e;
    }
    for (int e = tid - kRouteOne; e <= num_experts; e += 512) {
        if (e < 0) break;
        int c = 0;
        for (int j = 0; j < R; ++j) c += s_ids[j] < e;
        offsets[e] = c;
    }
}

// Threads of a workgroup that share a row of `pieces`: up to a power of two, so that short rows
// leave none idle (32768 tokens of 64 values, 8 routes each: the combine 9.0 us, 35.7 with a workgroup a row).
inline int log2_threads(int pieces) {
    int n = 0;
    while (n < 8 && (1 << n) < pieces) ++n;
    return n;
}

// rows[dst(t, k)] = x[t], a thread per piece of a token's row.
template <class U, bool PACKED>
__global__ __launch_bounds__(256) void scatter_rows_kernel(const uint16_t *__restrict__ x,
                                                           const int32_t *__restrict__ dst_of_route, int T, int top_k,
                                                           int row_len, int log2_row, uint16_t *__restrict__ rows) {
    constexpr int kLen = sizeof(U) / 2;
    const int R = T * top_k;
    // A row a workgroup (the usual case): t is a scalar, and so are the rows' addresses.
    const int t = PACKED ? (blockIdx.x * 256 + threadIdx.x) >> log2_row : blockIdx.x;
    int u = (PACKED ? threadIdx.x & ((1 << log2_row) - 1) : blockIdx.y * 256 + threadIdx.x) * kLen;
    if (t >= T || u >= row_len) return;
    u = min(u, row_len - kLen);
    const U v = load_any<U>(x + (size_t)t * row_len + u);
    for (int k = 0; k < top_k; ++k) {
        const int pos = dst_of_route[t * top_k + k];
        if ((unsigned)pos < (unsigned)R) store_any(rows + (size_t)pos * row_len + u, v);
    }
}

// ---- sums over a token's routes (combine; the dispatch's gradient without weights)
template <class TI, class TO, int VEC, bool WEIGHTED, int SLICES, bool PACKED>
__global__ __launch_bounds__(256) void join_rows_kernel(const TI *__restrict__ rows,
                                                        const int32_t *__restrict__ dst_of_route,
                                                        const float *__restrict__ weights, int T, int top_k, int H,
                                                        int log2_row, TO *__restrict__ y) {
    const int t = PACKED ? (blockIdx.x * 256 + threadIdx.x) >> log2_row : blockIdx.x, R = T * top_k;
    int h = (PACKED ? threadIdx.x & ((1 << log2_row) - 1) : blockIdx.y * 256 + threadIdx.x) * VEC;
    if (t >= T || h >= H) return;
    h = min(h, H - VEC);
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    for (int k0 = 0; k0 < top_k; k0 += 4) {
        MxVec<TI, VEC> v[4], v2[SLICES == 2 ? 4 : 1];
        int pos[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            pos[j] = k0 + j < top_k ? dst_of_route[t * top_k + k0 + j] : -1;
            if ((unsigned)pos[j] < (unsigned)R)
                v[j] = load_any<MxVec<TI, VEC>>(rows + (size_t)pos[j] * H + h);
            if (SLICES == 2 && (unsigned)pos[j] < (unsigned)R)
                v2[SLICES == 2 ? j : 0] = load_any<MxVec<TI, VEC>>(rows + ((size_t)R + pos[j]) * H + h);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((unsigned)pos[j] < (unsigned)R) {
                const float w = WEIGHTED ? weights[t * top_k + k0 + j] : 1.0f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float e = (float)v[j].v[i];
                    if constexpr (SLICES == 2) e += (float)v2[j].v[i];
                    acc[i] = fmaf(w, e, acc[i]);
                }
            }
    }
    MxVec<TO, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = (TO)acc[i];
    store_any(y + (size_t)t * H + h, o);
}

// A piece of a route's row: its gradient stored, its part of the dot product added.
template <class T, int VEC>
__device__ __forceinline__ float backward_piece(const T *__restrict__ g, const T *__restrict__ e, T *__restrict__ ge,
                                                float w, int h0, int H, float dot) {
    const int h = min(h0, H - VEC);
    const MxVec<T, VEC> gv = load_any<MxVec<T, VEC>>(g + h), ev = load_any<MxVec<T, VEC>>(e + h);
    MxVec<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        // What the last piece shares with the one before is counted there.
        dot = fmaf(h + i >= h0 ? (float)gv.v[i] : 0.0f, h + i >= h0 ? (float)ev.v[i] : 0.0f, dot);
        o.v[i] = (T)(w * (float)gv.v[i]);
    }
    store_any(ge + h, o);
    return dot;
}

// ---- gradients of the combine: a workgroup per token, its gradient row read once per route
// from the cache, the routes' dot products reduced in a fixed order.
template <class T, int VEC>
__global__ __launch_bounds__(256) void combine_rows_backward_kernel(
    const T *__restrict__ grad_y, const T *__restrict__ rows, const int32_t *__restrict__ dst_of_route,
    const float *__restrict__ weights, int R, int top_k, int H, T *__restrict__ grad_rows,
    float *__restrict__ grad_weights) {
    __shared__ float s_dot[32][4];
    const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *g = grad_y + (size_t)t * H;
    for (int k = 0; k < top_k; ++k) {
        const int pos = dst_of_route[t * top_k + k];
        float dot = 0.0f;
        if ((unsigned)pos < (unsigned)R) {
            const float w = weights[t * top_k + k];
            const T *e = rows + (size_t)pos * H;
            T *ge = grad_rows + (size_t)pos * H;
            for (int h0 = threadIdx.x * VEC; h0 < H; h0 += 256 * VEC)
                dot = backward_piece<T, VEC>(g, e, ge, w, h0, H, dot);
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
        if (lane == 0) s_dot[k][wave] = dot;
    }
    __syncthreads();
    if (threadIdx.x < top_k) {
        const float *d = s_dot[threadIdx.x];
        grad_weights[t * top_k + threadIdx.x] = (d[0] + d[1]) + (d[2] + d[3]);
    }
}

// The same for short rows: 2^log2_row lanes of a wave to a route, so that none of a workgroup's waves is idle
// (8192 tokens top-8 of 300 bf16 values: 21 us, 32 with a workgroup a token).
template <class T, int VEC>
__global__ __launch_bounds__(256) void combine_rows_backward_short_kernel(
    const T *__restrict__ grad_y, const T *__restrict__ rows, const int32_t *__restrict__ dst_of_route,
    const float *__restrict__ weights, int R, int top_k, int H, int log2_row, T *__restrict__ grad_rows,
    float *__restrict__ grad_weights) {
    const int r = (int)(((int64_t)blockIdx.x * 256 + threadIdx.x) >> log2_row);
    const int len = 1 << log2_row, lane = threadIdx.x & (len - 1);
    const int pos = r < R ? dst_of_route[r] : -1;
    float dot = 0.0f;
    if ((unsigned)pos < (unsigned)R) {
        const float w = weights[r];
        const T *g = grad_y + (size_t)(r / top_k) * H, *e = rows + (size_t)pos * H;
        T *ge = grad_rows + (size_t)pos * H;
        for (int h0 = lane * VEC; h0 < H; h0 += len * VEC) dot = backward_piece<T, VEC>(g, e, ge, w, h0, H, dot);
    }
    for (int d = len / 2; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
    if (r < R && lane == 0) grad_weights[r] = dot;
}

template <class U>
hipError_t run_dispatch(const int32_t *ids, const void *x, int T, int top_k, size_t row_bytes, int E, int32_t *offsets,
                        int32_t *src_route, int32_t *dst_of_route, void *rows, hipStream_t stream) {
    const int R = T * top_k, row_len = (int)(row_bytes / 2), units = (int)((row_bytes + sizeof(U) - 1) / sizeof(U));
    if (R <= kSortMax) {
        const dim3 grid((unsigned)T + 1, (unsigned)((units + 1023) / 1024));
        hipLaunchKernelGGL(dispatch_rows_kernel<U>, grid, dim3(256), 0, stream, ids, (const uint16_t *)x, R, top_k,
                           row_len, E, offsets, src_route, dst_of_route, (uint16_t *)rows);
        return hipGetLastError();
    }
    const hipError_t e = launch_moe_sort(ids, R, E, offsets, src_route, dst_of_route, stream);
    if (e != hipSuccess) return e;
    const int log2_row = log2_threads(units), tokens = 256 >> log2_row;
    const dim3 grid((unsigned)((T + tokens - 1) / tokens), (unsigned)((units + 255) / 256));
    if (log2_row == 8)
        hipLaunchKernelGGL((scatter_rows_kernel<U, false>), grid, dim3(256), 0, stream, (const uint16_t *)x,
                           dst_of_route, T, top_k, row_len, log2_row, (uint16_t *)rows);
    else
        hipLaunchKernelGGL((scatter_rows_kernel<U, true>), grid, dim3(256), 0, stream, (const uint16_t *)x,
                           dst_of_route, T, top_k, row_len, log2_row, (uint16_t *)rows);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_sort(const int32_t *ids, int n_routes, int n_experts, int32_t *offsets, int32_t *src_route,
                           int32_t *dst_of_route, hipStream_t stream) {
    const int chunks = n_routes / kChunk;
    int wide = 16;
    while (wide < n_experts) wide *= 2;
    hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)chunks), dim3(256), 0, stream, ids, n_routes, n_experts,
                       chunks, dst_of_route);
    hipLaunchKernelGGL(sort_scan_kernel, dim3(1), dim3(1024), 0, stream, n_experts, wide, chunks, dst_of_route,
                       offsets);
    hipLaunchKernelGGL(sort_place_kernel, dim3((unsigned)chunks), dim3(256), 0, stream, ids, n_routes, n_experts,
                       chunks, src_route, dst_of_route);
    return hipGetLastError();
}

hipError_t launch_mxfp4_route(const void *x, int dtype, const float *logits, int T, int H, int E, int top_k,
                              float *route_w, int32_t *ids, int32_t *offsets, int32_t *src_route,
                              int32_t *dst_of_route, void *xq, hipStream_t stream) {
    const int R = T * top_k;
    const int64_t n8 = (int64_t)T * (H / 8);
    if (n8 > kMxMaxGroups) return hipErrorInvalidConfiguration;
    return mx_by_dtype(dtype, [&](auto tag) {
        using X = typename decltype(tag)::type;
        if (R <= kRouteOne) {
            const dim3 grid((unsigned)(1 + (n8 + 1023) / 1024));
            auto go = [&](auto per) {
                hipLaunchKernelGGL((route_quantize_kernel<X, decltype(per)::value>), grid, dim3(1024), 0, stream, logits,
                                   T, E, top_k, route_w, ids, offsets, src_route, dst_of_route, (const X *)x, n8,
                                   (uint8_t *)xq);
                return hipGetLastError();
            };
            if (E <= 64) return go(std::integral_constant<int, 1>{});
            if (E <= 256) return go(std::integral_constant<int, 4>{});
            return go(std::integral_constant<int, 16>{});
        }
        const hipError_t e = launch_moe_top_k(logits, route_w, ids, T, E, top_k, stream);
        if (e != hipSuccess) return e;
        if (R > kSortOne) {
            const hipError_t q = launch_quantize_mxfp4(x, dtype, H, xq, T, H, stream);
            return q != hipSuccess ? q : launch_moe_sort(ids, R, E, offsets, src_route, dst_of_route, stream);
        }
        const int chunks = (R + kChunk - 1) / kChunk;
        hipLaunchKernelGGL(sort_quantize_kernel<X>, dim3((unsigned)(chunks + (n8 + 255) / 256)), dim3(256), 0, stream,
                           ids, R, E, offsets, src_route, dst_of_route, chunks, (const X *)x, n8, (uint8_t *)xq);
        return hipGetLastError();
    });
}

hipError_t launch_moe_dispatch_rows(const int32_t *ids, const void *x, int elem_bytes, int T, int top_k, int H, int E,
                                    int32_t *offsets, int32_t *src_route, int32_t *dst_of_route, void *rows,
                                    hipStream_t stream) {
    const size_t bytes = (size_t)H * elem_bytes;
    return bytes >= 16
               ? run_dispatch<uint4>(ids, x, T, top_k, bytes, E, offsets, src_route, dst_of_route, rows, stream)
               : run_dispatch<uint16_t>(ids, x, T, top_k, bytes, E, offsets, src_route, dst_of_route, rows, stream);
}

namespace {
template <class TI, class TO, int VEC, bool PACKED>
hipError_t run_join(const void *rows, const int32_t *dst, const float *weights, void *y, int T, int H, int top_k,
                    hipStream_t stream, int slices) {
    const int pieces = (H + VEC - 1) / VEC, log2_row = log2_threads(pieces), tokens = 256 >> log2_row;
    const dim3 grid((unsigned)((T + tokens - 1) / tokens), (unsigned)((pieces + 255) / 256));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, (const TI *)rows, dst, weights, T, top_k, H, log2_row,
                           (TO *)y);
        return hipGetLastError();
    };
    if (slices == 2) {
        if constexpr (sizeof(TI) == 4 && VEC == 4)  // the FFN's: H % 32 == 0
            return go(join_rows_kernel<TI, TO, VEC, true, 2, PACKED>);
        return hipErrorInvalidValue;
    }
    return weights != nullptr ? go(join_rows_kernel<TI, TO, VEC, true, 1, PACKED>)
                              : go(join_rows_kernel<TI, TO, VEC, false, 1, PACKED>);
}

template <class TI, class TO, int VEC>
hipError_t run_join_rows(const void *rows, const int32_t *dst, const float *weights, void *y, int T, int H, int top_k,
                         hipStream_t stream, int slices) {
    return H > 128 * VEC ? run_join<TI, TO, VEC, false>(rows, dst, weights, y, T, H, top_k, stream, slices)
                         : run_join<TI, TO, VEC, true>(rows, dst, weights, y, T, H, top_k, stream, slices);
}

template <class TI, class TO>
hipError_t run_join_types(const void *rows, const int32_t *dst, const float *weights, void *y, int T, int H, int top_k,
                          hipStream_t stream, int slices) {
    constexpr int kWide = 16 / sizeof(TI);
    return H >= kWide ? run_join_rows<TI, TO, kWide>(rows, dst, weights, y, T, H, top_k, stream, slices)
                      : run_join_rows<TI, TO, 1>(rows, dst, weights, y, T, H, top_k, stream, slices);
}
}  // namespace

hipError_t launch_moe_join_rows(const void *rows, int rows_dtype, const int32_t *dst_of_route, const float *weights,
                                void *y, int dtype, int T, int H, int top_k, hipStream_t stream, int slices) {
    return mx_by_dtype(rows_dtype, [&](auto in) {
        using TI = typename decltype(in)::type;
        if (rows_dtype == dtype)
            return run_join_types<TI, TI>(rows, dst_of_route, weights, y, T, H, top_k, stream, slices);
        if (rows_dtype != JJO_DTYPE_F32) return hipErrorInvalidValue;
        return dtype == JJO_DTYPE_F16
                   ? run_join_types<float, _Float16>(rows, dst_of_route, weights, y, T, H, top_k, stream, slices)
                   : run_join_types<float, __bf16>(rows, dst_of_route, weights, y, T, H, top_k, stream, slices);
    });
}

hipError_t launch_moe_combine_rows_backward(const void *grad_y, const void *rows, int dtype,
                                            const int32_t *dst_of_route, const float *weights, void *grad_rows,
                                            float *grad_weights, int T, int H, int top_k, hipStream_t stream) {
    return mx_by_dtype(dtype, [&](auto tag) {
        using E = typename decltype(tag)::type;
        constexpr int kWide = 16 / sizeof(E);
        auto run = [&](auto vec) {
            constexpr int V = decltype(vec)::value;
            const int log2_row = std::min(log2_threads((H + V - 1) / V), 6), routes = 256 >> log2_row;
            const int64_t groups = ((int64_t)T * top_k + routes - 1) / routes;
            // (A grid has fewer than 2^32 threads: 2^26 routes of 64 lanes go by tokens.)
            if (H <= 128 * V && groups * 256 < 1LL << 32) {
                hipLaunchKernelGGL((combine_rows_backward_short_kernel<E, V>), dim3((unsigned)groups), dim3(256), 0,
                                   stream, (const E *)grad_y, (const E *)rows, dst_of_route, weights, T * top_k, top_k,
                                   H, log2_row, (E *)grad_rows, grad_weights);
                return hipGetLastError();
            }
            hipLaunchKernelGGL((combine_rows_backward_kernel<E, V>), dim3((unsigned)T), dim3(256), 0, stream,
                               (const E *)grad_y, (const E *)rows, dst_of_route, weights, T * top_k, top_k, H,
                               (E *)grad_rows, grad_weights);
            return hipGetLastError();
        };
        return H >= kWide ? run(std::integral_constant<int, kWide>{}) : run(std::integral_constant<int, 1>{});
    });
}

}  // namespace jjo
