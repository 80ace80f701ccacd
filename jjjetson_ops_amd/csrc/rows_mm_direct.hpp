// Products of float matrices with few rows on the right (a decoded token, a small batch, experts with a few
// rows): the weights go from memory straight to the matrix instruction's operand registers.
//
// A workgroup has 16 weight rows (SwiGLU: of gate and of up), a wave of it every kWaves-th run of kSteps steps along
// K; a lane loads 16 bytes of a row a step (four lanes 64 contiguous bytes of each of 16 rows, the next step the other
// half of the line), and the same of up to 16 rows of x, which the caches hold.  The loads of the next
// run are in flight while this one is multiplied.  The waves' sums are added through LDS in their
// order and leave through the epilogue eight columns a thread.  Any K and alignment: a lane's piece that
// reaches behind the row's end is taken element by element.
//
// Bound by reading the weights.
#pragma once

#include "rows_mm_tile.hpp"

namespace jjo {
namespace {

template <class E, bool SWIGLU>
__global__ __launch_bounds__(512) void rows_direct_kernel(RowsMm p) {
    typedef typename E::type T;
    constexpr int kMats = SWIGLU ? 2 : 1;  // gate and up
    constexpr int kPiece = 16 / sizeof(T), kStep = 4 * kPiece, kSteps = 4;  // a step: 64 bytes of a row
    constexpr int kPitch = 16 * kMats + 4;
    extern __shared__ __align__(16) float sums[];  // [waves][16][kPitch]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6, r16 = lane & 15, q4 = lane >> 4;

    // Row tiles fastest: the workgroups that read the same weights follow each other on one XCD.
    const int total = gridDim.x, per = total / 8, rest = total % 8, xcd = blockIdx.x % 8;
    const int tile = xcd * per + min(xcd, rest) + (int)(blockIdx.x / 8), tile_q = tile % p.tiles_q;
    int expert = 0, q0 = tile_q * 16, end = p.Q;
    if (p.offsets != nullptr && !mx_expert_tile(p.offsets, p.n_experts, p.M, 16, tile_q, expert, q0, end)) return;
    const int p0 = tile / p.tiles_q * 16;

    const T *wrow[kMats];
    f32x4v acc[kMats];
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
        const T *const matrix = (const T *)(m == 0 ? p.p : p.p2) + expert * p.expert_stride;
        wrow[m] = matrix + min(p0 + r16, p.P - 1) * p.ldp + q4 * kPiece;
        acc[m] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }
    const T *const xrow = (const T *)p.q + min(q0 + r16, end - 1) * p.ldq + q4 * kPiece;

    // Run r of a wave: steps kSteps * (wave + waves * r) on.  Whole steps only, then the rest of the row.
    const int whole = p.K / kStep, runs = whole / kSteps;
    u32x4v w[2][kSteps][kMats], x[2][kSteps];
    auto load = [&](int run, auto buffer) {
        constexpr int B = decltype(buffer)::value;
        const int64_t k = (int64_t)run * kSteps * kStep;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int m = 0; m < kMats; ++m) w[B][s][m] = load_any<u32x4v>(wrow[m] + k + s * kStep);
            x[B][s] = load_any<u32x4v>(xrow + k + s * kStep);
        }
    };
    auto multiply = [&](auto buffer) {
        constexpr int B = decltype(buffer)::value;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int m = 0; m < kMats; ++m) acc[m] = rows_mfma<T>(w[B][s][m], x[B][s], acc[m]);
    };
    constexpr std::integral_constant<int, 0> kB0{};
    constexpr std::integral_constant<int, 1> kB1{};
    int run = wave;
    if (run < runs) load(run, kB0);
    for (; run < runs; run += 2 * waves) {
        if (run + waves < runs) load(run + waves, kB1);
        multiply(kB0);
        if (run + waves < runs) {
            if (run + 2 * waves < runs) load(run + 2 * waves, kB0);
            multiply(kB1);
        }
    }
    // The steps behind the last run, and the piece of a row behind the last step.
    for (int s = runs * kSteps + wave; s * kStep < p.K; s += waves) {
        const int64_t k = (int64_t)s * kStep;
        const int have = p.K - (int)k - q4 * kPiece;  // elements of this lane's piece
        auto piece = [&](const T *row) {
            u32x4v v{0u, 0u, 0u, 0u};
            if (have >= kPiece) {
                v = load_any<u32x4v>(row + k);
            } else if (have > 0) {
                MxVec<T, kPiece> e;
#pragma unroll
                for (int j = 0; j < kPiece; ++j) e.v[j] = j < have ? row[k + j] : (T)0.0f;
                v = __builtin_bit_cast(u32x4v, e);
            }
            return v;
        };
        const u32x4v b = piece(xrow);
#pragma unroll
        for (int m = 0; m < kMats; ++m) acc[m] = rows_mfma<T>(piece(wrow[m]), b, acc[m]);
    }

#pragma unroll
    for (int m = 0; m < kMats; ++m)
        *reinterpret_cast<f32x4v *>(sums + (wave * 16 + r16) * kPitch + 16 * m + 4 * q4) = acc[m];
    __syncthreads();
    for (int i = threadIdx.x; i < 32; i += blockDim.x) {  // 16 rows of two chunks of eight columns
        const int r = i / 2, chunk = i % 2, col = p0 + 8 * chunk, n = min(8, p.P - col);
        if (q0 + r >= end || n <= 0) continue;
        float v[8], up[8];
        auto take = [&](float *to, int at) {
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j] = 0.0f;
            for (int k = 0; k < waves; ++k) {
                const f32x4v *const from = reinterpret_cast<const f32x4v *>(sums + (k * 16 + r) * kPitch + at);
                const f32x4v a = from[0], b = from[1];
#pragma unroll
                for (int j = 0; j < 4; ++j) to[j] += a[j], to[4 + j] += b[j];
            }
        };
        take(v, 8 * chunk);
        if constexpr (SWIGLU) {
            take(up, 16 + 8 * chunk);
            rows_finish_swiglu<T>(p.epi, v, up, q0 + r, col, n, p.P, p.y);
        } else {
            rows_finish<T>(p.epi, v, q0 + r, col, n, p.P, p.y, p.ldy, false);
        }
    }
}

template <class E, bool SWIGLU>
hipError_t run_rows_direct(RowsMm p, int waves, hipStream_t stream) {
    const int tiles_p = (p.P + 15) / 16;
    p.tiles_q = (p.Q + 15) / 16 + (p.offsets != nullptr ? std::min(p.n_experts, p.M) : 0);
    const int64_t wgs = (int64_t)tiles_p * p.tiles_q;
    if (wgs * waves * 64 >= 1LL << 32) return hipErrorInvalidConfiguration;
    const auto kernel = rows_direct_kernel<E, SWIGLU>;
    const size_t lds = (size_t)waves * 16 * (SWIGLU ? 36 : 20) * sizeof(float);
    const hipError_t e = ensure_dynamic_lds((const void *)kernel, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(waves * 64), lds, stream, p);
    return hipGetLastError();
}

}  // namespace
}  // namespace jjo
