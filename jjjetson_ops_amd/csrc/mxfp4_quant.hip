// fp32 / fp16 / bf16 rows <-> MXFP4 on gfx950.
//
// Per block of 32: m = max|x|, scale 2^(floor(log2 m) - 2), codes = x / scale rounded to
// nearest even and limited to 6 (the OCP microscaling conversion).  Scale and division are
// exact (powers of two), so the bytes do not depend on how the work is cut.
//
// Bound by HBM: a value is read once (2 or 4 bytes) and 17/32 bytes are written.  A thread
// takes eight values, one 16-byte load (two for fp32), a quad of lanes one block: the block's
// maximum is two DPP steps and a wave stores 256 contiguous bytes of codes.  Both planes of
// contiguous rows are flat runs, so no thread divides; strided rows pay one division.
#include <hip/hip_runtime.h>

#include "mxfp4_common.hpp"

namespace jjo {
namespace {

// n8: groups of eight values in all, per_row of them in a row.
template <class T, bool STRIDED>
__global__ __launch_bounds__(256) void quantize_mxfp4_kernel(const T *__restrict__ x, int64_t row_stride,
                                                             int64_t per_row, int64_t n8, uint8_t *__restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;  // n8 % 4 == 0: quads leave as a whole
    const T *p = x + 8 * i;
    if constexpr (STRIDED) p = x + (i / per_row) * row_stride + 8 * (i % per_row);
    mx_quantize8(p, i, n8, out);
}

template <class T, bool STRIDED>
__global__ __launch_bounds__(256) void dequantize_mxfp4_kernel(const uint8_t *__restrict__ q, int64_t row_stride,
                                                               int64_t per_row, int64_t n8, T *__restrict__ y) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;
    const uint32_t c = reinterpret_cast<const uint32_t *>(q)[i];
    const uint32_t s = q[4 * n8 + (i >> 2)];
    // The product of an e2m1 value and a power of two is exact in fp32 (or subnormal, or
    // above its range at s = 253, 254).
    const float sc = s == 255u ? __uint_as_float(0x7fc00000u) : mx_scale_value(s);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t n = c >> (4 * k), m = n & 7u;
        // e2m1 bits to fp32: exponents 1..3 are 2^0..2^2, 0 and 1 the subnormals 0 and 0.5
        const uint32_t bits = m < 2u ? m * 0x3f000000u : 0x3f800000u + ((m - 2u) << 22);
        v[k] = __uint_as_float(bits | ((n & 8u) << 28)) * sc;
    }
    T *p = y + 8 * i;
    if constexpr (STRIDED) p = y + (i / per_row) * row_stride + 8 * (i % per_row);
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        MxVec<T, 8> o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.v[k] = (T)v[k];
        *reinterpret_cast<MxVec<T, 8> *>(p) = o;
    }
}

}  // namespace

hipError_t launch_quantize_mxfp4(const void *x, int dtype, int64_t row_stride, void *out, int64_t rows, int64_t cols,
                                 hipStream_t stream) {
    const int64_t n8 = rows * (cols / 8);
    if (n8 > kMxMaxGroups) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)((n8 + 255) / 256));
    return mx_by_dtype(dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (rows == 1 || row_stride == cols)
            hipLaunchKernelGGL((quantize_mxfp4_kernel<T, false>), grid, dim3(256), 0, stream, (const T *)x, row_stride,
                               cols / 8, n8, (uint8_t *)out);
        else
            hipLaunchKernelGGL((quantize_mxfp4_kernel<T, true>), grid, dim3(256), 0, stream, (const T *)x, row_stride,
                               cols / 8, n8, (uint8_t *)out);
        return hipGetLastError();
    });
}

hipError_t launch_dequantize_mxfp4(const void *q, void *y, int dtype, int64_t row_stride, int64_t rows, int64_t cols,
                                   hipStream_t stream) {
    const int64_t n8 = rows * (cols / 8);
    if (n8 > kMxMaxGroups) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)((n8 + 255) / 256));
    return mx_by_dtype(dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (rows == 1 || row_stride == cols)
            hipLaunchKernelGGL((dequantize_mxfp4_kernel<T, false>), grid, dim3(256), 0, stream, (const uint8_t *)q,
                               row_stride, cols / 8, n8, (T *)y);
        else
            hipLaunchKernelGGL((dequantize_mxfp4_kernel<T, true>), grid, dim3(256), 0, stream, (const uint8_t *)q,
                               row_stride, cols / 8, n8, (T *)y);
        return hipGetLastError();
    });
}

}  // namespace jjo
