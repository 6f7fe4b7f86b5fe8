// Cache rows to and from their 8-bit forms (row_format.h).
//
// Per group of 32 values x with largest finite magnitude A the scale is 2^e,
// e = max(-127, ceil(log2(A / 448))), and the codes are e4m3(x / 2^e).  Both
// steps are exact but for the rounding to the code: A is one of the 16-bit
// values, so with A = m 2^E, 1 <= m < 2, and 448 = 1.75 * 2^8 the exponent is
// E - 8, plus one where m > 1.75; and the division is by a power of two.
//
// One wave per row.
#include "row_format.h"

namespace kvx {
namespace {

constexpr int kThreads = 256;
constexpr int kWavesPerBlock = kThreads / 64;

template <int DTYPE>
__device__ __forceinline__ float to_float(uint16_t bits)
{
    if constexpr (DTYPE == KVX_DTYPE_BF16) return __uint_as_float(static_cast<uint32_t>(bits) << 16);
    return static_cast<float>(__builtin_bit_cast(_Float16, bits));
}

// Magnitude bits of a finite value, 0 for an infinity or a NaN: ordered as the values are.
__device__ __forceinline__ uint32_t finite_bits(float x)
{
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return b >= 0x7F800000u ? 0u : b;
}

// Scale byte e + 127 of a group whose largest finite magnitude has these bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top)
{
    const int32_t e = static_cast<int32_t>(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < 0 ? 0u : static_cast<uint32_t>(e);
}

// 448 limits what only an infinity exceeds; the conversion would make it a NaN.
__device__ __forceinline__ float limit(float x) { return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f); }

template <int DTYPE, int QUANT>
__global__ __launch_bounds__(kThreads) void kvx_quantize_rows(RowCopyArgs a)
{
    using F = RowForm<QUANT>;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kWavesPerBlock + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u;
    if (row >= a.rows) return;
    int64_t to = static_cast<int64_t>(row);
    if (a.slots != 0) {
        to = hot_row(reinterpret_cast<const int32_t *>(a.slots)[row], row / a.perReq, a.reqStride, a.hotRows,
                     a.overflowSlot);
    }
    if (to < 0) return;
    const uint16_t *src = reinterpret_cast<const uint16_t *>(a.rows16 + row * a.rowStride);
    uint8_t *dst = reinterpret_cast<uint8_t *>(a.hot) + static_cast<uint64_t>(to) * F::bytes;
    // a lane takes a pair of values: 16 lanes a group, 4 groups at a time
    for (int c = 0; c < F::codes; c += 128) {
        const int at = c + static_cast<int>(lane) * 2;
        const bool in = at < F::codes;
        const float x0 = in ? to_float<DTYPE>(src[at]) : 0.0f, x1 = in ? to_float<DTYPE>(src[at + 1]) : 0.0f;
        uint32_t top = max(finite_bits(x0), finite_bits(x1));
        for (int d = 1; d < 16; d <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
        const uint32_t byte = scale_byte(top);
        const float inv = __uint_as_float((254u - byte) << 23);
        const int pair = __builtin_amdgcn_cvt_pk_fp8_f32(limit(x0 * inv), limit(x1 * inv), 0, false);
        if (in) {
            *reinterpret_cast<uint16_t *>(dst + at) = static_cast<uint16_t>(pair);
            if ((lane & 15u) == 0) dst[F::scaleAt + at / kGroup] = static_cast<uint8_t>(byte);
        }
    }
    for (int r = static_cast<int>(lane); r < F::raw; r += 64) {
        reinterpret_cast<uint16_t *>(dst + F::codes)[r] = src[F::codes + r];
    }
    for (int z = F::scaleAt + F::scales + static_cast<int>(lane); z < F::bytes; z += 64) dst[z] = 0;
}

template <int DTYPE, int QUANT, int OUT>
__global__ __launch_bounds__(kThreads) void kvx_dequantize_rows(RowCopyArgs a)
{
    using F = RowForm<QUANT>;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kWavesPerBlock + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    int64_t from = static_cast<int64_t>(row);
    if (a.slots != 0) {
        from = hot_row(reinterpret_cast<const int32_t *>(a.slots)[row], row / a.perReq, a.reqStride, a.hotRows,
                       a.overflowSlot);
    }
    const uint8_t *src = reinterpret_cast<const uint8_t *>(a.hot) + static_cast<uint64_t>(from) * F::bytes;
    for (int at = static_cast<int>(threadIdx.x & 63u); at < kDim; at += 64) {
        float x = 0.0f;
        if (from >= 0 && at < F::codes) {
            const uint32_t byte = src[F::scaleAt + at / kGroup];
            const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
            x = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(src[at]), 0) * scale;
        } else if (from >= 0) {
            x = to_float<DTYPE>(reinterpret_cast<const uint16_t *>(src + F::codes)[at - F::codes]);
        }
        if constexpr (OUT == KVX_DTYPE_FP32) {
            reinterpret_cast<float *>(a.rows16)[row * kDim + at] = x;
        } else if constexpr (OUT == KVX_DTYPE_BF16) {
            reinterpret_cast<__bf16 *>(a.rows16)[row * kDim + at] = static_cast<__bf16>(x);
        } else {
            reinterpret_cast<_Float16 *>(a.rows16)[row * kDim + at] = static_cast<_Float16>(x);
        }
    }
}

template <int DTYPE, int QUANT>
void dequantize(const RowCopyArgs &a, uint32_t outDtype, dim3 grid, hipStream_t stream)
{
    auto *kernel = outDtype == KVX_DTYPE_BF16   ? kvx_dequantize_rows<DTYPE, QUANT, KVX_DTYPE_BF16>
                   : outDtype == KVX_DTYPE_FP16 ? kvx_dequantize_rows<DTYPE, QUANT, KVX_DTYPE_FP16>
                                                : kvx_dequantize_rows<DTYPE, QUANT, KVX_DTYPE_FP32>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a);
}

dim3 row_grid(uint64_t rows) { return dim3(static_cast<uint32_t>((rows + kWavesPerBlock - 1) / kWavesPerBlock)); }

}  // namespace

hipError_t launch_quantize_rows(const RowCopyArgs &a, uint32_t dtype, uint32_t quant, hipStream_t stream)
{
    auto *kernel = dtype == KVX_DTYPE_BF16
                       ? (quant == KVX_QUANT_LATENT ? kvx_quantize_rows<KVX_DTYPE_BF16, KVX_QUANT_LATENT>
                                                    : kvx_quantize_rows<KVX_DTYPE_BF16, KVX_QUANT_ROW>)
                       : (quant == KVX_QUANT_LATENT ? kvx_quantize_rows<KVX_DTYPE_FP16, KVX_QUANT_LATENT>
                                                    : kvx_quantize_rows<KVX_DTYPE_FP16, KVX_QUANT_ROW>);
    hipLaunchKernelGGL(kernel, row_grid(a.rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_dequantize_rows(const RowCopyArgs &a, uint32_t dtype, uint32_t quant, uint32_t outDtype,
                                  hipStream_t stream)
{
    if (dtype == KVX_DTYPE_BF16) {
        if (quant == KVX_QUANT_LATENT) dequantize<KVX_DTYPE_BF16, KVX_QUANT_LATENT>(a, outDtype, row_grid(a.rows), stream);
        else dequantize<KVX_DTYPE_BF16, KVX_QUANT_ROW>(a, outDtype, row_grid(a.rows), stream);
    } else {
        if (quant == KVX_QUANT_LATENT) dequantize<KVX_DTYPE_FP16, KVX_QUANT_LATENT>(a, outDtype, row_grid(a.rows), stream);
        else dequantize<KVX_DTYPE_FP16, KVX_QUANT_ROW>(a, outDtype, row_grid(a.rows), stream);
    }
    return hipGetLastError();
}

}  // namespace kvx
