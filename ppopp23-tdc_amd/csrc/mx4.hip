// Numbers into microscaled 4-bit floating point and back (format and layout: include/tdc.h).
//
// Memory traffic: x in, 17/32 byte a number out.  A thread takes one block of 32 numbers.
#include "ops_device.hpp"

namespace tdc {

template <int DT>
__global__ void __launch_bounds__(256) tdc_mx4_quantize_kernel(const void *x, long long rows, long long K, long long stride, long long blocks,
                                                           unsigned char *codes, unsigned char *scales) {
    using T = typename Num<DT>::type;
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    if (idx >= rows * blocks) return;
    const long long row = idx / blocks, kb = idx - row * blocks;
    const T *src = reinterpret_cast<const T *>(x) + row * stride + kb * 32;
    const int n = (int)max(0ll, min(32ll, K - kb * 32));
    float v[32], top = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        v[i] = i < n ? Num<DT>::up(src[i]) : 0.0f;
        top = larger(top, v[i]);
    }
    const int byte = mx4_scale_byte(top);
    const float scale = mx4_divisor(byte);
    *reinterpret_cast<uint4 *>(codes + idx * 16) =
        make_uint4(mx4_codes(v, scale), mx4_codes(v + 8, scale), mx4_codes(v + 16, scale), mx4_codes(v + 24, scale));
    scales[((kb >> 2) * rows + row) * 4 + (kb & 3)] = (unsigned char)byte;
}

template <int DT>
__global__ void __launch_bounds__(256) tdc_mx4_dequantize_kernel(const unsigned char *codes, const unsigned char *scales, long long rows,
                                                             long long K, long long blocks, void *y, long long stride) {
    using T = typename Num<DT>::type;
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    if (idx >= rows * blocks) return;
    const long long row = idx / blocks, kb = idx - row * blocks;
    const int n = (int)max(0ll, min(32ll, K - kb * 32));
    T *dst = reinterpret_cast<T *>(y) + row * stride + kb * 32;
    const float scale = mx4_scale(scales[((kb >> 2) * rows + row) * 4 + (kb & 3)]);
    const uint4 c = *reinterpret_cast<const uint4 *>(codes + idx * 16);
    const unsigned w[4] = {c.x, c.y, c.z, c.w};
    constexpr float value[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
    for (int i = 0; i < n; ++i) {
        const unsigned code = w[i >> 3] >> (4 * (i & 7));
        const float v = value[code & 7] * scale;
        dst[i] = Num<DT>::down(code & 8 ? -v : v);
    }
}

int launch_mx4_quantize(const void *x, int dtype, long long rows, long long K, long long stride, void *codes, void *scales, void *stream) {
    const long long blocks = mx4_padded(K) / 32;
    const unsigned grid = (unsigned)((rows * blocks + 255) / 256);
    const hipStream_t s = (hipStream_t)stream;
    auto *c = (unsigned char *)codes, *e = (unsigned char *)scales;
    if (dtype == TDC_F32) tdc_mx4_quantize_kernel<TDC_F32><<<grid, 256, 0, s>>>(x, rows, K, stride, blocks, c, e);
    else if (dtype == TDC_F16) tdc_mx4_quantize_kernel<TDC_F16><<<grid, 256, 0, s>>>(x, rows, K, stride, blocks, c, e);
    else tdc_mx4_quantize_kernel<TDC_BF16><<<grid, 256, 0, s>>>(x, rows, K, stride, blocks, c, e);
    return (int)hipGetLastError();
}

int launch_mx4_dequantize(const void *codes, const void *scales, long long rows, long long K, void *y, int dtype, long long stride,
                          void *stream) {
    const long long blocks = mx4_padded(K) / 32;
    const unsigned grid = (unsigned)((rows * blocks + 255) / 256);
    const hipStream_t s = (hipStream_t)stream;
    auto *c = (const unsigned char *)codes, *e = (const unsigned char *)scales;
    if (dtype == TDC_F32) tdc_mx4_dequantize_kernel<TDC_F32><<<grid, 256, 0, s>>>(c, e, rows, K, blocks, y, stride);
    else if (dtype == TDC_F16) tdc_mx4_dequantize_kernel<TDC_F16><<<grid, 256, 0, s>>>(c, e, rows, K, blocks, y, stride);
    else tdc_mx4_dequantize_kernel<TDC_BF16><<<grid, 256, 0, s>>>(c, e, rows, K, blocks, y, stride);
    return (int)hipGetLastError();
}

}  // namespace tdc
