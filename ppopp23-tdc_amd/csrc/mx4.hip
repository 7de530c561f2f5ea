// Numbers into microscaled 4-bit floating point and back (format and layout: include/tdc.h).
//
// Memory traffic: x on one side, 17/32 byte a number on the other.  Sixteen lanes take 128 numbers of a row, eight each: one request of
// 16 bytes (two in 32 bits), a block's largest magnitude from four neighbouring lanes, one word of codes a lane.  A thread goes
// on for 512 numbers, so that a quad of lanes ends up with one word of scales.
// Requests need no alignment beyond the number's own; only the last one of a row may end early.
//
// Measured: 100352 x 256 in bf16 12.6 us into 4 bits and 11.8 back, 5.2 and 5.5 TB/s, a copy's rate; 8192 x 8192 33 to 36 us.
#include "ops_device.hpp"

namespace tdc {

static constexpr int kRows = 16;      // of a workgroup of 256
static constexpr int kSteps = 4;      // runs of 128 numbers a thread has in flight: those of a word of scales

template <int DT>
__global__ void __launch_bounds__(256) tdc_mx4_quantize_kernel(const void *x, long long rows, long long K, long long stride, int groups,
                                                               int runs, unsigned *codes, unsigned *scales) {
    using T = typename Num<DT>::type;
    typedef T vec_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const long long rb = blockIdx.x / (unsigned)runs;
    const int g0 = (blockIdx.x - (unsigned)rb * runs) * kSteps, lane = threadIdx.x & 15;
    const long long row = rb * kRows + (threadIdx.x >> 4);
    if (row >= rows) return;
    const T *const src = reinterpret_cast<const T *>(x) + row * stride + lane * 8;
    vec_t p[kSteps];
    if ((long long)(g0 + kSteps) * 128 <= K) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) p[s] = *reinterpret_cast<const vec_t *>(src + (g0 + s) * 128ll);
    } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            p[s] = vec_t{};
            if ((g0 + s) * 128ll + lane * 8 + 8 <= K) p[s] = *reinterpret_cast<const vec_t *>(src + (g0 + s) * 128ll);
        }
        // (the numbers of a row's last request, where it ends early)
        if (K & 7) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int n = (int)(K - (g0 + s) * 128ll) - lane * 8;
                if (n > 0 && n < 8) {
#pragma unroll
                    for (int i = 0; i < 7; ++i)
                        if (i < n) p[s][i] = src[(g0 + s) * 128ll + i];
                }
            }
        }
    }
    unsigned word = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        if (g0 + s >= groups) continue;
        float v[8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = Num<DT>::up(p[s][i]);
            top = larger(top, v[i]);
        }
        const int byte = mx4_scale_byte(quad_larger(top));
        codes[(mx4_block_at(rows, row, (g0 + s) * 4 + (lane >> 2)) >> 2) + (lane & 3)] = mx4_codes(v, mx4_divisor(byte));
        word |= (unsigned)byte << 8 * s;
    }
    if ((lane & 3) == 0) scales[((g0 >> 2) * rows + row) * 4 + (lane >> 2)] = word;
}

template <int DT>
__global__ void __launch_bounds__(256) tdc_mx4_dequantize_kernel(const unsigned *codes, const unsigned *scales, long long rows, long long K,
                                                                 int groups, int runs, void *y, long long stride) {
    using T = typename Num<DT>::type;
    typedef T vec_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const long long rb = blockIdx.x / (unsigned)runs;
    const int g0 = (blockIdx.x - (unsigned)rb * runs) * kSteps, lane = threadIdx.x & 15;
    const long long row = rb * kRows + (threadIdx.x >> 4);
    if (row >= rows) return;
    T *const dst = reinterpret_cast<T *>(y) + row * stride + lane * 8;
    unsigned code[kSteps];
    const unsigned word = scales[((g0 >> 2) * rows + row) * 4 + (lane >> 2)];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int g = min(g0 + s, groups - 1);
        code[s] = codes[(mx4_block_at(rows, row, g * 4 + (lane >> 2)) >> 2) + (lane & 3)];
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const long long k = (long long)(g0 + s) * 128 + lane * 8;
        if (k >= K) continue;
        const int byte = (word >> 8 * s) & 255;
        float v[8];
        mx4_values(code[s], mx4_divisor(byte), v);
        vec_t p;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = Num<DT>::down(byte == 255 ? __builtin_nanf("") : v[i]);
        if (k + 8 <= K) *reinterpret_cast<vec_t *>(dst + k - lane * 8) = p;
        else
            for (int i = 0; i < 8; ++i)
                if (k + i < K) dst[k - lane * 8 + i] = p[i];
    }
}

static long long workgroups(long long rows, int runs) { return (rows + kRows - 1) / kRows * runs; }
static int runs_of(long long K) { return (int)((mx4_padded(K) / 128 + kSteps - 1) / kSteps); }
long long mx4_work_items(long long rows, long long K) { return workgroups(rows, runs_of(K)) * 256; }

int launch_mx4_quantize(const void *x, int dtype, long long rows, long long K, long long stride, void *codes, void *scales, void *stream) {
    const int groups = (int)(mx4_padded(K) / 128), runs = runs_of(K);
    const unsigned grid = (unsigned)workgroups(rows, runs);
    const hipStream_t s = (hipStream_t)stream;
    auto *c = (unsigned *)codes, *e = (unsigned *)scales;
    if (dtype == TDC_F32) tdc_mx4_quantize_kernel<TDC_F32><<<grid, 256, 0, s>>>(x, rows, K, stride, groups, runs, c, e);
    else if (dtype == TDC_F16) tdc_mx4_quantize_kernel<TDC_F16><<<grid, 256, 0, s>>>(x, rows, K, stride, groups, runs, c, e);
    else tdc_mx4_quantize_kernel<TDC_BF16><<<grid, 256, 0, s>>>(x, rows, K, stride, groups, runs, c, e);
    return (int)hipGetLastError();
}

int launch_mx4_dequantize(const void *codes, const void *scales, long long rows, long long K, void *y, int dtype, long long stride,
                          void *stream) {
    const int groups = (int)(mx4_padded(K) / 128), runs = runs_of(K);
    const unsigned grid = (unsigned)workgroups(rows, runs);
    const hipStream_t s = (hipStream_t)stream;
    auto *c = (const unsigned *)codes, *e = (const unsigned *)scales;
    if (dtype == TDC_F32) tdc_mx4_dequantize_kernel<TDC_F32><<<grid, 256, 0, s>>>(c, e, rows, K, groups, runs, y, stride);
    else if (dtype == TDC_F16) tdc_mx4_dequantize_kernel<TDC_F16><<<grid, 256, 0, s>>>(c, e, rows, K, groups, runs, y, stride);
    else tdc_mx4_dequantize_kernel<TDC_BF16><<<grid, 256, 0, s>>>(c, e, rows, K, groups, runs, y, stride);
    return (int)hipGetLastError();
}

}  // namespace tdc
