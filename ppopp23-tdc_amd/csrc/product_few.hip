// Products in 16 and 8 bits of few rows of x, both operands along the sum (see product_tile.hpp): tokens one by one.
//
// Bound by the weights' bytes, or by latency.  A workgroup of eight waves owns 16 rows of w and up to 16 of x; its waves share the sum, 256
// bytes of a row at a time, with operands straight in registers (a request is 64 bytes of each of sixteen rows) and the next ones on their
// way.  The waves' sums meet in LDS, in the order of the waves: no second launch.
// v_mfma_f32_16x16x32 (8 bits: the scaled 16x16x128): lane r + 16 g has a row's bytes 16 g .. 16 g + 15 of each 64, in 8 bits with the scale
// of the g-th block of 128 numbers; a lane ends up with four neighbouring outputs 4 g .. 4 g + 3 of row r of x.
//
// Measured, bf16, one row by weights that no cache holds: 16384 x 4096 26.5 us (5.1 TB/s; tiles of 32 rows with the sum in four parts 30.0),
// 4096 x 4096 9.2 (11.9), 1024 x 1024 from a cache 4.1 (7.3); in 8 bits 17.9 (17.9), eight rows by 4096 x 4096 7.6 (9.9).  Sixteen waves instead of eight:
// 32.3, 10.3, 4.1.
#include <algorithm>

#include "product_device.hpp"

namespace tdc {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
static constexpr int kWaves = 8;

template <int IN, int OUT>
__global__ void __launch_bounds__(kWaves * 64) tdc_product_few_kernel(const TileArgs a) {
    constexpr bool k8 = IN == TDC_MX8;
    __shared__ float part[kWaves][64][4];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 15, g = lane >> 4;
    const long long n0 = (long long)blockIdx.x * 16;
    const __amdgpu_buffer_rsrc_t from_w = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(a.w + n0 * a.w_stride), 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t from_x = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(a.x), 0, 0x7fffffff, 0x00020000);
    // (rows past the last repeat it: their products go nowhere)
    const int w_row = (int)min((long long)r, a.N - n0 - 1), x_row = min(r, (int)a.M - 1);
    const int w_at = w_row * (int)a.w_stride + g * 16, x_at = x_row * (int)a.x_stride + g * 16;
    const int bytes = (int)(min(a.x_limit, a.w_limit) * (k8 ? 1 : 2)), slices = (bytes + 255) / 256;
    i4_t w[2][4], x[2][4];
    int sw[2], sx[2];
    auto ask = [&](auto set, int slice) {
        constexpr int S = decltype(set)::value;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            // (what lies past the sum is zeros: an offset past the descriptor's 2 GiB)
            const int k = slice * 256 + p * 64, past = k + g * 16 < bytes ? 0 : (int)0x80000000;
            w[S][p] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(from_w, (w_at + k) | past, 0, 0));
            x[S][p] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(from_x, (x_at + k) | past, 0, 0));
        }
        if constexpr (k8) {
            // Scales of 512 numbers, a word for the g-th blocks of each 128 (a slice past the last repeats it: its numbers are zeros).
            const long long at = min(slice, slices - 1) / 2;
            sw[S] = *reinterpret_cast<const int *>(a.w_scales + (at * a.N + n0 + w_row) * 16 + g * 4);
            sx[S] = *reinterpret_cast<const int *>(a.x_scales + (at * a.M + x_row) * 16 + g * 4);
        }
    };
    f4_t acc = {0, 0, 0, 0};
    auto add = [&](auto set, int slice) {
        constexpr int S = decltype(set)::value;
        if constexpr (k8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int byte = (slice & 1) * 16 + h * 8;
                const i4_t &u = w[S][2 * h], &v = w[S][2 * h + 1], &y = x[S][2 * h], &z = x[S][2 * h + 1];
                const i8_t wv = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]}, xv = {y[0], y[1], y[2], y[3], z[0], z[1], z[2], z[3]};
                acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc, 0, 0, 0, (int)((unsigned)sw[S] >> byte), 0, (int)((unsigned)sx[S] >> byte));
            }
        } else {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                if constexpr (IN == TDC_F16) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, w[S][p]), __builtin_bit_cast(h8_t, x[S][p]), acc, 0, 0, 0);
                else acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, w[S][p]), __builtin_bit_cast(b8_t, x[S][p]), acc, 0, 0, 0);
            }
        }
    };
    const std::integral_constant<int, 0> zero;
    const std::integral_constant<int, 1> one;
    if (wave < slices) {
        ask(zero, wave);
        for (int s = wave; s < slices; s += 2 * kWaves) {
            ask(one, s + kWaves);
            __builtin_amdgcn_sched_barrier(0);      // (else the compiler asks for them when they are needed)
            add(zero, s);
            ask(zero, s + 2 * kWaves);
            __builtin_amdgcn_sched_barrier(0);
            add(one, s + kWaves);
        }
        *reinterpret_cast<f4_t *>(part[wave][lane]) = acc;
    }
    __syncthreads();
    const int summed = min(kWaves, slices);      // (the other waves had nothing)
    using T = typename Num<OUT>::type;
    const long long n = n0 + (t & 15);
    const int m = t >> 4;
    if (n >= a.N || m >= a.M) return;
    float z = 0.0f;
    for (int k = 0; k < summed; ++k) z += part[k][(t >> 2 & 3) * 16 + m][t & 3];
    if (a.bias) z += param<OUT>(a.bias, n, a.bias_dtype);
    if (a.residual) z += Num<OUT>::up(reinterpret_cast<const T *>(a.residual)[m * a.r_stride + n]);
    if (a.z) reinterpret_cast<T *>(a.z)[m * a.z_stride + n] = Num<OUT>::down(z);
    z = a.act == TDC_ACT_RELU ? act_of<TDC_ACT_RELU>(z) : a.act == TDC_ACT_SILU ? act_of<TDC_ACT_SILU>(z) : z;
    reinterpret_cast<T *>(a.y)[m * a.y_stride + n] = Num<OUT>::down(z);
}

// One row of x up to 16.  A wave's 256 bytes of the sum take some 1.05 us, the next ones on their way: 1 x 4096 x 4096 7.2, 1 x 64 x 8192 10.9 (6.7
// in 32 parts of tiles).
double few_time(long long N, long long bytes) {
    const double blocks = (double)((N + 15) / 16), turns = (double)((bytes + 256 * kWaves - 1) / (256 * kWaves));
    return 2.5 + 1.05 * turns * std::max(1.0, blocks / 512);
}
long long few_items(long long N) { return (N + 15) / 16 * kWaves * 64; }

int launch_product_few(const TileArgs &a, int in_dtype, int y_dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    const unsigned blocks = (unsigned)((a.N + 15) / 16);
    if (in_dtype == TDC_F16) tdc_product_few_kernel<TDC_F16, TDC_F16><<<blocks, kWaves * 64, 0, s>>>(a);
    else if (in_dtype == TDC_BF16) tdc_product_few_kernel<TDC_BF16, TDC_BF16><<<blocks, kWaves * 64, 0, s>>>(a);
    else if (y_dtype == TDC_F16) tdc_product_few_kernel<TDC_MX8, TDC_F16><<<blocks, kWaves * 64, 0, s>>>(a);
    else tdc_product_few_kernel<TDC_MX8, TDC_BF16><<<blocks, kWaves * 64, 0, s>>>(a);
    return (int)hipGetLastError();
}

}  // namespace tdc
