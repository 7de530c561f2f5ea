// Product of two matrices in microscaled 4-bit floating point: y = act(x w^T + bias + residual).
//
// v_mfma_scale_f32_16x16x128: a lane holds one block of 32 numbers of its row (lane mod 16), place lane / 16 of the four of
// a step, with that block's scale; products and sums are fp32.  The weights are the first operand, so that a lane ends
// up with four neighbouring outputs of one row.
#include "ops_device.hpp"

namespace tdc {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

static __device__ __forceinline__ f4_t mfma4(i4_t a, i4_t b, f4_t c, int sa, int sb) {
    const i8_t wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

// One wave per 32 x 32 outputs, four of them side by side along N.
template <int DT>
__global__ void __launch_bounds__(256) tdc_mx4_product_kernel(const ProductArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const unsigned across = (unsigned)((a.N + 127) / 128);
    const long long n0 = ((long long)(blockIdx.x % across) * 4 + wave) * 32, m0 = (long long)(blockIdx.x / across) * 32;
    if (n0 >= a.N) return;
    const unsigned char *xc[2], *wc[2];
    long long xr[2], wr[2];
    bool xin[2], win[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        xr[i] = m0 + 16 * i + r;
        wr[i] = n0 + 16 * i + r;
        xin[i] = xr[i] < a.M;
        win[i] = wr[i] < a.N;
        xc[i] = a.x_codes + (xin[i] ? xr[i] : 0) * a.ksteps * 64 + 16 * q;
        wc[i] = a.w_codes + (win[i] ? wr[i] : 0) * a.ksteps * 64 + 16 * q;
    }
    f4_t acc[2][2] = {};
    for (int k = 0; k < a.ksteps; ++k) {
        i4_t xf[2], wf[2];
        int xs[2], ws[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const i4_t zero = {0, 0, 0, 0};
            xf[i] = xin[i] ? *reinterpret_cast<const i4_t *>(xc[i] + (long long)k * 64) : zero;
            wf[i] = win[i] ? *reinterpret_cast<const i4_t *>(wc[i] + (long long)k * 64) : zero;
            xs[i] = xin[i] ? a.x_scales[(k * a.M + xr[i]) * 4 + q] : 0;
            ws[i] = win[i] ? a.w_scales[(k * a.N + wr[i]) * 4 + q] : 0;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mfma4(wf[i], xf[j], acc[i][j], ws[i], xs[j]);
    }
    using T = typename Num<DT>::type;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const long long n = n0 + 16 * i + 4 * q + e, m = m0 + 16 * j + r;
                if (n >= a.N || m >= a.M) continue;
                float v = acc[i][j][e];
                if (a.bias) v += param<DT>(a.bias, n, a.bias_dtype);
                if (a.residual) v += Num<DT>::up(reinterpret_cast<const T *>(a.residual)[m * a.r_stride + n]);
                v = a.act == TDC_ACT_RELU ? act_of<TDC_ACT_RELU>(v) : a.act == TDC_ACT_SILU ? act_of<TDC_ACT_SILU>(v) : v;
                reinterpret_cast<T *>(a.y)[m * a.y_stride + n] = Num<DT>::down(v);
            }
}

int launch_mx4_product(const ProductArgs &a, int y_dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    const unsigned grid = (unsigned)(((a.N + 127) / 128) * ((a.M + 31) / 32));
    if (y_dtype == TDC_F32) tdc_mx4_product_kernel<TDC_F32><<<grid, 256, 0, s>>>(a);
    else if (y_dtype == TDC_F16) tdc_mx4_product_kernel<TDC_F16><<<grid, 256, 0, s>>>(a);
    else tdc_mx4_product_kernel<TDC_BF16><<<grid, 256, 0, s>>>(a);
    return (int)hipGetLastError();
}

}  // namespace tdc
