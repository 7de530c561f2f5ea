// RMS norm over the last axis with the residual's addition, its result in 16 or 32 bits or in microscaled 8 bits, and its gradient.
//
//   h = x + residual (rounded to their type: what is handed on is what is normalised),  y = w h r,  r = 1 / sqrt(mean h^2 + eps)
//   g = w dy,  u = h r:  dx = dresidual = r (g - u mean(g u)) + dh,  dw = sum over the rows of dy u
//
// Bound by memory: every number is read once and written once.  In bf16: 100352 x 256 with its residual 30 us (6.8 TB/s), 25088 x 512 with its
// residual into 8 bits 14.8 (6.1 TB/s).  100352 x 512 in a training step, forward and backward in turn: with the residual and h in 8 bits besides 76 (6.1 TB/s), the gradient
// from that 79 (4.6 TB/s: what the forward pass left in the caches goes to memory meanwhile).  The same over and over by themselves: 86 (5.4 TB/s) and 65
// (5.6 TB/s), from h 76 (5.4 TB/s).
// A team of lanes keeps a row in registers, eight numbers a lane and
// request; small teams with several requests in flight where rows are short, a whole workgroup where they are long.  Everything
// between loads and stores is fp32; sums over rows are fp32 along a thread's own rows (256 at most) and 64 bits from there on.
#include <algorithm>
#include <type_traits>

#include "ops_device.hpp"

namespace tdc {

template <int TEAM>
static __device__ __forceinline__ float team_sum(float v, float *lds) {
    // (sixteen lanes by rotations within the vector unit)
    auto turned = [](float x, auto by) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + decltype(by)::value, 0xf, 0xf, true)); };
    v += turned(v, std::integral_constant<int, 8>{});
    v += turned(v, std::integral_constant<int, 4>{});
    v += turned(v, std::integral_constant<int, 2>{});
    v += turned(v, std::integral_constant<int, 1>{});
#pragma unroll
    for (int m = 16; m < (TEAM < 64 ? TEAM : 64); m <<= 1) v += __shfl_xor(v, m, 64);
    if constexpr (TEAM > 64) {
        __syncthreads();      // (the last row's sums have been read)
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < TEAM / 64; ++i) v += lds[i];
    }
    return v;
}
// Eight numbers of a row from column c on, zeros past the C-th.
template <int DT>
static __device__ __forceinline__ typename Pack<DT, 8>::type load8(const void *base, long long at, int c, int C) {
    using P = Pack<DT, 8>;
    if (c + 8 <= C) return P::load(base, at + c);
    typename P::type v = {};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (c + i < C) v[i] = reinterpret_cast<const typename Num<DT>::type *>(base)[at + c + i];
    return v;
}
template <int DT>
static __device__ __forceinline__ void keep8(void *base, long long at, int c, int C, const float (&v)[8]) {
    using P = Pack<DT, 8>;
    if (c + 8 <= C) P::store(base, at + c, P::down(v));
    else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (c + i < C) reinterpret_cast<typename Num<DT>::type *>(base)[at + c + i] = Num<DT>::down(v[i]);
    }
}
// Makes a vector new to the compiler, which would else keep what it has unpacked of it.
template <typename T>
static __device__ __forceinline__ void again(T &v) {
    typedef int words_t __attribute__((ext_vector_type(sizeof(T) / 4)));
    words_t w = __builtin_bit_cast(words_t, v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) {
        int one = w[i];
        asm volatile("" : "+v"(one));
        w[i] = one;
    }
    v = __builtin_bit_cast(T, w);
}
// Eight weights from column c on.
template <int DT>
static __device__ __forceinline__ void weights(const RmsArgs &a, int c, float (&w)[8]) {
    if (a.weight && c + 8 <= a.C) {
        if (DT == TDC_F32 || a.weight_dtype == TDC_F32) Pack<TDC_F32, 8>::up(Pack<TDC_F32, 8>::load(a.weight, c), w);
        else Pack<DT, 8>::up(Pack<DT, 8>::load(a.weight, c), w);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = c + j >= a.C ? 0.0f : a.weight ? param<DT>(a.weight, c + j, a.weight_dtype) : 1.0f;
}
// Where the scale of block b of a row is.
static __device__ __forceinline__ long long scale_at(long long rows, long long row, int b) {
    return ((b >> 4) * rows + row) * 16 + (b & 3) * 4 + (b >> 2 & 3);
}
static constexpr int kThreads = 256;

template <int DT, int MODE, int TEAM, int NV>
__global__ void __launch_bounds__(kThreads) tdc_rms_forward_kernel(const RmsArgs a) {
    using P = Pack<DT, 8>;
    constexpr int kRows = kThreads / TEAM;
    __shared__ float lds[TEAM > 64 ? TEAM / 64 : 1];
    const int l = threadIdx.x % TEAM;
    const float by_C = 1.0f / (float)a.C;
    typename P::type px[NV], pr[NV];
    auto ask = [&](long long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) px[i] = load8<DT>(a.x, row * a.x_stride, (l + TEAM * i) * 8, a.C);
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < NV; ++i) pr[i] = load8<DT>(a.residual, row * a.r_stride, (l + TEAM * i) * 8, a.C);
        }
    };
    long long row = (long long)blockIdx.x * kRows + threadIdx.x / TEAM;
    if (row < a.rows) ask(row);
    float w[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) weights<DT>(a, (l + TEAM * i) * 8, w[i]);
    for (const long long on = (long long)gridDim.x * kRows; row < a.rows; row += on) {
        float h[NV][8], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            P::up(px[i], h[i]);
            if (a.residual) {
                float r[8];
                P::up(pr[i], r);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = Num<DT>::up(Num<DT>::down(h[i][j] + r[j]));
                keep8<DT>(a.h, row * a.C, (l + TEAM * i) * 8, a.C, h[i]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
        }
        if (row + on < a.rows) ask(row + on);      // (the next row is on its way while this one is finished)
        const float r = rsqrtf(fmaf(team_sum<TEAM>(sum, lds), by_C, a.eps));
        if (a.rstd && l == 0) a.rstd[row] = r;
        const long long pitch = (a.C + 127) & ~127;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + TEAM * i) * 8;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = h[i][j] * r * w[i][j];
            if (MODE == kRmsOutputMx8 && c + 8 > a.C) {
                // (what lies past the last number is zeros, also where r is none or infinite)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j >= a.C) y[j] = 0.0f;
            }
            if constexpr (MODE != kRmsOutputMx8) keep8<DT>(a.y, row * a.C, c, a.C, y);
            if constexpr (MODE != kRmsPlain) {
                const float *const v = MODE == kRmsOutputMx8 ? y : h[i];
                float top = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = larger(top, v[j]);
                const int byte = mx8_scale_byte(quad_larger(top));
                if (c < pitch) {
                    *reinterpret_cast<uint2 *>(a.codes + row * pitch + c) = mx8_codes(v, mx4_divisor(byte));
                    if ((l & 3) == 0) a.scales[scale_at(a.rows, row, c >> 5)] = (unsigned char)byte;
                }
            }
        }
        if constexpr (MODE != kRmsPlain) {
            // the scale bytes past the last 128 numbers
            for (int b = (int)(pitch >> 5) + l; b < (a.C + 511) / 512 * 16; b += TEAM) a.scales[scale_at(a.rows, row, b)] = 0;
        }
    }
}

template <int DT, bool KEPT8, int TEAM, int NV>
__global__ void __launch_bounds__(kThreads) tdc_rms_backward_kernel(const RmsArgs a) {
    using P = Pack<DT, 8>;
    constexpr int kRows = kThreads / TEAM, kWidth = TEAM * NV * 8;
    __shared__ float lds[TEAM > 64 ? TEAM / 64 : 1];
    __shared__ float sums[kRows > 1 ? kRows * kWidth : 1];
    const int l = threadIdx.x % TEAM;
    float dw[NV][8] = {};
    float w[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) weights<DT>(a, (l + TEAM * i) * 8, w[i]);
    const float by_C = 1.0f / (float)a.C;
    const long long pitch = (a.C + 127) & ~127;
    for (long long row = (long long)blockIdx.x * kRows + threadIdx.x / TEAM; row < a.rows; row += (long long)gridDim.x * kRows) {
        typename P::type ph[NV], pg[NV], pd[NV];
        uint2 codes[NV];
        unsigned char scale[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (l + TEAM * i) * 8;
            if constexpr (KEPT8) {
                codes[i] = make_uint2(0, 0);
                scale[i] = 0;
                if (c < pitch) {
                    codes[i] = *reinterpret_cast<const uint2 *>(a.codes + row * pitch + c);
                    scale[i] = a.scales[scale_at(a.rows, row, c >> 5)];
                }
            } else ph[i] = load8<DT>(a.h, row * a.x_stride, c, a.C);
            pg[i] = load8<DT>(a.dy, row * a.dy_stride, c, a.C);
        }
        if (a.dh) {
#pragma unroll
            for (int i = 0; i < NV; ++i) pd[i] = load8<DT>(a.dh, row * a.dh_stride, (l + TEAM * i) * 8, a.C);
        }
        const float r = a.rstd[row];
        // (both times from what was loaded: u and g in fp32 would not fit beside the sums)
        auto unpack = [&](int i, float (&u)[8], float (&g)[8]) {
            if constexpr (KEPT8) {
                mx8_values(codes[i], mx4_divisor(scale[i]), u);
                if (scale[i] == 255) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] = __builtin_nanf("");
                }
            } else P::up(ph[i], u);
            P::up(pg[i], g);
        };
        float along = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float u[8], g[8];
            unpack(i, u, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                u[j] *= r;
                dw[i][j] = fmaf(g[j], u[j], dw[i][j]);
                along = fmaf(g[j] * w[i][j], u[j], along);
            }
        }
        along = team_sum<TEAM>(along, lds) * by_C;
        if (!a.dx) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (KEPT8) asm volatile("" : "+v"(codes[i].x), "+v"(codes[i].y));
            else again(ph[i]);
            again(pg[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float u[8], g[8], d[8] = {};
            unpack(i, u, g);
            if (a.dh) P::up(pd[i], d);
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = fmaf(r, fmaf(-u[j] * r, along, g[j] * w[i][j]), d[j]);
            keep8<DT>(a.dx, row * a.C, (l + TEAM * i) * 8, a.C, d);
        }
    }
    if (!a.dweight) return;
    float *const part = a.part + (long long)blockIdx.x * a.C;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) keep8<TDC_F32>(part, 0, (l + TEAM * i) * 8, a.C, dw[i]);
    } else {
        float *const mine = sums + threadIdx.x / TEAM * kWidth;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) mine[(l + TEAM * i) * 8 + j] = dw[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < a.C; c += 256) {
            double s = 0;
#pragma unroll
            for (int k = 0; k < kRows; ++k) s += sums[k * kWidth + c];
            part[c] = (float)s;
        }
    }
}

void rms_plan(RmsArgs &a, bool grad) {
    const int vectors = (a.C + 7) / 8;      // (1024 at most)
    // (100352 x 512 in bf16, gradient from 8 bits: 65 us with 32 lanes and two requests each, 70 with 16 and four, 71 with 64 and one; 25088 x 512
    // into 8 bits 14.5, 16.6, 15.8; 100352 x 256 the same with 16 lanes and two as with 32 and one)
    a.team = vectors <= 32 ? 16 : vectors <= 64 ? 32 : vectors <= 256 ? 64 : 256;
    a.held = vectors <= 16 ? 1 : vectors <= 2 * a.team ? 2 : 4;
    const int rows = kThreads / a.team;
    const long long groups = (a.rows + rows - 1) / rows;
    // Forward: eight workgroups to a compute unit.  Gradient: two, as many as its registers leave room for; 256 rows a thread at most.
    const long long most = grad ? 512 : 2048;
    a.blocks = (int)std::max(std::min(groups, most), grad ? (groups + 255) / 256 : 1);
}
long long rms_items(const RmsArgs &a, bool grad) {
    return std::max((long long)a.blocks * kThreads, grad ? ((long long)a.C + 63) / 64 * 1024 : 0);
}

template <int DT, int MODE, int TEAM, int NV>
static int forward_one(const RmsArgs &a, hipStream_t s) {
    tdc_rms_forward_kernel<DT, MODE, TEAM, NV><<<a.blocks, kThreads, 0, s>>>(a);
    return (int)hipGetLastError();
}
template <int DT, bool KEPT8, int TEAM, int NV>
static int backward_one(const RmsArgs &a, hipStream_t s) {
    tdc_rms_backward_kernel<DT, KEPT8, TEAM, NV><<<a.blocks, kThreads, 0, s>>>(a);
    if (hipError_t e = hipGetLastError()) return (int)e;
    return a.dweight ? launch_column_sums(a.part, a.dweight, a.C, a.blocks, a.weight_dtype, s) : 0;
}
#define TDC_RMS_TEAMS(one, ...)                                                                             \
    switch (a.team) {                                                                                       \
        case 16: return a.held == 1 ? one<__VA_ARGS__, 16, 1>(a, s) : one<__VA_ARGS__, 16, 2>(a, s);        \
        case 32: return one<__VA_ARGS__, 32, 2>(a, s);                                                      \
        case 64: return a.held == 2 ? one<__VA_ARGS__, 64, 2>(a, s) : one<__VA_ARGS__, 64, 4>(a, s);        \
        default: return a.held == 2 ? one<__VA_ARGS__, 256, 2>(a, s) : one<__VA_ARGS__, 256, 4>(a, s);      \
    }
template <int DT, int MODE>
static int forward_of(const RmsArgs &a, hipStream_t s) { TDC_RMS_TEAMS(forward_one, DT, MODE) }
template <int DT, bool KEPT8>
static int backward_of(const RmsArgs &a, hipStream_t s) { TDC_RMS_TEAMS(backward_one, DT, KEPT8) }
template <int DT>
static int forward_mode(const RmsArgs &a, int mode, hipStream_t s) {
    if (mode == kRmsPlain) return forward_of<DT, kRmsPlain>(a, s);
    return mode == kRmsOutputMx8 ? forward_of<DT, kRmsOutputMx8>(a, s) : forward_of<DT, kRmsKeptMx8>(a, s);
}
int launch_rms_forward(const RmsArgs &a, int dtype, int mode, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == TDC_F32) return forward_mode<TDC_F32>(a, mode, s);
    return dtype == TDC_F16 ? forward_mode<TDC_F16>(a, mode, s) : forward_mode<TDC_BF16>(a, mode, s);
}
int launch_rms_backward(const RmsArgs &a, int dtype, bool kept_mx8, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == TDC_F32) return kept_mx8 ? backward_of<TDC_F32, true>(a, s) : backward_of<TDC_F32, false>(a, s);
    if (dtype == TDC_F16) return kept_mx8 ? backward_of<TDC_F16, true>(a, s) : backward_of<TDC_F16, false>(a, s);
    return kept_mx8 ? backward_of<TDC_BF16, true>(a, s) : backward_of<TDC_BF16, false>(a, s);
}

}  // namespace tdc
