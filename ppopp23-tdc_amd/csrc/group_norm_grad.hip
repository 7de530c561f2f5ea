// Gradient of the group norm with an activation over channels-last tensors.
//
//   dz = dy act'(gamma_c xh + beta_c),  xh = (x - mean) rstd,  dbeta_c = sum dz,  dgamma_c = sum dz xh,
//   dx = rstd (gamma_c dz - mean_g(gamma dz) - xh mean_g(gamma dz xh))
//
// Memory traffic, dealt out like the forward's: x and dy of a workgroup's channels and pixels sit in its registers, read once
// where the pixels of an image fit (up to 128 KiB of each a workgroup) and that keeps the chip busy, else twice, in two launches of many
// small workgroups whose threads have two pixels on their way while they work on two.  The sums over pixels are
// kept per channel: weighted by gamma and added over a group they are the two group means, and added over workgroups the
// parameters' gradients (by the first workgroups of the second launch, or in a launch of their own).  No atomics, the
// same order on every run.
//
// Sums over a thread's pixels are chains of at most 256 in fp32: dz and dz xh have no common offset to lose.  Where they meet others' they are
// added in 64 bits, for there is no limit to how many of them there are: 3e5 images of two pixels with one dy everywhere, whose additions
// are all rounded the same way, had dbeta 2e-5 off.
//
// Measured: 32 x 112 x 112 x 128 in 16 bits, silu: 40.5 us for the sums (5.1 TB/s) and 55.5 for dx (5.5), the vector unit busy for 60 to 70 % beside
// the memory.  28 x 28 x 256: 12 us, latencies of two launches; 14 x 14 x 1024: 10.4, one launch and that of the parameters.
#include "norm_device.hpp"

namespace tdc {

enum { kWhole, kSums, kApply };

// dz and xh of a thread's channels of one pixel.
template <int DT, int V, int ACT>
static __device__ __forceinline__ void slopes(const typename Pack<DT, V>::type &x, const typename Pack<DT, V>::type &dy, const float (&mean)[V],
                                              const float (&rstd)[V], const float (&gamma)[V], const float (&beta)[V], float (&dz)[V],
                                              float (&xh)[V]) {
    Pack<DT, V>::up(x, xh);
    Pack<DT, V>::up(dy, dz);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        xh[j] = (xh[j] - mean[j]) * rstd[j];
        dz[j] = act_back<ACT>(dz[j], fmaf(xh[j], gamma[j], beta[j]));
    }
}

// The parameters' gradients: a workgroup of 256 adds up 4 of the 2 C columns of the per-channel sums.
static __device__ __forceinline__ void add_params(const NormArgs &a, unsigned block, double *sum) {
    const int col = block * 4 + (threadIdx.x & 3), lane = threadIdx.x >> 2, rows = a.batch * a.plan.chunks;
    double s = 0.0;
    if (col < 2 * a.C) {
#pragma unroll 8
        for (int r = lane; r < rows; r += 64) s += a.chan[(long long)r * 2 * a.C + col];
    }
    sum[threadIdx.x] = s;
    __syncthreads();
    for (int half = 32; half; half /= 2) {
        if (lane < half) sum[threadIdx.x] += sum[threadIdx.x + 4 * half];
        __syncthreads();
    }
    if (lane == 0 && col < 2 * a.C) {
        float *const to = col < a.C ? a.dbeta : a.dgamma;
        if (to) to[col < a.C ? col : col - a.C] = (float)sum[threadIdx.x];
    }
}
static __global__ void __launch_bounds__(256) tdc_norm_param_grad_kernel(const NormArgs a) {
    __shared__ double sum[256];
    add_params(a, blockIdx.x, sum);
}

// (of the second launch, the first `param_blocks` workgroups do the parameters)
template <int DT, int V, int NV, int MODE, int ACT>
__global__ void __launch_bounds__(MODE == kWhole ? 512 : 256) tdc_norm_grad_kernel(const NormArgs a, unsigned param_blocks) {
    using P = Pack<DT, V>;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    if (MODE == kApply && blockIdx.x < param_blocks) {
        add_params(a, blockIdx.x, reinterpret_cast<double *>(lds));
        return;
    }
    const Part p = part_of(a, V, blockIdx.x - param_blocks, gridDim.x - param_blocks);
    const int n = rows_of(p, p.tr), c = p.c0 + p.tc * V;
    constexpr bool whole = MODE == kWhole;
    typename P::type x[whole ? 1 : 2][NV], dy[whole ? 1 : 2][NV];
    if constexpr (whole) {
        hold<DT, V, NV>(a.x, a.x_is, a.x_ps, p, n, x[0]);
        hold<DT, V, NV>(a.dy, a.d_is, a.d_ps, p, n, dy[0]);
    }
    float mean[V], rstd[V], gamma[V], beta[V];
    int g[V];
    groups_of(a, c, g);
    if (n > 0) {
        params<DT, V>(a, c, gamma, beta);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const long long at = (long long)p.image * a.groups + g[j];
            mean[j] = a.mean[at];
            rstd[j] = a.rstd[at];
        }
    }
    // All pixels of this thread, which has some.
    auto each = [&](auto use) {
        if constexpr (whole) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i < n) use(0, i, i);
        } else {
            constexpr bool back = MODE == kApply;
            const Walk<DT, V> in(a.x, a.x_is, a.x_ps, p, n, back), din(a.dy, a.d_is, a.d_ps, p, n, back);
            walk<NV>(n, quotient(p.rows, p.by_R), [&](int set, int at) {
                in.ask(at, x[set]);
                din.ask(at, dy[set]);
            }, [&](int set, int at, auto some) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (i < some) use(set, i, back ? n - 1 - at - i : at + i);
            });
        }
    };
    float2 *const cell = reinterpret_cast<float2 *>(lds), *const stat = cell + (MODE == kApply ? 0 : a.plan.threads * V);
    const double inv = a.per_number;
    const Team t = team_of(a.plan.threads, p.ng);
    if constexpr (MODE != kApply) {
        if (n > 0) {
            float sz[V], sx[V];
#pragma unroll
            for (int j = 0; j < V; ++j) sz[j] = sx[j] = 0.0f;
            each([&](int set, int i, int) {
                float dz[V], xh[V];
                slopes<DT, V, ACT>(x[set][i], dy[set][i], mean, rstd, gamma, beta, dz, xh);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sz[j] += dz[j];
                    sx[j] = fmaf(dz[j], xh[j], sx[j]);
                }
            });
#pragma unroll
            for (int j = 0; j < V; ++j) cell[p.tr * p.width + p.tc * V + j] = make_float2(sz[j], sx[j]);
        }
        __syncthreads();
        float *const chan = a.chan + ((long long)p.image * a.plan.chunks + p.chunk) * 2 * a.C + p.c0;
        const int used = min(p.R, p.rows);
        for (int ch = threadIdx.x; ch < p.width; ch += a.plan.threads) {
            double z = 0.0, u = 0.0;
            for (int r = 0; r < used; ++r) {
                const float2 e = cell[r * p.width + ch];
                z += e.x;
                u += e.y;
            }
            const float2 s = make_float2((float)z, (float)u);
            chan[ch] = s.x;
            chan[a.C + ch] = s.y;
            const float w = a.gamma ? param<DT>(a.gamma, p.c0 + ch, a.param_dtype) : 1.0f;
            cell[ch] = make_float2(w * s.x, w * s.y);
        }
        __syncthreads();
        for (int i = t.first; i < p.ng; i += t.step) {
            const int g = p.g0 + i, lo = max(g * a.Cg, p.c0) - p.c0, channels = shared_channels(a, g, p.tile);
            double s = 0.0, u = 0.0;
            for (int e = t.at; e < channels; e += t.lanes) {
                s += cell[lo + e].x;
                u += cell[lo + e].y;
            }
            s = team_sum(s, t.lanes);
            u = team_sum(u, t.lanes);
            if (t.at == 0) {
                if (MODE == kSums) a.part[slot_of(a, p, g)] = make_float2((float)s, (float)u);
                else stat[i] = make_float2((float)(s * inv), (float)(u * inv));
            }
        }
        if (MODE == kSums) return;
    } else {
        const NormPlan &m = a.plan;
        for (int i = t.first; i < p.ng; i += t.step) {
            const int g = p.g0 + i, tiles = tiles_of(a, p, g).y;
            const float2 *part = a.part + ((long long)p.image * a.groups + g) * m.slots;
            double s = 0.0, u = 0.0;
            for (int k = 0; k < tiles; ++k)
                for (int e = t.at; e < m.chunks; e += t.lanes) {
                    const float2 v = part[e * m.tiles_per_group + k];
                    s += v.x;
                    u += v.y;
                }
            s = team_sum(s, t.lanes) * inv;
            u = team_sum(u, t.lanes) * inv;
            if (t.at == 0) stat[i] = make_float2((float)s, (float)u);
        }
    }
    __syncthreads();
    if (n == 0 || !a.out) return;
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 st = stat[g[j] - p.g0];
        s1[j] = st.x;
        s2[j] = st.y;
    }
    const long long out = p.image * a.o_is + (long long)(p.row0 + p.tr) * a.o_ps + c, step = p.R * a.o_ps;
    if constexpr (whole) pack_again(x[0]);
    each([&](int set, int i, int at) {
        float dz[V], xh[V];
        slopes<DT, V, ACT>(x[set][i], dy[set][i], mean, rstd, gamma, beta, dz, xh);
#pragma unroll
        for (int j = 0; j < V; ++j) dz[j] = rstd[j] * (fmaf(gamma[j], dz[j], -s1[j]) - xh[j] * s2[j]);
        P::store(a.out, out + at * step, P::down(dz));
    });
}

template <int DT, int V, int NV, int ACT>
static int run(const NormArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)a.plan.chunks * a.plan.tiles * a.batch, threads = a.plan.threads;
    const unsigned param_blocks = a.dgamma || a.dbeta ? (unsigned)(2 * a.C + 3) / 4 : 0;
    if (a.plan.whole) tdc_norm_grad_kernel<DT, V, NV, kWhole, ACT><<<grid, threads, a.plan.lds, s>>>(a, 0);
    else tdc_norm_grad_kernel<DT, V, 2, kSums, ACT><<<grid, threads, a.plan.lds, s>>>(a, 0);
    if (!a.plan.whole && a.out) tdc_norm_grad_kernel<DT, V, 2, kApply, ACT><<<param_blocks + grid, threads, a.plan.lds, s>>>(a, param_blocks);
    else if (param_blocks) tdc_norm_param_grad_kernel<<<param_blocks, 256, 0, s>>>(a);
    return (int)hipGetLastError();
}
template <int DT, int ACT>
static int by_shape(const NormArgs &a, hipStream_t s) {
    constexpr int VM = DT == TDC_F32 ? 4 : 8;
    if (a.plan.vec == VM) return a.plan.held == 4 ? run<DT, VM, 4, ACT>(a, s) : run<DT, VM, 16, ACT>(a, s);
    return a.plan.vec == 2 ? run<DT, 2, 16, ACT>(a, s) : run<DT, 1, 16, ACT>(a, s);
}
template <int DT>
static int by_act(const NormArgs &a, hipStream_t s) {
    if (a.act == TDC_ACT_RELU) return by_shape<DT, TDC_ACT_RELU>(a, s);
    if (a.act == TDC_ACT_SILU) return by_shape<DT, TDC_ACT_SILU>(a, s);
    return by_shape<DT, TDC_ACT_NONE>(a, s);
}

int launch_norm_backward(const NormArgs &a, int dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == TDC_F32) return by_act<TDC_F32>(a, s);
    if (dtype == TDC_F16) return by_act<TDC_F16>(a, s);
    return by_act<TDC_BF16>(a, s);
}

}  // namespace tdc
