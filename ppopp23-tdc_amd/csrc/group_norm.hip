// Group norm with an activation over channels-last tensors: forward and gradient.
//
//   y = act(gamma_c xh + beta_c),  xh = (x - mean) rstd,  mean / rstd over the pixels and channels of one image and group
//   dz = dy act'(gamma_c xh + beta_c),  dbeta_c = sum dz,  dgamma_c = sum dz xh,
//   dx = rstd (gamma_c dz - mean_g(gamma dz) - xh mean_g(gamma dz xh))
//
// Both directions are memory traffic and two launches: one reduces, one applies.  A workgroup owns `unit` neighbouring channels
// (whole groups, unless one group is wider than a workgroup) of a run of pixels; a thread moves `vec` channels of every R-th
// pixel with one request, so the lanes of a wave read runs of unit * vec numbers.  The partial results of a group are few
// (`slots` per image and group), and every workgroup of the second launch joins those of its own groups in its prologue: no
// atomics, no third launch, the same order on every run.
//
// Mean: summed in 64 bits (an add of which costs the vector unit what one in 32 does), so that it is off by the rounding of its
// last conversion alone, however the numbers cancel.  Variance: a thread sums (x - p)^2 about a value p of its own channel, so that an
// offset common to a channel cancels before it is squared, and sums of squared deviations are joined by
// M2 = sum M2_i + n_i (mean_i - mean)^2.  Everything else between load and store is fp32.
#include "ops_device.hpp"

namespace tdc {

static constexpr int kThreads = 256;

// What a workgroup owns.
struct Part {
    int image, tile, chunk;
    int c0, width, vecs;     // its channels, in all and as vectors
    int tr, tc, R;           // this thread's pixel row and vector, rows at a time (threads past them idle: tr >= R)
    int row0, rows;          // its pixels
    int g0, ng;              // its groups
};

static __device__ __forceinline__ Part part_of(const NormArgs &a, int vec, unsigned idx) {
    Part p;
    const NormPlan &n = a.plan;
    p.chunk = idx % n.chunks;
    idx /= n.chunks;
    p.tile = idx % n.tiles;
    p.image = idx / n.tiles;
    p.c0 = p.tile * n.unit;
    p.width = min(n.unit, a.C - p.c0);
    p.vecs = p.width / vec;
    p.R = kThreads / p.vecs;
    p.tr = threadIdx.x / p.vecs;
    p.tc = threadIdx.x - p.tr * p.vecs;
    p.row0 = p.chunk * n.chunk_rows;
    p.rows = min(n.chunk_rows, a.pixels - p.row0);
    p.g0 = p.c0 / a.Cg;
    p.ng = (p.c0 + p.width - 1) / a.Cg - p.g0 + 1;
    return p;
}
// Pixels of thread row r.
static __device__ __forceinline__ int rows_of(const Part &p, int r) { return r < p.rows && r < p.R ? (p.rows - r + p.R - 1) / p.R : 0; }

// So many lanes work on one group (a power of two, at most a wave), and this thread's place among them.
struct Team {
    int lanes, at, first, step;
};
static __device__ __forceinline__ Team team_of(int ng) {
    Team t;
    t.lanes = 64;
    while (t.lanes > 1 && ng * t.lanes > kThreads) t.lanes >>= 1;
    t.at = threadIdx.x & (t.lanes - 1);
    t.first = threadIdx.x / t.lanes;
    t.step = kThreads / t.lanes;
    return t;
}
template <typename T>
static __device__ __forceinline__ T team_sum(T v, int lanes) {
    for (int m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m, 64);
    return v;
}
// Channels that a group and a workgroup's tile share.
static __device__ __forceinline__ int shared_channels(const NormArgs &a, int g, int tile) {
    const int lo = max(g * a.Cg, tile * a.plan.unit), hi = min((g + 1) * a.Cg, min(a.C, (tile + 1) * a.plan.unit));
    return hi - lo;
}
static __device__ __forceinline__ long long slot_of(const NormArgs &a, const Part &p, int g) {
    return ((long long)p.image * a.groups + g) * a.plan.slots + p.chunk * a.plan.tiles_per_group + (p.tile - g * a.Cg / a.plan.unit);
}

template <int DT, int V>
__global__ void __launch_bounds__(kThreads) tdc_norm_stats_kernel(const NormArgs a) {
    using P = Pack<DT, V>;
    __shared__ double sums[kThreads * V];
    __shared__ float devs[kThreads * V];
    const Part p = part_of(a, V, blockIdx.x);
    const int n = rows_of(p, p.tr);
    float pivot[V], q[V];
    double s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) pivot[j] = q[j] = 0.0f;
    if (n > 0) {
        const long long at = p.image * a.x_is + (long long)(p.row0 + p.tr) * a.x_ps + p.c0 + p.tc * V, step = (long long)p.R * a.x_ps;
        P::up(P::load(a.x, at), pivot);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = pivot[j];
#pragma unroll 4
        for (int i = 1; i < n; ++i) {
            float v[V];
            P::up(P::load(a.x, at + i * step), v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] - pivot[j];
                s[j] += v[j];
                q[j] = fmaf(d, d, q[j]);
            }
        }
        const double inv = 1.0 / n;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = (float)(s[j] * inv - pivot[j]);
            sums[p.tr * p.width + p.tc * V + j] = s[j];
            devs[p.tr * p.width + p.tc * V + j] = q[j] - n * d * d;
        }
    }
    __syncthreads();
    const Team t = team_of(p.ng);
    for (int i = t.first; i < p.ng; i += t.step) {
        const int g = p.g0 + i, lo = max(g * a.Cg, p.c0) - p.c0, channels = shared_channels(a, g, p.tile);
        const int entries = channels * min(p.R, p.rows);
        double sum = 0.0;
        for (int e = t.at; e < entries; e += t.lanes) {
            const int r = e / channels;
            sum += sums[r * p.width + lo + e - r * channels];
        }
        sum = team_sum(sum, t.lanes);
        const double mean = sum / ((double)p.rows * channels);
        float m2 = 0.0f;
        for (int e = t.at; e < entries; e += t.lanes) {
            const int r = e / channels, n = rows_of(p, r), at = r * p.width + lo + e - r * channels;
            const float d = (float)(sums[at] / n - mean);
            m2 += devs[at] + n * d * d;
        }
        m2 = team_sum(m2, t.lanes);
        if (t.at == 0) a.stat[slot_of(a, p, g)] = NormStat{sum, m2};
    }
}

// Joins the partial results of a workgroup's groups: (mean, rstd) each.
static __device__ __forceinline__ void join_stats(const NormArgs &a, const Part &p, float2 *stat) {
    const Team t = team_of(p.ng);
    const NormPlan &n = a.plan;
    for (int i = t.first; i < p.ng; i += t.step) {
        const int g = p.g0 + i, tile0 = g * a.Cg / n.unit, tiles = ((g + 1) * a.Cg - 1) / n.unit - tile0 + 1;
        const NormStat *part = a.stat + ((long long)p.image * a.groups + g) * n.slots;
        double sum = 0.0;
        for (int k = 0; k < tiles; ++k)
            for (int c = t.at; c < n.chunks; c += t.lanes) sum += part[c * n.tiles_per_group + k].sum;
        const double all = (double)a.pixels * a.Cg, mean = team_sum(sum, t.lanes) / all;
        float m2 = 0.0f;
        for (int k = 0; k < tiles; ++k) {
            const int channels = shared_channels(a, g, tile0 + k);
            for (int c = t.at; c < n.chunks; c += t.lanes) {
                const NormStat v = part[c * n.tiles_per_group + k];
                const float count = (float)channels * min(n.chunk_rows, a.pixels - c * n.chunk_rows);
                const float d = (float)(v.sum / count - mean);
                m2 += v.m2 + count * d * d;
            }
        }
        m2 = team_sum(m2, t.lanes);
        if (t.at == 0) {
            stat[i] = make_float2((float)mean, 1.0f / sqrtf(m2 / (float)all + a.eps));
            // (the first chunk's workgroups keep them; of several that share a group, the first)
            if (p.chunk == 0 && p.tile == tile0) {
                if (a.mean) a.mean[(long long)p.image * a.groups + g] = stat[i].x;
                if (a.rstd) a.rstd[(long long)p.image * a.groups + g] = stat[i].y;
            }
        }
    }
    __syncthreads();
}

template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kThreads) tdc_norm_apply_kernel(const NormArgs a) {
    using P = Pack<DT, V>;
    __shared__ float2 stat[kThreads * V];
    const Part p = part_of(a, V, blockIdx.x);
    join_stats(a, p, stat);
    const int n = rows_of(p, p.tr);
    if (n == 0) return;
    float mean[V], scale[V], shift[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = p.c0 + p.tc * V + j;
        const float2 st = stat[c / a.Cg - p.g0];
        mean[j] = st.x;
        scale[j] = st.y * (a.gamma ? param<DT>(a.gamma, c, a.param_dtype) : 1.0f);
        shift[j] = a.beta ? param<DT>(a.beta, c, a.param_dtype) : 0.0f;
    }
    const long long c = p.c0 + p.tc * V, row = p.row0 + p.tr;
    const long long in = p.image * a.x_is + row * a.x_ps + c, out = p.image * a.o_is + row * a.o_ps + c;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        float v[V];
        P::up(P::load(a.x, in + (long long)i * p.R * a.x_ps), v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = act_of<ACT>(fmaf(v[j] - mean[j], scale[j], shift[j]));
        P::store(a.out, out + (long long)i * p.R * a.o_ps, P::down(v));
    }
}

// The same into 4 bits: a thread takes one block of 32 channels of a pixel, straight from the 32-bit values.  A tile ends at a
// multiple of 32 channels or at the last one; the last tile also writes the blocks that pad a row.
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kThreads) tdc_norm_apply_mx4_kernel(const NormArgs a) {
    using P = Pack<DT, V>;
    __shared__ float2 stat[kThreads * V];
    __shared__ float mean[kThreads * V], scale[kThreads * V], shift[kThreads * V];
    const Part p = part_of(a, V, blockIdx.x);
    join_stats(a, p, stat);
    for (int i = threadIdx.x; i < p.width; i += kThreads) {
        const int c = p.c0 + i;
        const float2 st = stat[c / a.Cg - p.g0];
        mean[i] = st.x;
        scale[i] = st.y * (a.gamma ? param<DT>(a.gamma, c, a.param_dtype) : 1.0f);
        shift[i] = a.beta ? param<DT>(a.beta, c, a.param_dtype) : 0.0f;
    }
    __syncthreads();
    const int padded = (a.C + 127) / 128 * 128, blocks = ((p.c0 + p.width == a.C ? padded : p.c0 + p.width) - p.c0) / 32;
    for (int i = threadIdx.x; i < p.rows * blocks; i += kThreads) {
        const int r = i / blocks, kb = i - r * blocks, n = min(32, p.width - kb * 32);
        const long long in = p.image * a.x_is + (long long)(p.row0 + r) * a.x_ps + p.c0 + kb * 32;
        const long long row = (long long)p.image * a.pixels + p.row0 + r, block = p.c0 / 32 + kb;
        float v[32], top = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; k += V) {
            float u[V];
#pragma unroll
            for (int j = 0; j < V; ++j) u[j] = 0.0f;
            if (k < n) {
                P::up(P::load(a.x, in + k), u);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int c = kb * 32 + k + j;
                    u[j] = act_of<ACT>(fmaf(u[j] - mean[c], scale[c], shift[c]));
                }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[k + j] = u[j];
                top = larger(top, u[j]);
            }
        }
        const int byte = mx4_scale_byte(top);
        const float divisor = mx4_divisor(byte);
        *reinterpret_cast<uint4 *>(a.codes + mx4_block_at(a.rows, row, block)) =
            make_uint4(mx4_codes(v, divisor), mx4_codes(v + 8, divisor), mx4_codes(v + 16, divisor), mx4_codes(v + 24, divisor));
        a.scales[((block >> 4) * a.rows + row) * 16 + (block & 3) * 4 + (block >> 2 & 3)] = (unsigned char)byte;
    }
    // (the scale bytes past a row's last block)
    if (p.c0 + p.width == a.C) {
        const int past = (a.C + 511) / 512 * 16 - padded / 32;
        for (int i = threadIdx.x; i < p.rows * past; i += kThreads) {
            const int r = i / past, block = padded / 32 + i - r * past;
            const long long row = (long long)p.image * a.pixels + p.row0 + r;
            a.scales[((block >> 4) * a.rows + row) * 16 + (block & 3) * 4 + (block >> 2 & 3)] = 0;
        }
    }
}

// Sums over a chunk's pixels: of dz and dz xh per channel, and of gamma times them per group.
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kThreads) tdc_norm_grad_sums_kernel(const NormArgs a) {
    using P = Pack<DT, V>;
    __shared__ float2 cell[kThreads * V];
    const Part p = part_of(a, V, blockIdx.x);
    const int n = rows_of(p, p.tr);
    float sz[V], sx[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sz[j] = sx[j] = 0.0f;
    if (n > 0) {
        float mean[V], rstd[V], gamma[V], beta[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = p.c0 + p.tc * V + j;
            const long long g = (long long)p.image * a.groups + c / a.Cg;
            mean[j] = a.mean[g];
            rstd[j] = a.rstd[g];
            gamma[j] = a.gamma ? param<DT>(a.gamma, c, a.param_dtype) : 1.0f;
            beta[j] = a.beta ? param<DT>(a.beta, c, a.param_dtype) : 0.0f;
        }
        const long long c = p.c0 + p.tc * V, row = p.row0 + p.tr;
        const long long at = p.image * a.x_is + row * a.x_ps + c, dat = p.image * a.d_is + row * a.d_ps + c;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            float v[V], d[V];
            P::up(P::load(a.x, at + (long long)i * p.R * a.x_ps), v);
            P::up(P::load(a.dy, dat + (long long)i * p.R * a.d_ps), d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (v[j] - mean[j]) * rstd[j];
                const float dz = d[j] * act_slope<ACT>(fmaf(xh, gamma[j], beta[j]));
                sz[j] += dz;
                sx[j] = fmaf(dz, xh, sx[j]);
            }
        }
    }
    if (p.tr < p.R) {
#pragma unroll
        for (int j = 0; j < V; ++j) cell[p.tr * p.width + p.tc * V + j] = make_float2(sz[j], sx[j]);
    }
    __syncthreads();
    float *const chan = a.chan + ((long long)p.image * a.plan.chunks + p.chunk) * 2 * a.C + p.c0;
    const int used = min(p.R, p.rows);
    for (int ch = threadIdx.x; ch < p.width; ch += kThreads) {
        float2 s = cell[ch];
        for (int r = 1; r < used; ++r) {
            const float2 e = cell[r * p.width + ch];
            s.x += e.x;
            s.y += e.y;
        }
        chan[ch] = s.x;
        chan[a.C + ch] = s.y;
        const float gamma = a.gamma ? param<DT>(a.gamma, p.c0 + ch, a.param_dtype) : 1.0f;
        cell[ch] = make_float2(gamma * s.x, gamma * s.y);
    }
    __syncthreads();
    const Team t = team_of(p.ng);
    for (int i = t.first; i < p.ng; i += t.step) {
        const int g = p.g0 + i, lo = max(g * a.Cg, p.c0) - p.c0, channels = shared_channels(a, g, p.tile);
        float s = 0.0f, x = 0.0f;
        for (int e = t.at; e < channels; e += t.lanes) {
            s += cell[lo + e].x;
            x += cell[lo + e].y;
        }
        s = team_sum(s, t.lanes);
        x = team_sum(x, t.lanes);
        if (t.at == 0) a.part[slot_of(a, p, g)] = make_float2(s, x);
    }
}

// The gradients: the first `param_blocks` workgroups add up 16 of the 2 C columns of the per-channel sums each, the others
// write dx.
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kThreads) tdc_norm_grad_apply_kernel(const NormArgs a, int param_blocks) {
    using P = Pack<DT, V>;
    __shared__ float2 stat[kThreads * V];
    if ((int)blockIdx.x < param_blocks) {
        float *const sum = reinterpret_cast<float *>(stat);
        const int col = blockIdx.x * 16 + (threadIdx.x & 15), lane = threadIdx.x >> 4;
        float s = 0.0f;
        if (col < 2 * a.C) {
            const int rows = a.batch * a.plan.chunks;
#pragma unroll 8
            for (int r = lane; r < rows; r += 16) s += a.chan[(long long)r * 2 * a.C + col];
        }
        sum[threadIdx.x] = s;
        __syncthreads();
        if (lane == 0 && col < 2 * a.C) {
            for (int r = 1; r < 16; ++r) s += sum[r * 16 + threadIdx.x];
            float *const to = col < a.C ? a.dbeta : a.dgamma;
            if (to) to[col < a.C ? col : col - a.C] = s;
        }
        return;
    }
    const Part p = part_of(a, V, blockIdx.x - param_blocks);
    {
        const Team t = team_of(p.ng);
        const NormPlan &n = a.plan;
        for (int i = t.first; i < p.ng; i += t.step) {
            const int g = p.g0 + i, tiles = ((g + 1) * a.Cg - 1) / n.unit - g * a.Cg / n.unit + 1;
            const float2 *part = a.part + ((long long)p.image * a.groups + g) * n.slots;
            float s = 0.0f, x = 0.0f;
            for (int k = 0; k < tiles; ++k)
                for (int c = t.at; c < n.chunks; c += t.lanes) {
                    const float2 v = part[c * n.tiles_per_group + k];
                    s += v.x;
                    x += v.y;
                }
            const float inv = 1.0f / ((float)a.pixels * a.Cg);
            s = team_sum(s, t.lanes) * inv;
            x = team_sum(x, t.lanes) * inv;
            if (t.at == 0) stat[i] = make_float2(s, x);
        }
        __syncthreads();
    }
    const int n = rows_of(p, p.tr);
    if (n == 0) return;
    float mean[V], rstd[V], gamma[V], beta[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = p.c0 + p.tc * V + j;
        const long long g = (long long)p.image * a.groups + c / a.Cg;
        const float2 st = stat[c / a.Cg - p.g0];
        mean[j] = a.mean[g];
        rstd[j] = a.rstd[g];
        s1[j] = st.x;
        s2[j] = st.y;
        gamma[j] = a.gamma ? param<DT>(a.gamma, c, a.param_dtype) : 1.0f;
        beta[j] = a.beta ? param<DT>(a.beta, c, a.param_dtype) : 0.0f;
    }
    const long long c = p.c0 + p.tc * V, row = p.row0 + p.tr;
    const long long at = p.image * a.x_is + row * a.x_ps + c, dat = p.image * a.d_is + row * a.d_ps + c,
                    out = p.image * a.o_is + row * a.o_ps + c;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        float v[V], d[V];
        P::up(P::load(a.x, at + (long long)i * p.R * a.x_ps), v);
        P::up(P::load(a.dy, dat + (long long)i * p.R * a.d_ps), d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float xh = (v[j] - mean[j]) * rstd[j];
            const float dz = d[j] * act_slope<ACT>(fmaf(xh, gamma[j], beta[j]));
            v[j] = rstd[j] * (fmaf(gamma[j], dz, -s1[j]) - xh * s2[j]);
        }
        P::store(a.out, out + (long long)i * p.R * a.o_ps, P::down(v));
    }
}

template <int DT, int V, int ACT>
static int forward(const NormArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)a.plan.chunks * a.plan.tiles * a.batch;
    tdc_norm_stats_kernel<DT, V><<<grid, kThreads, 0, s>>>(a);
    if (a.codes) tdc_norm_apply_mx4_kernel<DT, V, ACT><<<grid, kThreads, 0, s>>>(a);
    else tdc_norm_apply_kernel<DT, V, ACT><<<grid, kThreads, 0, s>>>(a);
    return (int)hipGetLastError();
}
template <int DT, int V, int ACT>
static int backward(const NormArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)a.plan.chunks * a.plan.tiles * a.batch;
    const int param_blocks = a.dgamma || a.dbeta ? (2 * a.C + 15) / 16 : 0;
    tdc_norm_grad_sums_kernel<DT, V, ACT><<<grid, kThreads, 0, s>>>(a);
    if (param_blocks || a.out)
        tdc_norm_grad_apply_kernel<DT, V, ACT><<<param_blocks + (a.out ? grid : 0), kThreads, 0, s>>>(a, param_blocks);
    return (int)hipGetLastError();
}
template <int DT, int V>
static int by_act(const NormArgs &a, bool grad, hipStream_t s) {
    if (a.act == TDC_ACT_RELU) return grad ? backward<DT, V, TDC_ACT_RELU>(a, s) : forward<DT, V, TDC_ACT_RELU>(a, s);
    if (a.act == TDC_ACT_SILU) return grad ? backward<DT, V, TDC_ACT_SILU>(a, s) : forward<DT, V, TDC_ACT_SILU>(a, s);
    return grad ? backward<DT, V, TDC_ACT_NONE>(a, s) : forward<DT, V, TDC_ACT_NONE>(a, s);
}
template <int DT>
static int by_vec(const NormArgs &a, bool grad, hipStream_t s) {
    constexpr int VM = DT == TDC_F32 ? 4 : 8;
    if (a.plan.vec == VM) return by_act<DT, VM>(a, grad, s);
    if (a.plan.vec == 2) return by_act<DT, 2>(a, grad, s);
    return by_act<DT, 1>(a, grad, s);
}
static int by_type(const NormArgs &a, int dtype, bool grad, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == TDC_F32) return by_vec<TDC_F32>(a, grad, s);
    if (dtype == TDC_F16) return by_vec<TDC_F16>(a, grad, s);
    return by_vec<TDC_BF16>(a, grad, s);
}

int launch_norm_forward(const NormArgs &a, int dtype, void *stream) { return by_type(a, dtype, false, stream); }
int launch_norm_backward(const NormArgs &a, int dtype, void *stream) { return by_type(a, dtype, true, stream); }

}  // namespace tdc
