// Group norm with an activation over channels-last tensors, forward, into numbers or into 4 bits.
//
//   y = act(gamma_c (x - mean) rstd + beta_c),  mean / rstd over the pixels and channels of one image and group
//
// Memory traffic.  A workgroup owns `unit` neighbouring channels (whole groups, unless one group is wider than that) of a run of
// pixels, and holds them in registers: a thread asks for `vec` channels of every R-th pixel, all requests at once.  Where the
// pixels of an image fit (up to 256 KiB a workgroup), and that does not leave most of the chip idle, that is all: x is read once, the
// statistics meet in LDS, y is written.  Else one launch leaves partial statistics, and a second reads x again and joins, while it comes, the partial results of its own
// groups: no atomics, no third launch, the same order on every run.  These two are made of many small workgroups whose threads have
// four requests on their way while they work on four.
//
// Mean: summed in 64 bits (an add of which costs the vector unit what one in 32 does), so that it is off by the rounding of its
// last conversion alone, however the numbers cancel.  Variance: a thread sums the squared deviations of the numbers it holds from their own
// mean, of numbers that pass from the first of them in 64 bits, and those of threads and workgroups are joined by
// M2 = sum M2_i + n_i (mean_i - mean)^2: an offset common to a group cancels before it is squared, and a number far out is no reference that
// costs the others theirs.  Everything else between load and store is fp32.
//
// Measured (16 bits): 32 x 56 x 56 x 256, relu, one launch: 21.7 us, 4.7 TB/s where a copy of that size reaches 5.1.  32 x 112 x 112 x 128,
// silu, two launches: 31.5 us of statistics behind another kernel's write-back (3.3 TB/s) and 35 for the rest, 5.9 TB/s as
// part of x comes from the caches.  32 x 28 x 28 x 512, silu, into 4 bits: 17.2 us, of which the vector unit is busy for 62 % (25
// instructions a number: two passes over the statistics, exp2 and a reciprocal, scale and codes) in turn with the loads.  One image of
// 7 x 7 x 512: 5.0 us, of which an empty launch is 2.5.
#include "norm_device.hpp"

namespace tdc {

// Number i of a channel (`last` of those at hand): four at a time are added in 32 bits where they have 16, which is exact unless one is
// 2^11 times another, the others and the fours in 64.
template <int DT>
static __device__ __forceinline__ void add_up(int i, bool last, float v, float &four, double &sum) {
    if constexpr (DT == TDC_F32) sum += v;
    else {
        four = i % 4 == 0 ? v : four + v;
        if (last || i % 4 == 3) sum += four;
    }
}

// Neighbouring channels of a thread that share a place (`run` of them, a power of two): all of them end up with its sum.
template <typename T, int V>
static __device__ __forceinline__ void join_run(T (&s)[V], int run) {
#pragma unroll
    for (int w = 1; w < V; w *= 2)
        if (run > w) {
#pragma unroll
            for (int j = 0; j < V; j += 2 * w) {
                const T both = s[j] + s[j + w];
#pragma unroll
                for (int k = 0; k < 2 * w; ++k) s[j + k] = both;
            }
        }
}

// A sum of `count` numbers and the squared deviations from their mean, over some lanes' places of one group.
struct PartSum {
    double sum;
    float m2;
    int count;
};
// `mine` places of each of `used` thread rows, from lane `at` on in steps of `step`; `lanes` of them add up.
static __device__ __forceinline__ PartSum sum_places(const Part &p, const double *sums, const float *devs, int places, int lo, int mine, int used,
                                                     int run, int at, int step, int lanes) {
    // (a thread row has one pixel more or less: reciprocals of both counts; places by multiplication, exact for so few)
    const int most = rows_of(p, 0), longer = p.rows - (most - 1) * p.R;
    const float per = __builtin_amdgcn_rcpf((float)mine);
    const double inv_most = inverse(most * run), inv_less = most > 1 ? inverse((most - 1) * run) : 0.0;
    PartSum r{0.0, 0.0f, 0};
    for (int e = at; e < mine * used; e += step) {
        const int row = (int)((e + 0.5f) * per);
        r.sum += sums[row * places + lo + e - row * mine];
        r.count += (row < longer ? most : most - 1) * run;
    }
    r.sum = team_sum(r.sum, lanes);
    r.count = team_sum(r.count, lanes);
    const double mean = r.sum * inverse(max(r.count, 1));
    for (int e = at; e < mine * used; e += step) {
        const int row = (int)((e + 0.5f) * per), i = row * places + lo + e - row * mine;
        const bool full = row < longer;
        const float d = (float)(sums[i] * (full ? inv_most : inv_less) - mean);
        r.m2 += devs[i] + (full ? most : most - 1) * run * d * d;
    }
    r.m2 = team_sum(r.m2, lanes);
    return r;
}

// The statistics of this workgroup's part of its groups: `done(i, sum, m2)` for the group i of them, in one lane, from the threads'
// sums s and squared deviations q about the means of their places.  Few groups: several waves add up one, their results meet in
// `waves`.
template <int V, typename Done>
static __device__ __forceinline__ void join_threads(const NormArgs &a, const Part &p, int n, const double (&s)[V], const float (&q)[V], int run,
                                                    double *sums, float *devs, PartSum *waves, Done done) {
    const int places = p.vecs * a.plan.places;      // of a thread row
    if (n > 0) {
        const int at = p.tr * places + p.tc * a.plan.places;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if ((j & (run - 1)) == 0) {
                sums[at + (j >> a.plan.run_shift)] = s[j];
                devs[at + (j >> a.plan.run_shift)] = q[j];
            }
    }
    __syncthreads();
    const int used = min(p.R, p.rows), all = a.plan.threads >> 6, wave = threadIdx.x >> 6;
    auto first = [&](int i) { return (max((p.g0 + i) * a.Cg, p.c0) - p.c0) >> a.plan.run_shift; };
    auto mine = [&](int i) { return shared_channels(a, p.g0 + i, p.tile) >> a.plan.run_shift; };
    if (p.ng < all) {
        const int share = small_quotient(all, p.ng), i = small_quotient(wave, share), k = wave - i * share;
        if (i < p.ng) {
            const PartSum r = sum_places(p, sums, devs, places, first(i), mine(i), used, run, k * 64 + (threadIdx.x & 63), share * 64, 64);
            if ((threadIdx.x & 63) == 0) waves[wave] = r;
        }
        __syncthreads();
        if ((int)threadIdx.x < p.ng) {
            const PartSum *const w = waves + threadIdx.x * share;
            double sum = 0.0;
            int count = 0;
            for (int k = 0; k < share; ++k) {
                sum += w[k].sum;
                count += w[k].count;
            }
            const double mean = sum * inverse(count);
            float m2 = 0.0f;
            for (int k = 0; k < share; ++k) {
                const float d = (float)(w[k].sum * inverse(max(w[k].count, 1)) - mean);
                m2 += w[k].m2 + w[k].count * d * d;
            }
            done(threadIdx.x, sum, m2);
        }
    } else {
        const Team t = team_of(a.plan.threads, p.ng);
        for (int i = t.first; i < p.ng; i += t.step) {
            const PartSum r = sum_places(p, sums, devs, places, first(i), mine(i), used, run, t.at, t.lanes, t.lanes);
            if (t.at == 0) done(i, r.sum, r.m2);
        }
    }
}

// Of vectors that stay in registers: the deviations from the mean of the place itself.
template <int DT, int V, int NV>
static __device__ __forceinline__ void held_sums(int n, typename Pack<DT, V>::type (&x)[NV], int run, double (&s)[V], float (&q)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        s[j] = 0.0;
        q[j] = 0.0f;
    }
    float four[V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (i < n) {
            float v[V];
            Pack<DT, V>::up(x[i], v);
#pragma unroll
            for (int j = 0; j < V; ++j) add_up<DT>(i, i == n - 1, v[j], four[j], s[j]);
        }
    join_run(s, run);
    pack_again(x);
    float mean[V];
    const double inv = inverse(max(n, 1) * run);
#pragma unroll
    for (int j = 0; j < V; ++j) mean[j] = (float)(s[j] * inv);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (i < n) {
            float v[V];
            Pack<DT, V>::up(x[i], v);
#pragma unroll
            for (int j = 0; j < V; ++j) q[j] = fmaf(v[j] - mean[j], v[j] - mean[j], q[j]);
        }
    join_run(q, run);
}

// Of any number of pixels: the deviations from a channel's first number, then moved to the mean of the place.  Where that first number lies far
// out the sum of squares is up to n times what remains, so it is one of doubles (which add and multiply at the rate of floats): in fp32 an
// image with one number in its corner had a variance up to 1e-3 off at 256 pixels a thread.
template <int DT, int V, int NV>
static __device__ __forceinline__ void passing_sums(const NormArgs &a, const Part &p, int n, int run, double (&s)[V], float (&q)[V]) {
    using P = Pack<DT, V>;
    if (n == 0) return;
    const Walk<DT, V> in(a.x, a.x_is, a.x_ps, p, n);
    float first[V];
    P::up(P::load(in.base, in.at), first);
    double dev[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = dev[j] = 0.0;
    typename P::type x[2][NV];
    walk<NV>(n, quotient(p.rows, p.by_R), [&](int set, int at) { in.ask(at, x[set]); }, [&](int set, int, auto some) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < some) {
                float v[V];
                P::up(x[set][i], v);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const double d = (double)v[j] - (double)first[j];
                    s[j] += d;
                    dev[j] = fma(d, d, dev[j]);
                }
            }
    });
    double own[V];
    const double inv = inverse(n);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        own[j] = s[j] * inv;      // (about the first number)
        dev[j] = fmax(dev[j] - s[j] * own[j], 0.0);
        own[j] += first[j];
        s[j] = fma(n, (double)first[j], s[j]);
    }
    join_run(s, run);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const double e = own[j] - s[j] * (inv * (1.0 / V) * a.plan.places);
        q[j] = (float)fma(n * e, e, dev[j]);
    }
    join_run(q, run);
}

// One group's (mean, rstd); the first workgroup that has it keeps them for the caller.
static __device__ __forceinline__ float2 finish_stats(const NormArgs &a, const Part &p, int g, double mean, float m2, bool keep) {
    const float2 st = make_float2((float)mean, 1.0f / sqrtf(m2 * (float)a.per_number + a.eps));
    if (keep) {
        if (a.mean) a.mean[(long long)p.image * a.groups + g] = st.x;
        if (a.rstd) a.rstd[(long long)p.image * a.groups + g] = st.y;
    }
    return st;
}
// Joins the partial results of a workgroup's groups.
static __device__ __forceinline__ void join_stats(const NormArgs &a, const Part &p, float2 *stat) {
    const Team t = team_of(a.plan.threads, p.ng);
    const NormPlan &n = a.plan;
    for (int i = t.first; i < p.ng; i += t.step) {
        const int g = p.g0 + i, tile0 = tiles_of(a, p, g).x, tiles = tiles_of(a, p, g).y;
        const NormStat *part = a.stat + ((long long)p.image * a.groups + g) * n.slots;
        double sum = 0.0;
        for (int k = 0; k < tiles; ++k)
            for (int c = t.at; c < n.chunks; c += t.lanes) sum += part[c * n.tiles_per_group + k].sum;
        const double mean = team_sum(sum, t.lanes) * a.per_number;
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
        if (t.at == 0) stat[i] = finish_stats(a, p, g, mean, m2, p.chunk == 0 && p.tile == tile0);
    }
}

// Where a thread's share of a block of 32 channels goes, and V numbers of a row into it: 32 / V neighbouring lanes hold a block.
template <int V>
struct Mx4Place {
    unsigned char *codes, *scales;      // of row 0; of the scales only in a block's first lane
    __device__ __forceinline__ Mx4Place(const NormArgs &a, int c)
        : codes(a.codes + mx4_block_at(a.rows, 0, c >> 5) + (c & 31) / 2),
          scales(c & 31 ? nullptr : a.scales + (long long)(c >> 9) * a.rows * 16 + (c >> 5 & 3) * 4 + (c >> 7 & 3)) {}
    __device__ __forceinline__ void store(long long row, const float (&v)[V]) const {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        float most = quad_larger(__uint_as_float(top));
        if (V == 4) most = larger(most, __shfl_xor(most, 4, 64));
        const int byte = mx4_scale_byte(most);
        const float divisor = mx4_divisor(byte);
        unsigned char *const to = codes + ((row >> 5) * 2048 + (row & 31) * 16);
        if constexpr (V == 8) *reinterpret_cast<unsigned *>(to) = mx4_codes(v, divisor);
        else {
            unsigned r = 0;
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], divisor, 0);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], divisor, 1);
            *reinterpret_cast<unsigned short *>(to) = (unsigned short)r;
        }
        if (scales) scales[row * 16] = (unsigned char)byte;
    }
};
// What pads a row: blocks up to a multiple of 128 numbers, scale bytes up to one of 512.
static __device__ __forceinline__ void store_mx4_padding(const NormArgs &a, const Part &p) {
    const int from = (a.C + 31) / 32, blocks = (a.C + 127) / 128 * 4, past = (a.C + 511) / 512 * 16 - from;
    for (int i = threadIdx.x; i < p.rows * past; i += a.plan.threads) {
        const int r = i / past, block = from + i - r * past;
        const long long row = (long long)p.image * a.pixels + p.row0 + r;
        if (block < blocks) *reinterpret_cast<uint4 *>(a.codes + mx4_block_at(a.rows, row, block)) = make_uint4(0, 0, 0, 0);
        a.scales[((block >> 4) * a.rows + row) * 16 + (block & 3) * 4 + (block >> 2 & 3)] = 0;
    }
}

// MODE: everything in one launch, or its first or second half.
enum { kWhole, kStats, kApply };

template <int DT, int V, int NV, int MODE, int ACT, bool MX4>
__global__ void __launch_bounds__(MODE == kWhole ? 1024 : 256) tdc_norm_kernel(const NormArgs a) {
    using P = Pack<DT, V>;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const Part p = part_of(a, V, blockIdx.x, gridDim.x);
    // (a vector past the last channel has no numbers; in 4 bits it fills a block up with zeros)
    const int c = p.c0 + p.tc * V, all = rows_of(p, p.tr), n = c < a.C ? all : 0;
    const int run = 1 << a.plan.run_shift, most = a.plan.threads * a.plan.places;
    double *const sums = reinterpret_cast<double *>(lds);
    float *const devs = reinterpret_cast<float *>(sums + most);
    PartSum *const waves = reinterpret_cast<PartSum *>(devs + most);
    float2 *const stat = MODE == kApply ? reinterpret_cast<float2 *>(lds) : reinterpret_cast<float2 *>(waves + a.plan.threads / 64);
    double s[V];
    float q[V];
    if constexpr (MODE == kStats) {
        passing_sums<DT, V, NV>(a, p, n, run, s, q);
        join_threads(a, p, n, s, q, run, sums, devs, waves, [&](int i, double sum, float m2) { a.stat[slot_of(a, p, p.g0 + i)] = NormStat{sum, m2}; });
        return;
    }
    float mean[V], scale[V], shift[V];
#pragma unroll
    for (int j = 0; j < V; ++j) mean[j] = scale[j] = shift[j] = 0.0f;
    auto constants = [&]() {
        int g[V];
        groups_of(a, c, g);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 st = stat[g[j] - p.g0];
            mean[j] = st.x;
            scale[j] *= st.y;
        }
    };
    const long long row = p.row0 + p.tr, out = p.image * a.o_is + row * a.o_ps + c, step = p.R * a.o_ps, first = p.image * (long long)a.pixels + row;
    auto finish = [&](const Mx4Place<V> &place, const typename P::type &x, int i) {
        float v[V];
        P::up(x, v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = act_of<ACT>(fmaf(v[j] - mean[j], scale[j], shift[j]));
        if constexpr (MX4) place.store(first + i * p.R, v);
        else P::store(a.out, out + i * step, P::down(v));
    };
    if constexpr (MODE == kWhole) {
        typename P::type x[NV];
        hold<DT, V, NV>(a.x, a.x_is, a.x_ps, p, n, x);
        held_sums<DT, V, NV>(n, x, run, s, q);
        if (n > 0) params<DT, V>(a, c, scale, shift);
        join_threads(a, p, n, s, q, run, sums, devs, waves, [&](int i, double sum, float m2) {
            stat[i] = finish_stats(a, p, p.g0 + i, sum * a.per_number, m2, true);
        });
        __syncthreads();
        if (all > 0) {
            if (n > 0) constants();
            const Mx4Place<V> place(a, c);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i < all) finish(place, x[i], i);
        }
    } else {
        if (n > 0) params<DT, V>(a, c, scale, shift);
        join_stats(a, p, stat);
        __syncthreads();
        if (all > 0) {
            if (n > 0) constants();
            const Mx4Place<V> place(a, c);
            Part there = p;
            if (n == 0) there.tc = 0;
            const Walk<DT, V> in(a.x, a.x_is, a.x_ps, there, all, true);
            typename P::type x[2][NV];
            walk<NV>(all, quotient(p.rows, p.by_R), [&](int set, int at) { in.ask(at, x[set]); }, [&](int set, int at, auto some) {
                if (MX4 && a.plan.round) {
#pragma unroll
                    for (int i = 0; i < NV; ++i)
                        if (n == 0) x[set][i] = typename P::type{};
                }
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (i < some) finish(place, x[set][i], all - 1 - at - i);
            });
        }
    }
    if (MX4 && p.c0 + p.width == a.C) store_mx4_padding(a, p);
}

// The second half into 4 bits where the channels are no whole number of vectors: a thread takes a block of 32 channels of a pixel.
template <int DT, int ACT>
__global__ void __launch_bounds__(256) tdc_norm_blocks_kernel(const NormArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    using T = typename Num<DT>::type;
    const Part p = part_of(a, a.plan.vec, blockIdx.x, gridDim.x);
    float2 *const stat = reinterpret_cast<float2 *>(lds);
    join_stats(a, p, stat);
    __syncthreads();
    const int blocks = (p.width + 31) / 32;      // (tiles start at multiples of 32 channels)
    for (int i = threadIdx.x; i < p.rows * blocks; i += a.plan.threads) {
        const int r = i / blocks, kb = i - r * blocks, n = min(32, p.width - kb * 32), c = p.c0 + kb * 32;
        const T *const in = reinterpret_cast<const T *>(a.x) + p.image * a.x_is + (long long)(p.row0 + r) * a.x_ps + c;
        const long long row = (long long)p.image * a.pixels + p.row0 + r, block = c / 32;
        float v[32], top = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            v[j] = 0.0f;
            if (j < n) {
                const float2 st = stat[quotient(c + j, a.plan.by_group) - p.g0];
                const float gamma = a.gamma ? param<DT>(a.gamma, c + j, a.param_dtype) : 1.0f;
                const float beta = a.beta ? param<DT>(a.beta, c + j, a.param_dtype) : 0.0f;
                v[j] = act_of<ACT>(fmaf(Num<DT>::up(in[j]) - st.x, st.y * gamma, beta));
            }
            top = larger(top, v[j]);
        }
        const int byte = mx4_scale_byte(top);
        const float divisor = mx4_divisor(byte);
        *reinterpret_cast<uint4 *>(a.codes + mx4_block_at(a.rows, row, block)) =
            make_uint4(mx4_codes(v, divisor), mx4_codes(v + 8, divisor), mx4_codes(v + 16, divisor), mx4_codes(v + 24, divisor));
        a.scales[((block >> 4) * a.rows + row) * 16 + (block & 3) * 4 + (block >> 2 & 3)] = (unsigned char)byte;
    }
    if (p.c0 + p.width == a.C) store_mx4_padding(a, p);
}

template <int DT, int V, int NV, int ACT, bool MX4>
static int run(const NormArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)a.plan.chunks * a.plan.tiles * a.batch, threads = a.plan.threads;
    if (a.plan.whole) tdc_norm_kernel<DT, V, NV, kWhole, ACT, MX4><<<grid, threads, a.plan.lds, s>>>(a);
    else {
        tdc_norm_kernel<DT, V, 4, kStats, TDC_ACT_NONE, false><<<grid, threads, a.plan.lds, s>>>(a);
        tdc_norm_kernel<DT, V, 4, kApply, ACT, MX4><<<grid, threads, a.plan.lds, s>>>(a);
    }
    return (int)hipGetLastError();
}
template <int DT, int V, int ACT>
static int run_blocks(const NormArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)a.plan.chunks * a.plan.tiles * a.batch, threads = a.plan.threads;
    tdc_norm_kernel<DT, V, 4, kStats, TDC_ACT_NONE, false><<<grid, threads, a.plan.lds, s>>>(a);
    tdc_norm_blocks_kernel<DT, ACT><<<grid, threads, a.plan.lds, s>>>(a);
    return (int)hipGetLastError();
}
template <int DT, int ACT>
static int by_shape(const NormArgs &a, hipStream_t s) {
    constexpr int VM = DT == TDC_F32 ? 4 : 8;
    const NormPlan &n = a.plan;
    if (a.codes && n.vec != VM) {
        return n.vec == 2 ? run_blocks<DT, 2, ACT>(a, s) : run_blocks<DT, 1, ACT>(a, s);
    }
    if (a.codes) return n.held == 4 ? run<DT, VM, 4, ACT, true>(a, s) : run<DT, VM, 16, ACT, true>(a, s);
    if (n.vec == VM) return n.held == 4 ? run<DT, VM, 4, ACT, false>(a, s) : run<DT, VM, 16, ACT, false>(a, s);
    return n.vec == 2 ? run<DT, 2, 16, ACT, false>(a, s) : run<DT, 1, 16, ACT, false>(a, s);
}
template <int DT>
static int by_act(const NormArgs &a, hipStream_t s) {
    if (a.act == TDC_ACT_RELU) return by_shape<DT, TDC_ACT_RELU>(a, s);
    if (a.act == TDC_ACT_SILU) return by_shape<DT, TDC_ACT_SILU>(a, s);
    return by_shape<DT, TDC_ACT_NONE>(a, s);
}

int launch_norm_forward(const NormArgs &a, int dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == TDC_F32) return by_act<TDC_F32>(a, s);
    if (dtype == TDC_F16) return by_act<TDC_F16>(a, s);
    return by_act<TDC_BF16>(a, s);
}

}  // namespace tdc
