// Device-side pieces shared by the group norm kernels: what a workgroup owns, its pixels in registers, sums over groups.
#pragma once
#include <type_traits>

#include "ops_device.hpp"

namespace tdc {

// The quotient of a number below 2^32.
static __device__ __forceinline__ unsigned quotient(unsigned n, const Divisor &d) {
    const unsigned q = __umulhi(n, d.mul);
    return q + (n - q * d.by >= d.by);
}
// 1 / n to the last bits of a double: two steps of Newton's method from 23 bits.
static __device__ __forceinline__ double inverse(int n) {
    double r = __builtin_amdgcn_rcpf((float)n);
    r = fma(r, fma(-(double)n, r, 1.0), r);
    return fma(r, fma(-(double)n, r, 1.0), r);
}

// What a workgroup owns.
struct Part {
    int image, tile, chunk;
    int c0, width, vecs;     // its channels, in all and as vectors
    int tr, tc, R;           // this thread's pixel row and vector, rows at a time (threads past them idle: tr >= R)
    Divisor by_R;
    int row0, rows;          // its pixels
    int g0, ng;              // its groups
};

// Workgroups are dealt to the dies round robin: each die gets a run of neighbouring tiles, which share cache lines.
static __device__ __forceinline__ Part part_of(const NormArgs &a, int vec, unsigned block, unsigned blocks) {
    Part p;
    const NormPlan &n = a.plan;
    const unsigned die = block & 7, longer = blocks & 7;
    const unsigned idx = die * (blocks >> 3) + min(die, longer) + (block >> 3);
    const unsigned across = quotient(idx, n.by_tiles);
    p.tile = idx - across * n.tiles;
    p.image = quotient(across, n.by_chunks);
    p.chunk = across - p.image * n.chunks;
    p.c0 = p.tile * n.unit;
    p.width = min(n.unit, a.C - p.c0);
    p.vecs = ((p.width + n.round) & ~n.round) >> __builtin_ctz(vec);
    p.by_R = n.by_rows[p.width < n.unit];
    p.R = p.by_R.by;
    p.tr = small_quotient(threadIdx.x, p.vecs);
    p.tc = threadIdx.x - p.tr * p.vecs;
    p.row0 = p.chunk * n.chunk_rows;
    p.rows = min(n.chunk_rows, a.pixels - p.row0);
    p.g0 = quotient(p.c0, n.by_group);
    p.ng = quotient(p.c0 + p.width - 1, n.by_group) - p.g0 + 1;
    return p;
}
// Pixels of thread row r.
static __device__ __forceinline__ int rows_of(const Part &p, int r) { return r < p.rows && r < p.R ? quotient(p.rows - r + p.R - 1, p.by_R) : 0; }
// The groups of a thread's V channels from c on.
template <int V>
static __device__ __forceinline__ void groups_of(const NormArgs &a, int c, int (&g)[V]) {
    g[0] = quotient(c, a.plan.by_group);
    int in = c - g[0] * a.Cg;
#pragma unroll
    for (int j = 1; j < V; ++j) {
        const bool next = ++in == a.Cg;
        g[j] = g[j - 1] + next;
        if (next) in = 0;
    }
}

// This thread's vectors of a tensor, all requested at once.
template <int DT, int V, int NV>
static __device__ __forceinline__ void hold(const void *base, long long image_stride, long long pixel_stride, const Part &p, int n,
                                            typename Pack<DT, V>::type (&v)[NV]) {
    const long long at = p.image * image_stride + (long long)(p.row0 + p.tr) * pixel_stride + p.c0 + p.tc * V, step = p.R * pixel_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        v[i] = typename Pack<DT, V>::type{};
        if (i < n) v[i] = Pack<DT, V>::load(base, at + i * step);
    }
}

// A thread's pixels of a tensor one after the other, or from its last one back.  (The second launch goes back: it meets first what the
// first one has left in the caches last.  32 x 112 x 112 x 128 numbers of 16 bits, both launches: 70 us one way, 67 back.)
template <int DT, int V>
struct Walk {
    const void *base;
    long long at, step;
    int last;
    __device__ __forceinline__ Walk(const void *tensor, long long image_stride, long long pixel_stride, const Part &p, int n, bool back = false)
        : base(tensor), at(p.image * image_stride + (long long)(p.row0 + p.tr) * pixel_stride + p.c0 + p.tc * V), step(p.R * pixel_stride), last(n - 1) {
        if (back) {
            at += last * step;
            step = -step;
        }
    }
    // (the pixels past the last repeat it: requests without a branch, so that the compiler can count them)
    template <int NV>
    __device__ __forceinline__ void ask(int first, typename Pack<DT, V>::type (&v)[NV]) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = Pack<DT, V>::load(base, at + min(first + i, last) * step);
    }
};
// Pixels 0 .. n - 1 of a thread that has some: `ask(set, at)` requests those from `at` on into one of two sets of NV, `use(set, at, some)`
// takes the first `some` of them.  While one set is worked on the other is on its way; in the rounds that all threads have (`all`
// pixels) nothing is conditional, and `some` is a constant NV.
template <int NV, typename Ask, typename Use>
static __device__ __forceinline__ void walk(int n, int all, Ask ask, Use use) {
    using All = std::integral_constant<int, NV>;
    ask(0, 0);
    int at = 0;
    for (; at + 2 * NV <= all; at += 2 * NV) {
        ask(1, at + NV);
        use(0, at, All{});
        ask(0, at + 2 * NV);
        use(1, at + NV, All{});
    }
    for (; at < n; at += 2 * NV) {
        ask(1, at + NV);
        use(0, at, min(n - at, NV));
        ask(0, at + 2 * NV);
        if (at + NV < n) use(1, at + NV, min(n - at - NV, NV));
    }
}

// Makes a thread's vectors new to the compiler, which would else keep all of them unpacked from one use to the next.
template <typename T, int NV>
static __device__ __forceinline__ void pack_again(T (&v)[NV]) {
    if constexpr (sizeof(T) == 16) {
        typedef int i4_t __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            i4_t w = __builtin_bit_cast(i4_t, v[i]);
            asm volatile("" : "+v"(w));
            v[i] = __builtin_bit_cast(T, w);
        }
    }
}

// So many lanes work on one group (a power of two, at most a wave), and this thread's place among them.
struct Team {
    int lanes, at, first, step;
};
// The first of the tiles that share a group of this workgroup, and how many they are.
static __device__ __forceinline__ int2 tiles_of(const NormArgs &a, const Part &p, int g) {
    if (a.plan.tiles_per_group == 1) return make_int2(p.tile, 1);
    const int first = g * a.Cg / a.plan.unit;
    return make_int2(first, ((g + 1) * a.Cg - 1) / a.plan.unit - first + 1);
}
static __device__ __forceinline__ Team team_of(int threads, int ng) {
    Team t;
    int shift = 6;
    while (shift && ng << shift > threads) --shift;
    t.lanes = 1 << shift;
    t.at = threadIdx.x & (t.lanes - 1);
    t.first = threadIdx.x >> shift;
    t.step = threads >> shift;
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
    return ((long long)p.image * a.groups + g) * a.plan.slots + p.chunk * a.plan.tiles_per_group + (p.tile - tiles_of(a, p, g).x);
}

// Parameters of a thread's channels.
template <int DT, int V>
static __device__ __forceinline__ void params(const NormArgs &a, int c, float (&gamma)[V], float (&beta)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        gamma[j] = a.gamma ? param<DT>(a.gamma, c + j, a.param_dtype) : 1.0f;
        beta[j] = a.beta ? param<DT>(a.beta, c + j, a.param_dtype) : 0.0f;
    }
}

}  // namespace tdc
