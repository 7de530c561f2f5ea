// Device-side pieces shared by the matrix products (4-bit, 8-bit, 16-bit): requests into LDS, waits, and how a tile's sums
// leave.
#pragma once
#include <type_traits>

#include "ops_device.hpp"

namespace tdc {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i8_t __attribute__((ext_vector_type(8)));
typedef float f16_t __attribute__((ext_vector_type(16)));

// Eight neighbouring numbers of a row as one request.
template <int DT>
struct Eight {
    using T = typename Num<DT>::type;
    typedef T vec_t __attribute__((ext_vector_type(8)));
    typedef T mem_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
// Eight neighbouring numbers of a row of which `left` (at least 1) are there: whole, or by fours, twos and one.  WHOLE: all eight are.
template <int DT, bool WHOLE>
static __device__ __forceinline__ typename Eight<DT>::vec_t load8(const void *base, long long at, long long left) {
    using T = typename Num<DT>::type;
    const T *from = reinterpret_cast<const T *>(base) + at;
    if (WHOLE || left >= 8) return *reinterpret_cast<const typename Eight<DT>::mem_t *>(from);
    typename Pack<DT, 4>::type four = {};
    typename Pack<DT, 2>::type two = {};
    T one = {};
    const int l = (int)left;
    if (l & 4) four = Pack<DT, 4>::load(from, 0);
    if (l & 2) two = Pack<DT, 2>::load(from, l & 4);
    if (l & 1) one = from[l & 6];
    typename Eight<DT>::vec_t r = {};
    if (l & 4) r = typename Eight<DT>::vec_t{four[0], four[1], four[2], four[3], l & 2 ? two[0] : one, two[1], l & 2 ? one : T{}, T{}};
    else r = typename Eight<DT>::vec_t{l & 2 ? two[0] : one, two[1], l & 2 ? one : T{}, T{}, T{}, T{}, T{}, T{}};
    return r;
}
template <int DT, bool WHOLE>
static __device__ __forceinline__ void store8(void *base, long long at, long long left, const typename Eight<DT>::vec_t &v) {
    using T = typename Num<DT>::type;
    T *const to = reinterpret_cast<T *>(base) + at;
    if (WHOLE || left >= 8) {
        *reinterpret_cast<typename Eight<DT>::mem_t *>(to) = v;
        return;
    }
    const int l = (int)left;
    if (l & 4) Pack<DT, 4>::store(to, 0, typename Pack<DT, 4>::type{v[0], v[1], v[2], v[3]});
    const typename Pack<DT, 4>::type rest = {l & 4 ? v[4] : v[0], l & 4 ? v[5] : v[1], l & 4 ? v[6] : v[2], T{}};
    if (l & 2) Pack<DT, 2>::store(to, l & 4, typename Pack<DT, 2>::type{rest[0], rest[1]});
    if (l & 1) to[l & 6] = l & 2 ? rest[2] : rest[0];
}
// The row of w that is row r of a block: bits 2 and 3 change places, which makes a lane's outputs 8 i .. 8 i + 7 neighbours.
static __device__ __forceinline__ int weight_row(int r) { return (r & 19) | (r & 4) << 1 | (r & 8) >> 1; }

// A request straight into LDS: 16 bytes a lane, from `at` + `offset` on, in the order of the lanes.
static __device__ __forceinline__ void bring(const unsigned char *base, int at, int offset, unsigned char *to) {
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(base), 0, 0x7fffffff, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16, at, offset, 0, 0);
}
// Waits until all but the wave's newest `left` requests have come and its LDS operations are done, then for the other waves.  (A fence in
// place of the waits would wait for every request.)
template <int left>
static __device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((left & 15) | (left >> 4) << 14 | 7 << 4);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
template <int DT>
static __device__ __forceinline__ float bias_of(const ProductOut &a, long long n, bool wanted) {
    return wanted && a.bias && n < a.N ? param<DT>(a.bias, n, a.bias_dtype) : 0.0f;
}

// A wave's outputs from row m on and from column n on; `bias` is that of its columns, `stage` its own 4 KiB NB of LDS.  Z: what the activation
// is taken of leaves too, in y's 16 bits (the slope is taken there; in 32 it would cost twice y's bytes); PART: sums that others join, and nothing with them.  Of a block a lane
// has row r of x, and of w 16 u + 8 q .. 16 u + 8 q + 7, u = 0, 1.  32 rows at a time go through LDS, where a lane takes eight outputs of a
// row and its neighbours those beside them: residuals and outputs are whole cache lines.  (The first halves of a row's eights lie
// before the second ones, 16 bytes moved by the row, so that neither side meets a bank twice.)  The residuals of the next rows are on
// their way while these are finished.
// A tile runs this once, with one wave a vector unit where tiles are large: instructions count, and so does the code itself, which comes from
// memory.  The rows loop, one copy serves all activations, whole tiles have no bounds to check (64 tiles of 256 x 256 with a sum of 32:
// 17.3 us unrolled, with a copy for each activation; 11.7 now).
template <int DT, int MB, int NB, bool Z = false, bool PART = false>
static __device__ __forceinline__ void finish_tile(const ProductOut &a, const f16_t (&acc)[NB][MB], long long m, long long n, const float *bias,
                                                   unsigned char *stage) {
    constexpr int kAcross = NB * 4, kDown = 64 / kAcross, kTurns = 32 / kDown;     // lanes of a row, rows at a time
    constexpr int kAtOnce = kTurns < 4 ? kTurns : 4, kGroups = kTurns / kAtOnce;
    using V = typename Eight<DT>::vec_t;
    const int lane = threadIdx.x & 63, r = lane & 31, q = lane >> 5, down = lane / kAcross, c = lane % kAcross * 8;
    auto place = [&](int row, int eight, int half) {
        return reinterpret_cast<float4 *>(stage + row * NB * 128 + ((half * kAcross + eight) ^ (row & 15 & (NB * 8 - 1))) * 16);
    };
    const float4 lo = *reinterpret_cast<const float4 *>(bias + c), hi = *reinterpret_cast<const float4 *>(bias + c + 4);
    const float add[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const long long left = a.N - n - c;
    auto finish = [&](auto whole, auto with_residual) {
        constexpr bool kWhole = decltype(whole)::value, kResidual = decltype(with_residual)::value;
        // (this lane's places, from row to row; a row past the last is not touched)
        long long y_at = (m + down) * a.y_stride + n + c, z_at = (m + down) * a.z_stride + n + c, r_at = (m + down) * a.r_stride + n + c;
        int rows = kWhole || left > 0 ? (int)min((long long)32 * MB, a.M - m) - down : 0;      // of this lane, from `down` on
        V now[kAtOnce], next[kAtOnce];
        int asked = rows;
        auto ask = [&] {
#pragma unroll
            for (int s = 0; s < kAtOnce; ++s) {
                if constexpr (kWhole) next[s] = load8<DT, true>(a.residual, r_at, left);
                else {
                    next[s] = V{};
                    if (asked > 0) next[s] = load8<DT, false>(a.residual, r_at, left);
                }
                r_at += kDown * a.r_stride;
                asked -= kDown;
            }
        };
        if constexpr (kResidual) ask();
#pragma unroll
        for (int i = 0; i < MB; ++i) {
#pragma unroll
            for (int k = 0; k < 2 * NB; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int e = 8 * (k % 2) + 4 * h;
                    const f16_t &v = acc[k / 2][i];
                    *place(r, k * 2 + q, h) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                }
            asm volatile("" ::: "memory");      // (a wave's own LDS operations come in order)
#pragma unroll 1
            for (int g = 0; g < kGroups; ++g) {
                if constexpr (kResidual) {
#pragma unroll
                    for (int s = 0; s < kAtOnce; ++s) now[s] = next[s];
                    if (i * kGroups + g + 1 < MB * kGroups) ask();
                }
#pragma unroll
                for (int s = 0; s < kAtOnce; ++s) {
                    const int row = (g * kAtOnce + s) * kDown + down;
                    const float4 u = *place(row, c / 8, 0), w = *place(row, c / 8, 1);
                    float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
                    V out, sum;
                    if constexpr (!PART) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            v[j] += add[j];
                            if constexpr (kResidual) v[j] += Num<DT>::up(now[s][j]);
                            if constexpr (Z) sum[j] = Num<DT>::down(v[j]);
                        }
                        if (a.act == TDC_ACT_RELU) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = act_of<TDC_ACT_RELU>(v[j]);
                        } else if (a.act == TDC_ACT_SILU) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = act_of<TDC_ACT_SILU>(v[j]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) out[j] = Num<DT>::down(v[j]);
                    if (kWhole || rows > 0) {
                        store8<DT, kWhole>(a.y, y_at, left, out);
                        if constexpr (Z) store8<DT, kWhole>(a.z, z_at, left, sum);
                    }
                    rows -= kDown;
                    y_at += kDown * a.y_stride;
                    if constexpr (Z) z_at += kDown * a.z_stride;
                }
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const std::true_type yes;
    const std::false_type no;
    const bool whole = m + 32 * MB <= a.M && n + 32 * NB <= a.N;
    if constexpr (PART) {
        if (whole) finish(yes, no);
        else finish(no, no);
    } else if (a.residual) {
        if (whole) finish(yes, yes);
        else finish(no, yes);
    } else if (whole) finish(yes, no);
    else finish(no, no);
}

// Lets a kernel have more than 64 KiB of LDS; once per kernel and device.
static int allow_lds(const void *fn, int bytes, unsigned long long &done) {
    int device = 0;
    if (hipError_t e = hipGetDevice(&device)) return (int)e;
    const unsigned long long bit = 1ull << (device & 63);
    if (__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit) return 0;
    if (hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return (int)e;
    __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
    return 0;
}

}  // namespace tdc
