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
// The residual of eight neighbouring outputs of a row: zeros where there is none (rows from M on, outputs from N on).
template <int DT>
static __device__ __forceinline__ typename Eight<DT>::vec_t residual8(const ProductOut &a, long long m, long long n) {
    using T = typename Num<DT>::type;
    typename Eight<DT>::vec_t r = {};
    if (a.residual && m < a.M) {
        const T *const from = reinterpret_cast<const T *>(a.residual) + m * a.r_stride + n;
        if (n + 8 <= a.N) r = *reinterpret_cast<const typename Eight<DT>::mem_t *>(from);
        else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (n + i < a.N) r[i] = from[i];
        }
    }
    return r;
}
template <int DT>
static __device__ __forceinline__ void store8(void *base, long long at, long long left, const typename Eight<DT>::vec_t &v) {
    using T = typename Num<DT>::type;
    T *const to = reinterpret_cast<T *>(base) + at;
    if (left >= 8) *reinterpret_cast<typename Eight<DT>::mem_t *>(to) = v;
    else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < left) to[i] = v[i];
    }
}
// Eight neighbouring outputs of a row (those before N): residual on sums with the bias, activation, store; what the activation
// was taken of besides if Z.
template <int DT, int ACT, bool Z>
static __device__ __forceinline__ void finish8(const ProductOut &a, long long m, long long n, const float (&v)[8], typename Eight<DT>::vec_t r) {
    typename Eight<DT>::vec_t out, sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float z = v[i] + Num<DT>::up(r[i]);
        out[i] = Num<DT>::down(act_of<ACT>(z));
        sum[i] = Num<DT>::down(z);
    }
    store8<DT>(a.y, m * a.y_stride + n, a.N - n, out);
    if constexpr (Z) store8<DT>(a.z, m * a.z_stride + n, a.N - n, sum);
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

// A wave's outputs from row m on and from column n on; `bias` is that of its columns, `stage` its own 4 KiB NB of LDS (PART: sums that others join, without an activation).  Of a block a lane
// has row r of x, and of w 16 u + 8 q .. 16 u + 8 q + 7, u = 0, 1.  32 rows at a time go through LDS, where a lane takes eight outputs of a
// row and its neighbours those beside them: residuals and outputs are whole cache lines.  (The first halves of a row's eights lie
// before the second ones, 16 bytes moved by the row, so that neither side meets a bank twice.)  The residuals of the next 32 rows are on
// their way while these are finished.
template <int DT, int MB, int NB, bool Z = false, bool PART = false>
static __device__ __forceinline__ void finish_tile(const ProductOut &a, const f16_t (&acc)[NB][MB], long long m, long long n, const float *bias,
                                                   unsigned char *stage) {
    constexpr int kAcross = NB * 4, kDown = 64 / kAcross, kTurns = 32 / kDown;     // lanes of a row, rows at a time
    const int lane = threadIdx.x & 63, r = lane & 31, q = lane >> 5, down = lane / kAcross, c = lane % kAcross * 8;
    auto place = [&](int row, int eight, int half) {
        return reinterpret_cast<float4 *>(stage + row * NB * 128 + ((half * kAcross + eight) ^ (row & 15 & (NB * 8 - 1))) * 16);
    };
    const float4 lo = *reinterpret_cast<const float4 *>(bias + c), hi = *reinterpret_cast<const float4 *>(bias + c + 4);
    const float add[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    auto finish = [&](auto act) {
        typename Eight<DT>::vec_t res[2][kTurns];
        auto ask = [&](int i) {
#pragma unroll
            for (int s = 0; s < kTurns; ++s) res[i & 1][s] = residual8<DT>(a, m + i * 32 + s * kDown + down, n + c);
        };
        ask(0);
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
            if (i + 1 < MB) ask(i + 1);
            asm volatile("" ::: "memory");      // (a wave's own LDS operations come in order)
#pragma unroll
            for (int s = 0; s < kTurns; ++s) {
                const int row = s * kDown + down;
                const float4 u = *place(row, c / 8, 0), w = *place(row, c / 8, 1);
                const float v[8] = {u.x + add[0], u.y + add[1], u.z + add[2], u.w + add[3], w.x + add[4], w.y + add[5], w.z + add[6], w.w + add[7]};
                if (m + i * 32 + row < a.M && n + c < a.N) finish8<DT, decltype(act)::value, Z>(a, m + i * 32 + row, n + c, v, res[i & 1][s]);
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if constexpr (PART) finish(std::integral_constant<int, TDC_ACT_NONE>{});
    else if (a.act == TDC_ACT_RELU) finish(std::integral_constant<int, TDC_ACT_RELU>{});
    else if (a.act == TDC_ACT_SILU) finish(std::integral_constant<int, TDC_ACT_SILU>{});
    else finish(std::integral_constant<int, TDC_ACT_NONE>{});
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
