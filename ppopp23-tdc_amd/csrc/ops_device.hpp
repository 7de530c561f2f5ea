// Device-side pieces shared by the channels-last operators: numbers in memory to fp32 and back, activations.
#pragma once
#include <hip/hip_runtime.h>

#include "ops_internal.hpp"

namespace tdc {

template <int DT>
struct Num;
template <>
struct Num<TDC_F32> {
    using type = float;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Num<TDC_F16> {
    using type = _Float16;
    static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }
};
template <>
struct Num<TDC_BF16> {
    using type = __bf16;
    static __device__ __forceinline__ float up(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 down(float v) { return (__bf16)v; }
};

// V neighbouring numbers as one request, which needs the alignment of one of them.
template <int DT, int V>
struct Pack {
    using T = typename Num<DT>::type;
    typedef T type __attribute__((ext_vector_type(V)));
    typedef T mem_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    static __device__ __forceinline__ void up(const type &p, float (&v)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = Num<DT>::up(p[i]);
    }
    static __device__ __forceinline__ type down(const float (&v)[V]) {
        type p;
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = Num<DT>::down(v[i]);
        return p;
    }
    static __device__ __forceinline__ type load(const void *base, long long at) {
        return *reinterpret_cast<const mem_t *>(reinterpret_cast<const T *>(base) + at);
    }
    static __device__ __forceinline__ void store(void *base, long long at, const type &p) {
        *reinterpret_cast<mem_t *>(reinterpret_cast<T *>(base) + at) = p;
    }
};
// (a vector of one number is the number)
template <int DT>
struct Pack<DT, 1> {
    using T = typename Num<DT>::type;
    using type = T;
    static __device__ __forceinline__ void up(const type &p, float (&v)[1]) { v[0] = Num<DT>::up(p); }
    static __device__ __forceinline__ type down(const float (&v)[1]) { return Num<DT>::down(v[0]); }
    static __device__ __forceinline__ type load(const void *base, long long at) { return reinterpret_cast<const T *>(base)[at]; }
    static __device__ __forceinline__ void store(void *base, long long at, const type &p) { reinterpret_cast<T *>(base)[at] = p; }
};

// One parameter (gamma, beta, bias): fp32 or the tensor's type.
template <int DT>
__device__ __forceinline__ float param(const void *p, long long i, int param_dtype) {
    if constexpr (DT != TDC_F32)
        if (param_dtype != TDC_F32) return Num<DT>::up(reinterpret_cast<const typename Num<DT>::type *>(p)[i]);
    return reinterpret_cast<const float *>(p)[i];
}

// 1 / (1 + e^-z), by the exponential to base two and the reciprocal of the hardware (1 ulp each).  Its argument z log2 e is rounded once
// to fp32, which makes e^-z |z| 2^-24 of itself less exact (1e-6 at z = -20): where |z| is large the activation is small against the
// norm's own error of z, by which its results are judged.
__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
    if constexpr (ACT == TDC_ACT_RELU) return z < 0.0f ? 0.0f : z;      // (a NaN stays one)
    if constexpr (ACT == TDC_ACT_SILU) return z * sigmoid(z);
    return z;
}
// dy times the derivative at z.  "relu" chooses: a NaN passes dy on, and an infinite dy where nothing passes is 0.
// "silu": from 128 on s is 0 or 1 to the last bit, and so is the derivative.  A z kept in 16 bits may have become infinite there,
// which times 0 would be a NaN; where z is one, s is.
template <int ACT>
__device__ __forceinline__ float act_back(float dy, float z) {
    if constexpr (ACT == TDC_ACT_RELU) return z <= 0.0f ? 0.0f : dy;
    if constexpr (ACT == TDC_ACT_SILU) {
        const float s = sigmoid(z);
        return dy * (s * (1.0f + __builtin_amdgcn_fmed3f(z, -128.0f, 128.0f) * (1.0f - s)));
    }
    return dy;
}

// ---- blocks of 32 numbers in 4 bits ----

// The scale byte of a block from its largest magnitude.  (The exponent field of a number below 2^-126 reads as one too
// many, but every such block has the smallest scale.)
__device__ __forceinline__ int mx4_scale_byte(float top) {
    const int e = (int)(__float_as_uint(top) >> 23);
    return e == 255 ? 255 : max(e - 2, 0);
}
__device__ __forceinline__ float mx4_scale(int byte) {
    return byte == 255 ? __builtin_nanf("") : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((unsigned)byte << 23);
}
// The larger magnitude, a NaN if either is one: magnitudes compare as integers, NaN above infinity.
__device__ __forceinline__ float larger(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

// What a block's numbers are divided by (one that stands for NaNs: by anything).
__device__ __forceinline__ float mx4_divisor(int byte) { return byte == 255 ? 1.0f : mx4_scale(byte); }
// Eight codes.  (The instruction rounds to nearest even and saturates.)
__device__ __forceinline__ unsigned mx4_codes(const float *v, float divisor) {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], divisor, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], divisor, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], divisor, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], divisor, 3);
}
// What eight codes stand for.
__device__ __forceinline__ void mx4_values(unsigned codes, float scale, float (&v)[8]) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
}
// The largest magnitude of four neighbouring lanes (quad_perm: each lane's neighbour, then the other pair).
__device__ __forceinline__ float quad_larger(float top) {
    top = larger(top, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, top), 0xB1, 0xf, 0xf, true)));
    return larger(top, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, top), 0x4E, 0xf, 0xf, true)));
}

// ---- blocks of 32 numbers in 8 bits (E4M3; scales as above) ----

__device__ __forceinline__ int mx8_scale_byte(float top) {
    const int e = (int)(__float_as_uint(top) >> 23);
    return e == 255 ? 255 : max(e - 8, 0);
}
// Eight codes.  (The instruction rounds to nearest even, but makes NaNs of what rounds past 448: those saturate before.)
__device__ __forceinline__ uint2 mx8_codes(const float *v, float divisor) {
    typedef short s2_t __attribute__((ext_vector_type(2)));
    const float most = 448.0f * divisor;
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_fmed3f(v[i], -most, most);
    s2_t lo = {0, 0}, hi = {0, 0};
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, c[0], c[1], divisor, false);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, c[2], c[3], divisor, true);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, c[4], c[5], divisor, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, c[6], c[7], divisor, true);
    return make_uint2(__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi));
}
// What eight codes stand for.
__device__ __forceinline__ void mx8_values(uint2 codes, float scale, float (&v)[8]) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, true);
    const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, true);
    v[0] = a[0] * scale, v[1] = a[1] * scale, v[2] = b[0] * scale, v[3] = b[1] * scale;
    v[4] = c[0] * scale, v[5] = c[1] * scale, v[6] = d[0] * scale, v[7] = d[1] * scale;
}

// The quotient of two numbers below 2^20: an approximate reciprocal is near enough for those.
static __device__ __forceinline__ int small_quotient(int n, int d) { return (int)((n + 0.5f) * __builtin_amdgcn_rcpf((float)d)); }

}  // namespace tdc
