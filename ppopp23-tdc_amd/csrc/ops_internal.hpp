// Declarations shared by the channels-last operators' kernels (group_norm.hip, mx4.hip, mx4_product.hip) and their C entry
// points (ops_api.cpp).  Nothing here is exported.
#pragma once

#include <cstddef>
#include <cstdint>

#include <hip/hip_runtime.h>

#include "tdc.h"

namespace tdc {

inline int dtype_bytes(int dtype) { return dtype == TDC_F32 ? 4 : 2; }
inline long long round_up(long long v, long long to) { return (v + to - 1) / to * to; }

// Numbers of a row in 4 bits, rounded up to the 128 of one matrix instruction.
inline long long mx4_padded(long long K) { return round_up(K, 128); }
// Code bytes of `rows` rows, and the place of block b (of 32 numbers) of a row.
inline long long mx4_code_bytes(long long rows, long long K) { return round_up(rows, 32) * mx4_padded(K) / 2; }
__host__ __device__ inline long long mx4_block_at(long long rows, long long row, long long b) {
    return ((b >> 2) * ((rows + 31) >> 5) + (row >> 5)) * 2048 + (b & 3) * 512 + (row & 31) * 16;
}
// Scale bytes of a row.
inline long long mx4_scale_bytes(long long K) { return round_up(K, 512) / 32; }

// A divisor known before the launch, for quotients of unsigned numbers without a division (of which the compiler makes 25
// instructions): mul = floor(2^32 / by) gives the quotient or one less.
struct Divisor {
    unsigned by, mul;
};

// How a norm's work is dealt out.  A workgroup of `threads` owns `unit` channels (unit / vec vectors, a thread each) of `chunk_rows`
// pixels of one image, at most `held` pixels a thread, which it keeps in registers.  Where one workgroup holds all pixels
// (chunks = 1) a norm is one launch; else `slots` partial results per image and group meet in a second one.
struct NormPlan {
    int vec;            // channels a thread moves at once
    int unit;           // channels of a workgroup
    int tiles;          // workgroups across the channels
    int tiles_per_group;// at most so many of them share a group (1 unless a group is wider than a workgroup)
    int threads;
    int held;           // the kernel's registers: pixels a thread (of x, and of dy)
    int chunks;         // workgroups along the pixels of an image
    int chunk_rows;
    int slots;          // chunks * tiles_per_group
    int places;         // sums a thread keeps apart: its vector may span groups
    int lds;            // bytes
    bool whole;         // one workgroup has all pixels and channels of its groups
    int round;          // 31 where a row's last block of 32 is not full: its vectors are counted as if it were, else 0
    int run_shift;      // log2 of the channels of a vector that share a place
    Divisor by_tiles, by_chunks, by_group;
    Divisor by_rows[2]; // the pixels that its threads move at a time: a workgroup of `unit` channels, the last one across the channels
};

// Partial statistics of one group: the sum, and the squared deviations from its mean.
struct NormStat {
    double sum;
    float m2, unused;
};

struct NormArgs {
    const void *x, *dy, *gamma, *beta;
    void *out;                      // y or dx
    float *mean, *rstd;
    float *dgamma, *dbeta;
    NormStat *stat;                 // forward: [image][group][slot]
    float2 *part;                   // backward: the same places, sums of gamma dz and gamma dz xh
    float *chan;                    // backward: [image][chunk][2][C]
    unsigned char *codes, *scales;  // forward in 4 bits
    long long x_ps, x_is, o_ps, o_is, d_ps, d_is;
    long long rows;                 // batch * pixels
    int batch, pixels, C, groups, Cg, act, param_dtype;
    float eps;
    double per_number;              // 1 / (pixels * Cg)
    NormPlan plan;
};

// All return a hipError_t as int.
int launch_norm_forward(const NormArgs &a, int dtype, void *stream);
int launch_norm_backward(const NormArgs &a, int dtype, void *stream);

long long mx4_work_items(long long rows, long long K);      // of either launch
int launch_mx4_quantize(const void *x, int dtype, long long rows, long long K, long long stride, void *codes, void *scales, void *stream);
int launch_mx4_dequantize(const void *codes, const void *scales, long long rows, long long K, void *y, int dtype, long long stride,
                          void *stream);

struct ProductArgs {
    const unsigned char *x_codes, *x_scales, *w_codes, *w_scales;
    const void *x;                  // numbers in place of codes (see product_takes_numbers), or null
    long long K, x_stride;
    int x_dtype;
    const void *bias, *residual;
    void *y;
    long long M, N, y_stride, r_stride;
    int ksteps;                     // padded K / 128
    int bias_dtype, act;
};
bool product_takes_numbers(long long M, long long N, long long K);
long long product_work_items(long long M, long long N, long long K, bool numbers);
int launch_mx4_product(const ProductArgs &a, int y_dtype, void *stream);

}  // namespace tdc
