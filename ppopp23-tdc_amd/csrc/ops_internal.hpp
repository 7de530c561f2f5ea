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

// Where a product's sums go: y = act(sums + bias + residual).
struct ProductOut {
    const void *bias, *residual;
    void *y, *z;                    // (z: what the activation is taken of, where a gradient will want it)
    long long M, N, y_stride, r_stride, z_stride;
    int bias_dtype, act;
};

struct ProductArgs : ProductOut {
    const unsigned char *x_codes, *x_scales, *w_codes, *w_scales;
    const void *x;                  // numbers in place of codes (see product_takes_numbers), or null
    long long K, x_stride;
    int x_dtype;
    int ksteps;                     // padded K / 128
};
// A product in 16 or 8 bits (see product_tile.hpp).  The sum runs over `steps` steps of 64 bytes.
struct TileArgs : ProductOut {
    const unsigned char *x, *w, *x_scales, *w_scales;
    long long x_stride, w_stride;   // bytes between the rows in memory: along the sum, or (an operand across it) its places
    long long x_outer, w_outer;     // rows in memory along the sum, else numbers of one row (a multiple of 8)
    long long x_limit, w_limit;     // numbers of the sum that are there
    int steps, split_steps, splits; // of the sum, of one part of it, parts
    int tiles_m, tiles_n;
    unsigned blocks;                // workgroups of a part
    float *part;                    // sums of the parts: [splits][M][part_stride]
    long long part_stride;
};
enum { kTile256, kTile256x128, kTile128Deep, kTile128, kTile64, kTile32, kFewRows };
// How a product is dealt out.
struct TilePlan {
    int kernel;                     // which tile
    int tm, tn, splits, split_steps, steps;
    long long blocks, part_stride;
    long long part_bytes;
    long long items;                // work items of its largest launch
};
enum { kAlong, kWAcross, kAcross };     // how x and w lie: both along the sum, w across it, both across it
TilePlan tile_plan(long long M, long long N, long long K, int in_dtype, int layout);
// `a` with everything but what the plan says; y_dtype is TDC_F16 or TDC_BF16.
int launch_product_bf16(TileArgs a, const TilePlan &p, int layout, void *stream);
int launch_product_f16(TileArgs a, const TilePlan &p, int layout, void *stream);
int launch_product_mx8(TileArgs a, const TilePlan &p, int y_dtype, void *stream);
int launch_join(const TileArgs &a, int y_dtype, void *stream);
double few_time(long long N, long long bytes);       // estimated, us
long long few_items(long long N);
int launch_product_few(const TileArgs &a, int in_dtype, int y_dtype, void *stream);      // both along the sum

// dz = dy act'(z) in rows of `pitch` numbers (zeros past the N-th), its sums over the rows besides; also a copy of rows (no activation).
struct ActGradArgs {
    const void *dy, *kept;          // kept: z, or for ReLU its result; rows of N
    void *dz;                       // or null
    void *sums;                     // [N], or null
    float *part;                    // [chunks][N]
    long long M, N, dy_stride, pitch;
    int act, chunks, sums_dtype;
    long long chunk_rows;
    int tiles;                      // workgroups across the columns
    int across;                     // vectors of eight columns of a workgroup (a power of two)
};
void act_grad_plan(ActGradArgs &a);      // pitch and the last five
long long act_grad_items(const ActGradArgs &a);
int launch_act_grad(const ActGradArgs *jobs, int n, int dtype, void *stream);      // up to three of them
int launch_column_sums(const float *part, void *out, long long N, int chunks, int out_dtype, void *stream);
int launch_zeros(void *out, long long N, int dtype, void *stream);      // N numbers

// Numbers in 8 bits.
inline long long mx8_pitch(long long K) { return round_up(K, 128); }
int launch_mx8_quantize(const void *x, int dtype, long long rows, long long K, long long stride, void *codes, void *scales, void *stream);
int launch_mx8_dequantize(const void *codes, const void *scales, long long rows, long long K, void *y, int dtype, long long stride,
                          void *stream);

// RMS norm.
struct RmsArgs {
    const void *x, *residual, *weight, *dy, *dh;
    void *y, *h;                    // h: x + residual, or null
    void *dx;
    float *rstd;
    unsigned char *codes, *scales;  // of y or of h
    float *part;                    // gradient: [workgroups][C]
    void *dweight;
    long long rows, x_stride, r_stride, dy_stride, dh_stride;
    int C, weight_dtype;
    float eps;
    int team, held;                 // lanes of a row, vectors of eight that each keeps
    int blocks;                     // workgroups
};
enum { kRmsPlain, kRmsOutputMx8, kRmsKeptMx8 };      // 8 bits: none, y, what the gradient needs of h
void rms_plan(RmsArgs &a, bool grad);                // the last three
long long rms_items(const RmsArgs &a, bool grad);
int launch_rms_forward(const RmsArgs &a, int dtype, int mode, void *stream);
int launch_rms_backward(const RmsArgs &a, int dtype, bool kept_mx8, void *stream);

bool product_takes_numbers(long long M, long long N, long long K);
long long product_work_items(long long M, long long N, long long K, bool numbers);
int launch_mx4_product(const ProductArgs &a, int y_dtype, void *stream);

}  // namespace tdc
