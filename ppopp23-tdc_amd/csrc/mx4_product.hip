// Product of two matrices in microscaled 4-bit floating point: y = act(x w^T + bias + residual).
//
// v_mfma_scale_f32_32x32x64: a lane holds one block of 32 numbers of its row (lane mod 32), the lower or the upper half of the 64
// (lane / 32), with that block's scale; products and sums are fp32.  The weights are the first operand, so that a lane ends up with
// neighbouring outputs of one row.  (16x16x128 does as much per instruction but takes the matrix unit 35 cycles where 32x32x64, with
// twice the work, takes 36: registers only, one wave a SIMD, 4.6 against 8.9 PFLOP/s, 6.4 on random numbers for their power.)
#include <algorithm>

#include "product_device.hpp"

namespace tdc {

// One matrix instruction; the low bytes of the scale words are this step's.
static __device__ __forceinline__ f16_t mfma4(i4_t a, i4_t b, f16_t c, int sa, int sb) {
    const i8_t wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

// ---- tiles ----
//
// A workgroup of four waves owns 64 MB rows of x and 64 NB of w, a wave a quarter of it: MB x NB blocks of 32 x 32.  A step is
// 128 numbers of each row.  Codes go straight from global memory into one of four LDS buffers, a step each, 1 KiB a request:
// asked for three steps ahead of their use, waited for one ahead; scales do so for four steps at a time.  A wave's step has a
// part for each two blocks of weights; each part starts the LDS reads of the next part's weights and of the next step's x, so
// that one wave to a SIMD keeps the matrix unit fed across its one barrier a step.  LDS holds the codes as they lie in
// memory: a block's read is 1 KiB in a row, which meets no bank twice.
//
// Measured, tiles of 256, 8192 x 8192 x 8192: 252 to 260 us on a layer's numbers.  While outputs took 10 to 15 us more, in random codes: 316 us, 3.5 PFLOP/s; 237 on zeros, 4.7, so that a quarter of it is the clock that
// the power leaves.  Without the outputs 294 and 202, without new codes besides 233 and 181 (registers only: 172 and 124).  On zeros, where
// power does not bind, half of the matrix unit's time is idle all the same; on random codes matrix instructions take half of the busy
// cycles and LDS 28 %: one wave a SIMD with a barrier every step keeps neither full.  The same workgroups going from tile to tile, the next one's codes on their way while this one's outputs
// leave, took as long.
//
template <int MB, int NB>
struct Tile {
    static constexpr int M = 64 * MB, N = 64 * NB;
    static constexpr int kBuffer = (M + N) * 64;              // bytes of a step's codes: x, then w
    static constexpr int kScales = (M + N) * 16;              // bytes of four steps' scales
    static constexpr int kLds = 4 * kBuffer + 2 * kScales + N * 4;     // (and the bias)
    static constexpr int kX = MB, kChunks = MB + NB;          // requests of a wave and step: of x, in all
    static constexpr int kScaleRequests = (M + N) / 256;      // of a wave and four steps
    static constexpr int kParts = NB / 2;
    // Where all steps are in LDS at once: as many buffers, and what the outputs pass through.
    static constexpr __host__ __device__ int short_buffers(int steps) { return steps > 2 ? steps : 2; }
    static constexpr __host__ __device__ int short_lds(int steps) { return short_buffers(steps) * kBuffer + kScales + N * 4; }
};

// Which tile a workgroup has, if any: neighbouring workgroups of a die take tiles of eight rows by as many columns as run at once, which
// share operands in its L2.
template <int MB, int NB>
static __device__ __forceinline__ bool tile_of(int tiles_m, int tiles_n, long long &m0, long long &n0) {
    const int total = tiles_m * tiles_n, per_die = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per_die + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_die || id >= total) return false;
    const int group = id / (8 * tiles_n), rest = id - group * 8 * tiles_n, high = min(8, tiles_m - group * 8);
    m0 = (long long)(group * 8 + rest % high) * Tile<MB, NB>::M;
    n0 = (long long)(rest / high) * Tile<MB, NB>::N;
    return true;
}
// Codes of a step for a tile: request i of a wave is half a block of 32 rows, of x for i below kX, of w from there on.  (Blocks past the
// last repeat it: their products go nowhere.)
template <int MB, int NB>
static __device__ __forceinline__ const unsigned char *codes_of(const ProductArgs &a, int i, long long step, long long m0, long long n0) {
    const bool of_x = i < Tile<MB, NB>::kX;
    return (of_x ? a.x_codes : a.w_codes) + (step * (((of_x ? a.M : a.N) + 31) >> 5) + ((of_x ? m0 : n0) >> 5)) * 2048;
}
template <int MB, int NB>
static __device__ __forceinline__ int chunk_of(const ProductArgs &a, int i, int wave, long long m0, long long n0) {
    using L = Tile<MB, NB>;
    const int c = (i < L::kX ? i : i - L::kX) * 4 + wave;
    return (int)min((long long)(c / 2), (i < L::kX ? ((a.M + 31) >> 5) - (m0 >> 5) : ((a.N + 31) >> 5) - (n0 >> 5)) - 1) * 2048 + c % 2 * 1024;
}
template <int DT, int MB, int NB>
__global__ void __launch_bounds__(256, MB * NB > 8 ? 1 : 2) tdc_mx4_product_tile_kernel(const ProductArgs a, int tiles_m, int tiles_n) {
    using L = Tile<MB, NB>;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 31, q = lane >> 5;
    const int wm = wave & 1, wn = wave >> 1;

    long long m0, n0;
    if (!tile_of<MB, NB>(tiles_m, tiles_n, m0, n0)) return;
    const float b = bias_of<DT>(a, n0 + t, t < L::N);

    // Codes: request i of a wave.
    int from[L::kChunks];
#pragma unroll
    for (int i = 0; i < L::kChunks; ++i) from[i] = chunk_of<MB, NB>(a, i, wave, m0, n0);
    auto fetch = [&](int i, int step) {
        bring(codes_of<MB, NB>(a, i, min(step, a.ksteps - 1), m0, n0), lane * 16, from[i], lds + (step & 3) * L::kBuffer + (i * 4 + wave) * 1024);
    };
    // Scales of four steps: rows of x, then of w, a row a thread.
    const int groups = (a.ksteps + 3) / 4, last_m = (int)min((long long)L::M, a.M - m0) - 1, last_n = (int)min((long long)L::N, a.N - n0) - 1;
    unsigned char *const lds_scales = lds + 4 * L::kBuffer;
    auto fetch_scales = [&](int g) {
        const long long at = min(g, groups - 1);
        unsigned char *const to = lds_scales + (g & 1) * L::kScales + wave * 1024;
#pragma unroll
        for (int i = 0; i < L::kScaleRequests; ++i) {
            const bool of_x = i * 256 + wave * 64 < L::M;
            const unsigned char *const base = of_x ? a.x_scales + (at * a.M + m0) * 16 : a.w_scales + (at * a.N + n0) * 16;
            const int row = i * 256 + t, in = of_x ? min(row, last_m) : min(row - L::M, last_n);
            bring(base, in * 16, 0, to + i * 4096);
        }
    };

    // Row r of a block; its places q and 2 + q for the two halves of a step.
    const int x_row = wm * 32 * MB + r, w_row = wn * 32 * NB + weight_row(r);
    const int x_at = wm * MB * 2048 + q * 512 + r * 16, w_at = L::M * 64 + wn * NB * 2048 + q * 512 + weight_row(r) * 16;
    auto x_frag = [&](int i, int half, int buffer) { return *reinterpret_cast<const i4_t *>(lds + buffer + x_at + i * 2048 + half * 1024); };
    auto w_frag = [&](int j, int half, int buffer) { return *reinterpret_cast<const i4_t *>(lds + buffer + w_at + j * 2048 + half * 1024); };
    auto read_scales = [&](int g, int (&sx)[MB][2], int (&sw)[NB][2]) {
        const unsigned char *const at = lds_scales + (g & 1) * L::kScales + q * 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MB; ++i) sx[i][h] = *reinterpret_cast<const int *>(at + (x_row + i * 32) * 16 + h * 8);
#pragma unroll
            for (int j = 0; j < NB; ++j) sw[j][h] = *reinterpret_cast<const int *>(at + (L::M + w_row + j * 32) * 16 + h * 8);
        }
    };
    f16_t acc[NB][MB];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.0f;

    // (an odd number of steps is rounded up: the scales past the last are zero, and so is what that step adds)
    const int steps = (a.ksteps + 1) / 2 * 2;
    float *const bias = reinterpret_cast<float *>(lds_scales + 2 * L::kScales);
    fetch_scales(0);
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int i = 0; i < L::kChunks; ++i) fetch(i, s);
    if (t < L::N) bias[t] = b;
    meet<L::kChunks>();
    i4_t x[2][MB][2], w[2][2][2];
    int sx[MB][2], sw[NB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < MB; ++i) x[0][i][h] = x_frag(i, h, 0);
        w[0][0][h] = w_frag(0, h, 0);
        w[0][1][h] = w_frag(1, h, 0);
    }
    read_scales(0, sx, sw);

    // Step `step`, of which S = step mod 2.
    auto run = [&](auto parity, int step) {
        constexpr int S = decltype(parity)::value, P = L::kParts;
        const int now = (step & 3) * L::kBuffer, next = (step + 1 & 3) * L::kBuffer;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int set = P == 1 ? S : p & 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int j = 0; j < 2; ++j) w[set ^ 1][j][h] = p + 1 < P ? w_frag(2 * p + 2 + j, h, now) : w_frag(j, h, next);
#pragma unroll
                for (int i = p * MB / P; i < (p + 1) * MB / P; ++i) x[S ^ 1][i][h] = x_frag(i, h, next);
                constexpr int kSlots = 2 * P;
                const int slot = 2 * p + h;
#pragma unroll
                for (int i = slot * L::kChunks / kSlots; i < (slot + 1) * L::kChunks / kSlots; ++i) fetch(i, step + 3);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < MB; ++i)
                        acc[2 * p + j][i] = mfma4(w[set][j][h], x[S][i][h], acc[2 * p + j][i], sw[2 * p + j][h], sx[i][h]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MB; ++i) sx[i][h] = (int)((unsigned)sx[i][h] >> 8);
#pragma unroll
            for (int j = 0; j < NB; ++j) sw[j][h] = (int)((unsigned)sw[j][h] >> 8);
        }
        meet<L::kChunks>();      // (the codes of the step after the next have to be there: all requests but this step's)
    };
    // (no branch stands between a step's requests and its matrix instructions, or the compiler moves these behind the barrier; the
    // last three steps bring codes that no one needs)
    int step = 0;
    for (int g = 0; g < groups; ++g) {
        // Four steps: their scales are in registers, those of the next four are asked for here and read when these are done.
        fetch_scales(g + 1);
        for (const int end = min(step + 4, steps); step < end; step += 2) {
            run(std::integral_constant<int, 0>{}, step);
            run(std::integral_constant<int, 1>{}, step + 1);
        }
        read_scales(g + 1, sx, sw);
    }
    meet<0>();       // (nothing may still be on its way into LDS when the workgroup ends)

    finish_tile<DT, MB, NB>(a, acc, m0 + wm * 32 * MB, n0 + wn * 32 * NB, bias + wn * 32 * NB, lds + wave * NB * 4096);
}

// ---- short sums ----
//
// Bound by the outputs' bytes, and by the way there.  Tiles of 128 x 128 as above, but all codes of up to 512 numbers of a row are in
// LDS at once, asked for together and waited for once; up to 256 numbers leave room for three workgroups on a compute unit, of which
// one can store while others load.  (Making x into 4 bits here as well, once for every tile across, took longer than a launch of its
// own that leaves codes: 25088 rows of 128 by 512 18.5 us against 17.6, 4096 of 512 by 4096 41 against 22.)
//
// Measured: 25088 rows of 128 by 512, outputs in bf16, with a residual: 12.9 us (51 MB and 5 TB/s of it, two and a half us the launch).  Without one,
// while outputs took longer: 12.6;
// 5.2 of the 12.6 are the stores, 3 the way of the sums through LDS.
template <int DT>
__global__ void __launch_bounds__(256, (DT == TDC_F32 ? 2 : 3)) tdc_mx4_product_short_kernel(const ProductArgs a, int tiles_m, int tiles_n) {
    using L = Tile<2, 2>;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 31, q = lane >> 5;
    const int wm = wave & 1, wn = wave >> 1;
    long long m0, n0;
    if (!tile_of<2, 2>(tiles_m, tiles_n, m0, n0)) return;
    const float b = bias_of<DT>(a, n0 + t, t < L::N);
    unsigned char *const lds_scales = lds + L::short_buffers(a.ksteps) * L::kBuffer;
    float *const bias = reinterpret_cast<float *>(lds_scales + L::kScales);
#pragma unroll
    for (int i = 0; i < L::kChunks; ++i) {
        const int from = chunk_of<2, 2>(a, i, wave, m0, n0);
        for (int step = 0; step < a.ksteps; ++step)
            bring(codes_of<2, 2>(a, i, step, m0, n0), lane * 16, from, lds + step * L::kBuffer + (i * 4 + wave) * 1024);
    }
    // Scales: rows of x, then of w, a row a thread.
    if (wave < 2) bring(a.x_scales + m0 * 16, (int)min((long long)t, a.M - m0 - 1) * 16, 0, lds_scales + wave * 1024);
    else bring(a.w_scales + n0 * 16, (int)min((long long)t - L::M, a.N - n0 - 1) * 16, 0, lds_scales + wave * 1024);
    if (t < L::N) bias[t] = b;
    meet<0>();
    // Row r of a block; its places q and 2 + q for the two halves of a step.
    const int w_in = weight_row(r), x_at = wm * 4096 + q * 512 + r * 16, w_at = L::M * 64 + wn * 4096 + q * 512 + w_in * 16;
    int sx[2][2], sw[2][2];
    f16_t acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sx[i][h] = *reinterpret_cast<const int *>(lds_scales + (wm * 64 + i * 32 + r) * 16 + q * 4 + h * 8);
            sw[i][h] = *reinterpret_cast<const int *>(lds_scales + (L::M + wn * 64 + i * 32 + w_in) * 16 + q * 4 + h * 8);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][h][e] = 0.0f;
        }
    for (int step = 0; step < a.ksteps; ++step) {
        const unsigned char *const at = lds + step * L::kBuffer;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i4_t x[2], w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[i] = *reinterpret_cast<const i4_t *>(at + x_at + i * 2048 + h * 1024);
                w[i] = *reinterpret_cast<const i4_t *>(at + w_at + i * 2048 + h * 1024);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    acc[j][i] = mfma4(w[j], x[i], acc[j][i], (int)((unsigned)sw[j][h] >> 8 * step), (int)((unsigned)sx[i][h] >> 8 * step));
        }
    }
    meet<0>();
    finish_tile<DT, 2, 2>(a, acc, m0 + wm * 64, n0 + wn * 64, bias + wn * 64, lds + wave * 8192);
}

// ---- few outputs ----
//
// Bound by the weights' bytes, or by latency.  A workgroup owns 32 rows of w and 32 of x; its waves share K, 512 numbers at a
// time, with their codes straight in registers: a block of 32 rows by 64 numbers is one request of 1 KiB.  The waves' sums meet
// in LDS, in the order of the waves.  XS: x in 4 bits (TDC_MX4), or numbers of that type, which a workgroup makes into 4 bits in LDS
// by itself: for few rows that costs less than a launch.
//
// Measured: one row of 4096 by 16384 weights, x in bf16: 8.0 to 9.8 us (36 MB, 3.7 to 4.5 TB/s); 33 rows of 2000 by 1001, x in fp32: 11.4, 64
// workgroups of which every one across makes the same 32 rows into 4 bits, one after the other with weights and sums; 196 rows of 1024 by 256 in 4 bits: 5.6.
// `rows` rows of x from row m0 on into codes in LDS, eight numbers a thread, four such runs on their way: block b of row m at
// (b rows + m) 16, its scale byte behind all codes, words of four steps.
template <int XS>
static __device__ __forceinline__ void take_numbers(const ProductArgs &a, long long m0, int rows, unsigned char *codes, unsigned char *scales) {
    using P = Pack<XS, 8>;
    const int octets = a.ksteps * 16;
    for (int at = threadIdx.x; at < rows * octets; at += 4 * blockDim.x) {
        typename P::type p[4];
        int row[4], octet[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = min(at + k * (int)blockDim.x, rows * octets - 1);      // (a repeated one is not stored)
            row[k] = small_quotient(i, octets);
            octet[k] = i - row[k] * octets;
            const long long from = (m0 + row[k]) * a.x_stride;
            if (octet[k] * 8 + 8 <= a.K) p[k] = P::load(a.x, from + octet[k] * 8);
            else {
                p[k] = typename P::type{};
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (octet[k] * 8 + j < a.K) p[k][j] = reinterpret_cast<const typename Num<XS>::type *>(a.x)[from + octet[k] * 8 + j];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[8], top = 0.0f;
            P::up(p[k], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = larger(top, v[j]);
            const int byte = mx4_scale_byte(quad_larger(top)), b = octet[k] >> 2;
            if (at + k * (int)blockDim.x >= rows * octets) continue;
            *reinterpret_cast<unsigned *>(codes + (b * rows + row[k]) * 16 + (octet[k] & 3) * 4) = mx4_codes(v, mx4_divisor(byte));
            if ((octet[k] & 3) == 0) scales[(b >> 4) * rows * 16 + row[k] * 16 + (b & 3) * 4 + (b >> 2 & 3)] = (unsigned char)byte;
        }
    }
}

template <int DT, int XS>
__global__ void __launch_bounds__(1024) tdc_mx4_product_few_kernel(const ProductArgs a, int blocks_m) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), waves = blockDim.x >> 6, r = lane & 31, q = lane >> 5;
    const long long n0 = (long long)(blockIdx.x / (unsigned)blocks_m) * 32, m0 = (long long)(blockIdx.x % (unsigned)blocks_m) * 32;
    const long long x_blocks = (a.M + 31) >> 5, w_blocks = (a.N + 31) >> 5;
    const int groups = (a.ksteps + 3) / 4, M = (int)min(a.M - m0, 32ll);      // (rows of this workgroup)
    const long long w_row = min(n0 + r, a.N - 1), x_row = min(m0 + r, a.M - 1);

    i4_t w[4][2], x[4][2];
    int sw[2], sx[2];
    // (steps past the last repeat it, their scales are zero)
    auto ask = [&](int g) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const long long k = min(g * 4 + s, a.ksteps - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[s][h] = *reinterpret_cast<const i4_t *>(a.w_codes + (k * w_blocks + (n0 >> 5)) * 2048 + h * 1024 + lane * 16);
                if constexpr (XS == TDC_MX4)
                    x[s][h] = *reinterpret_cast<const i4_t *>(a.x_codes + (k * x_blocks + (m0 >> 5)) * 2048 + h * 1024 + lane * 16);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sw[h] = *reinterpret_cast<const int *>(a.w_scales + ((long long)g * a.N + w_row) * 16 + q * 4 + h * 8);
            if constexpr (XS == TDC_MX4) sx[h] = *reinterpret_cast<const int *>(a.x_scales + ((long long)g * a.M + x_row) * 16 + q * 4 + h * 8);
        }
    };
    unsigned char *const x_lds = lds, *const sx_lds = lds + a.ksteps * 64 * M;
    if (wave < groups) ask(wave);
    if constexpr (XS != TDC_MX4) {
        // (the scale bytes past a row's last block)
        for (int i = t; i < M * 16; i += blockDim.x) sx_lds[(groups - 1) * M * 16 + i] = 0;
        __syncthreads();
        take_numbers<XS>(a, m0, M, x_lds, sx_lds);
        __syncthreads();
    }
    f16_t acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
    for (int g = wave; g < groups; g += waves) {
        if constexpr (XS != TDC_MX4) {
            const int m = min(r, M - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int k = min(g * 4 + s, a.ksteps - 1);
                    x[s][h] = *reinterpret_cast<const i4_t *>(x_lds + ((k * 4 + 2 * h + q) * M + m) * 16);
                }
                sx[h] = *reinterpret_cast<const int *>(sx_lds + (g * M + m) * 16 + q * 4 + h * 8);
            }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = mfma4(w[s][h], x[s][h], acc, (int)((unsigned)sw[h] >> 8 * s), (int)((unsigned)sx[h] >> 8 * s));
        if (g + waves < groups) ask(g + waves);
    }
    // Sums of the waves: output e of a lane, row 8 (e / 4) + 4 q + e mod 4 of w and r of x.
    if constexpr (XS != TDC_MX4) __syncthreads();
    float *const part = reinterpret_cast<float *>(lds);
    using T = typename Num<DT>::type;
    if (wave < groups) {
#pragma unroll
        for (int e = 0; e < 16; ++e) part[(wave * 16 + e) * 64 + lane] = acc[e];
    }
    __syncthreads();
    const int summed = min(waves, groups);      // (the others had none)
    for (int o = t; o < 32 * M; o += blockDim.x) {
        const int n = o & 31, m = o >> 5, at = ((n >> 3) * 4 + (n & 3)) * 64 + (n >> 2 & 1) * 32 + m;
        if (n0 + n >= a.N) continue;
        float v = 0.0f;
        for (int k = 0; k < summed; ++k) v += part[k * 1024 + at];
        if (a.bias) v += param<DT>(a.bias, n0 + n, a.bias_dtype);
        if (a.residual) v += Num<DT>::up(reinterpret_cast<const T *>(a.residual)[(m0 + m) * a.r_stride + n0 + n]);
        v = a.act == TDC_ACT_RELU ? act_of<TDC_ACT_RELU>(v) : a.act == TDC_ACT_SILU ? act_of<TDC_ACT_SILU>(v) : v;
        reinterpret_cast<T *>(a.y)[(m0 + m) * a.y_stride + n0 + n] = Num<DT>::down(v);
    }
}

template <int DT, int MB, int NB>
static int launch_tile(const ProductArgs &a, hipStream_t s) {
    using L = Tile<MB, NB>;
    static unsigned long long done = 0;
    auto *const fn = &tdc_mx4_product_tile_kernel<DT, MB, NB>;
    if (int e = allow_lds((const void *)fn, L::kLds, done)) return e;
    const int tm = (int)((a.M + L::M - 1) / L::M), tn = (int)((a.N + L::N - 1) / L::N);
    const unsigned grid = (unsigned)(((long long)tm * tn + 7) / 8 * 8);
    fn<<<grid, 256, L::kLds, s>>>(a, tm, tn);
    return (int)hipGetLastError();
}
template <int DT>
static int launch_short(const ProductArgs &a, hipStream_t s) {
    using L = Tile<2, 2>;
    static unsigned long long done = 0;
    auto *const fn = &tdc_mx4_product_short_kernel<DT>;
    if (int e = allow_lds((const void *)fn, L::short_lds(4), done)) return e;
    const int tm = (int)((a.M + L::M - 1) / L::M), tn = (int)((a.N + L::N - 1) / L::N);
    const unsigned grid = (unsigned)(((long long)tm * tn + 7) / 8 * 8);
    fn<<<grid, 256, L::short_lds(a.ksteps), s>>>(a, tm, tn);
    return (int)hipGetLastError();
}
// A wave for every 512 numbers of K, four to sixteen of them; sixteen also to make many numbers into 4 bits.
static int few_waves(long long M, int ksteps, bool numbers) {
    const int groups = (ksteps + 3) / 4;
    return groups > 8 || (numbers && std::min(M, 32ll) * ksteps > 64) ? 16 : groups > 4 ? 8 : 4;
}
template <int DT, int XS>
static int launch_few(const ProductArgs &a, hipStream_t s) {
    const int groups = (a.ksteps + 3) / 4, rows = (int)std::min(a.M, 32ll), waves = few_waves(a.M, a.ksteps, XS != TDC_MX4);
    const int x_bytes = XS == TDC_MX4 ? 0 : rows * (a.ksteps * 64 + groups * 16), lds = std::max(std::min(waves, groups) * 4096, x_bytes);
    const unsigned bm = (unsigned)((a.M + 31) / 32), bn = (unsigned)((a.N + 31) / 32);
    tdc_mx4_product_few_kernel<DT, XS><<<bm * bn, waves * 64, lds, s>>>(a, (int)bm);
    return (int)hipGetLastError();
}

// Timed in turn over M 16 .. 100352, N 64 .. 8192, K 64 .. 8192 (us, M x N x K), and carried on beyond: few rows of x by very many weights
// (N from 49152 on with K from 4096) run tiles whose rows are mostly empty, untimed:
//   32 x 32 outputs a workgroup while there are 512 of them, or 1024 of short sums: 1024 x 512 x 2048 7.5 against 9.6 in tiles of 128,
//   1024 x 1024 x 512 5.3 against 6.6, but 1024 x 1024 x 1024 7.6 against 7.6 and 2048 x 1024 x 512 9.0 against 6.9;
//   all steps at once up to 512 numbers: 25088 x 512 x 128 12.6 against 15.0 step by step, 100352 x 256 x 64 17.9 against 24.0, 4096 x 4096
//   x 512 16.9 against 17.6 (more than 512 would leave a compute unit one workgroup);
//   tiles of 256 for long sums that fill the compute units: 4096 x 8192 x 8192 164 against 184, 25088 x 512 x 8192 69 against 78, but
//   8192 x 8192 x 2048 114 against 112 (a tile's first loads and its stores run alone) and 1024 x 8192 x 8192 64 against 45.
static long long tiles(long long M, long long N, long long edge) { return ((M + edge - 1) / edge) * ((N + edge - 1) / edge); }
enum { kFew, kShort, kTiles128, kTiles256 };
static int pick(long long M, long long N, int ksteps) {
    if (tiles(M, N, 32) <= (ksteps <= 4 ? 1024 : 512)) return kFew;
    if (ksteps <= 4) return kShort;
    return ksteps >= 32 && tiles(M, N, 256) >= 192 ? kTiles256 : kTiles128;
}
template <int DT>
static int launch_product(const ProductArgs &a, hipStream_t s) {
    if (a.x) {
        if (a.x_dtype == TDC_F32) return launch_few<DT, TDC_F32>(a, s);
        return a.x_dtype == TDC_F16 ? launch_few<DT, TDC_F16>(a, s) : launch_few<DT, TDC_BF16>(a, s);
    }
    switch (pick(a.M, a.N, a.ksteps)) {
        case kFew: return launch_few<DT, TDC_MX4>(a, s);
        case kShort: return launch_short<DT>(a, s);
        case kTiles256: return launch_tile<DT, 4, 4>(a, s);
        default: return launch_tile<DT, 2, 2>(a, s);
    }
}

// x as it comes, without a launch of its own: 64 Ki numbers a workgroup (34 KiB of LDS), as each repeats the work for its rows; eight
// rows of any number of weights, more where no compute unit does it twice.
bool product_takes_numbers(long long M, long long N, long long K) {
    const long long rows = std::min(M, 32ll), workgroups = ((M + 31) / 32) * ((N + 31) / 32);
    return rows * mx4_padded(K) <= 65536 && (M <= 8 || workgroups <= 256);
}

long long product_work_items(long long M, long long N, long long K, bool numbers) {
    const int ksteps = (int)(mx4_padded(K) / 128);
    const bool taken = numbers && product_takes_numbers(M, N, K);
    const int kernel = taken ? kFew : pick(M, N, ksteps);
    if (kernel == kFew) return tiles(M, N, 32) * few_waves(M, ksteps, taken) * 64;
    return (tiles(M, N, kernel == kTiles256 ? 256 : 128) + 7) / 8 * 8 * 256;
}

int launch_mx4_product(const ProductArgs &a, int y_dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (y_dtype == TDC_F32) return launch_product<TDC_F32>(a, s);
    if (y_dtype == TDC_F16) return launch_product<TDC_F16>(a, s);
    return launch_product<TDC_BF16>(a, s);
}

}  // namespace tdc
