// What surrounds the products in 16 and 8 bits: how one is dealt out, the join of a sum's parts, and what the gradients need
// before their products: dz = dy act'(z), its sums over the rows, copies of rows that no request could take as they lie.
#include <algorithm>
#include <cmath>

#include "product_device.hpp"

namespace tdc {

// ---- how a product is dealt out ----

// Tiles, the time of a step and what a tile takes besides (us), as timed with one workgroup a compute unit (M x N x K in bf16, kernel
// by kernel; a compute unit that holds several gives each its share): 32 x 128 256 x 4096 x 4096 22.9, 64 x 128 512 x 4096 x 4096 28.1,
// 128 x 128 1024 x 4096 x 4096 40.3, 256 x 128 8192 x 1024 x 4096 71, 256 x 256 4096 x 4096 x 4096 115 (0.6 a step where few compute units
// work: their clock).  Larger tiles do more a step, smaller ones leave fewer compute units without work, and so do parts of the sum, which
// cost a launch and their bytes: 1024 x 1024 x 1024 7.7 in tiles of 32 rows, 11.7 of 128, 26.6 of 256; 128 x 512 x 25088 19.3 in 14 parts
// of 32 rows, 106 whole; 8192 x 8192 x 1024 140 in tiles of 256, 167 in 128 x 128 three a compute unit, 192 one by one; 25088 x 512 x 128 13.6
// three a compute unit, 15.6 in tiles of 256.  Small tiles wait for memory alone: one row by 16384 x 4096 weights that no cache holds 36.4
// with a workgroup a compute unit, 30.0 with two, 34.5 with four.
struct Timing {
    int m, n;
    double step, besides;
    int together;      // workgroups of a compute unit that hide each other's `besides`
    double alone;      // a step of a workgroup by itself
    int parts;         // a sum's parts fill the compute units so many times
};
static const Timing kTimings[] = {{256, 256, 0.82, 7.0, 1, 0.82, 1},   {256, 128, 0.51, 4.0, 1, 0.51, 1},  {128, 128, 0.28, 2.0, 1, 0.28, 1},
                                   {128, 128, 0.31, 1.5, 3, 0.31, 1}, {64, 128, 0.175, 0.8, 1, 0.24, 2}, {32, 128, 0.14, 0.8, 1, 0.22, 2}};

TilePlan tile_plan(long long M, long long N, long long K, int in_dtype, int layout) {
    const long long step = in_dtype == TDC_MX8 ? 64 : 32, steps = (K + step - 1) / step;
    TilePlan best{};
    double best_time = 0;
    for (int kernel = kTile256; kernel <= kTile32; ++kernel) {
        const Timing &t = kTimings[kernel];
        const long long tm = (M + t.m - 1) / t.m, tn = (N + t.n - 1) / t.n, all = tm * tn;
        // Parts as they fill the compute units, or half of that; eight steps each at least.
        const long long most = std::min(256 * t.parts / all, steps / 8);
        for (const long long want : {1ll, most / 2, most}) {
            if (want < 1) continue;
            const long long split_steps = want == 1 ? steps : round_up((steps + want - 1) / want, 8), splits = (steps + split_steps - 1) / split_steps;
            const double each = (double)(all * splits) / 256, rounds = t.together == 1 ? std::ceil(each) : std::max(each, 1.0);
            double time = 4.0 + std::max(rounds * t.step, t.alone) * (double)split_steps + rounds * t.besides / t.together + (t.together > 1 ? t.besides : 0.0);
            if (splits > 1) time += 5.5 + (double)splits * M * N * 8 / 4e6;
            if (best.steps && time >= best_time) continue;
            best_time = time;
            best.kernel = kernel;
            best.steps = (int)steps;
            best.tm = (int)tm;
            best.tn = (int)tn;
            best.splits = (int)splits;
            best.split_steps = (int)split_steps;
            best.blocks = round_up(all, 8);
        }
    }
    if (layout == kAlong && M <= 16 && few_time(N, K * (in_dtype == TDC_MX8 ? 1 : 2)) < best_time) {
        best = TilePlan{};
        best.kernel = kFewRows;
        best.splits = 1;
        best.items = few_items(N);
        return best;
    }
    best.part_stride = round_up(N, 4);
    best.part_bytes = best.splits > 1 ? best.splits * M * best.part_stride * 4 : 0;
    best.items = std::max(best.blocks * best.splits * 256, best.splits > 1 ? (M * (best.part_stride / 4) + 31) / 32 * 256 : 0);
    return best;
}

// ---- the join ----

// Four neighbouring outputs a thread: the parts in their order, then what a tile does with its sums.  GROUPS: so many threads share the
// outputs, a run of the parts each, and meet in LDS (98 parts of 128 x 512: 25 us with one, a chain of loads).
template <int DT, int ACT, int GROUPS>
__global__ void __launch_bounds__(256) tdc_product_join_kernel(const TileArgs a, int across) {
    constexpr int kThreads = 256 / GROUPS;
    __shared__ float4 lds[GROUPS > 1 ? 256 : 1];
    const int t = threadIdx.x % kThreads, g = threadIdx.x / kThreads;
    const long long id = (long long)blockIdx.x * kThreads + t, m = id / across, n = (id - m * across) * 4;
    using T = typename Num<DT>::type;
    const long long part = a.M * a.part_stride;
    const int each = (a.splits + GROUPS - 1) / GROUPS, end = min(a.splits, (g + 1) * each);
    float4 v = make_float4(0, 0, 0, 0);
    if (m < a.M) {
        const float *const from = a.part + m * a.part_stride + n;
#pragma unroll 8
        for (int s = g * each; s < end; ++s) {
            const float4 w = *reinterpret_cast<const float4 *>(from + s * part);
            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
    }
    if constexpr (GROUPS > 1) {
        lds[threadIdx.x] = v;
        __syncthreads();
        if (g) return;
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) {
            const float4 w = lds[k * kThreads + t];
            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
    }
    if (m >= a.M) return;
    const float sums[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + i >= a.N) return;
        float z = sums[i];
        if (a.bias) z += param<DT>(a.bias, n + i, a.bias_dtype);
        if (a.residual) z += Num<DT>::up(reinterpret_cast<const T *>(a.residual)[m * a.r_stride + n + i]);
        if (a.z) reinterpret_cast<T *>(a.z)[m * a.z_stride + n + i] = Num<DT>::down(z);
        reinterpret_cast<T *>(a.y)[m * a.y_stride + n + i] = Num<DT>::down(act_of<ACT>(z));
    }
}
template <int DT, int ACT>
static int launch_join_act(const TileArgs &a, hipStream_t s) {
    const int across = (int)(a.part_stride / 4);
    const long long threads = a.M * across;
    if (a.splits > 16) tdc_product_join_kernel<DT, ACT, 8><<<(unsigned)((threads + 31) / 32), 256, 0, s>>>(a, across);
    else tdc_product_join_kernel<DT, ACT, 1><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(a, across);
    return (int)hipGetLastError();
}
template <int DT>
static int launch_join_of(const TileArgs &a, hipStream_t s) {
    if (a.act == TDC_ACT_RELU) return launch_join_act<DT, TDC_ACT_RELU>(a, s);
    return a.act == TDC_ACT_SILU ? launch_join_act<DT, TDC_ACT_SILU>(a, s) : launch_join_act<DT, TDC_ACT_NONE>(a, s);
}
int launch_join(const TileArgs &a, int y_dtype, void *stream) {
    return y_dtype == TDC_F16 ? launch_join_of<TDC_F16>(a, (hipStream_t)stream) : launch_join_of<TDC_BF16>(a, (hipStream_t)stream);
}

// ---- dz ----

// A workgroup of 256 owns `across` vectors of eight columns and `chunk_rows` rows.  Sums over the rows: a thread's own rows in fp32 (those of
// a chunk: see act_grad_plan), then over threads and chunks in 64 bits, in a fixed order.  (Sums are of dz before its rounding.)
// dz itself is rounded: the matrix instructions that multiply it take 16 bits.
template <int DT, int ACT>
static __device__ __forceinline__ void act_grad(const ActGradArgs &a, unsigned block, float (&lds)[256][9]) {
    using P = Pack<DT, 8>;
    using T = typename Num<DT>::type;
    const unsigned chunk = block / (unsigned)a.tiles, tile = block - chunk * a.tiles;
    const int down = 256 / a.across, c = threadIdx.x % a.across, r = threadIdx.x / a.across;
    const long long n = ((long long)tile * a.across + c) * 8, row0 = chunk * a.chunk_rows, rows = min(a.chunk_rows, a.M - row0);
    float sum[8] = {};
    // Four rows are on their way at a time.
    auto rows_of = [&](auto load) {
        for (long long i = r; i < rows; i += 4 * down) {
            typename P::type dy[4], kept[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const long long m = row0 + min(i + k * down, rows - 1);      // (a repeated one is not used)
                dy[k] = load(a.dy, m * a.dy_stride + n);
                if constexpr (ACT != TDC_ACT_NONE) kept[k] = load(a.kept, m * a.N + n);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i + k * down >= rows) break;
                float v[8];
                P::up(dy[k], v);
                if constexpr (ACT != TDC_ACT_NONE) {
                    float z[8];
                    P::up(kept[k], z);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = act_back<ACT>(v[j], z[j]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += v[j];
                if (a.dz) P::store(a.dz, (row0 + i + k * down) * a.pitch + n, P::down(v));
            }
        }
    };
    if (n + 8 <= a.N) rows_of([](const void *base, long long at) { return P::load(base, at); });
    else if (n < a.N) rows_of([&](const void *base, long long at) { return load8<DT, false>(base, at, a.N - n); });
    if (!a.sums) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) lds[threadIdx.x][j] = sum[j];
    __syncthreads();
    // (column k of the workgroup, by the first threads)
    for (int k = threadIdx.x; k < a.across * 8; k += 256) {
        const long long at = (long long)tile * a.across * 8 + k;
        if (at >= a.N) continue;
        double s = 0;
        for (int i = 0; i < down; ++i) s += lds[i * a.across + k / 8][k % 8];
        if (a.chunks > 1) a.part[chunk * a.N + at] = (float)s;
        else if (a.sums_dtype == TDC_F32) reinterpret_cast<float *>(a.sums)[at] = (float)s;
        else reinterpret_cast<T *>(a.sums)[at] = Num<DT>::down((float)s);
    }
}
// Up to three such jobs side by side.
struct ActGradJobs {
    ActGradArgs job[3];
    unsigned end[3];      // workgroups up to a job's last
};
template <int DT>
__global__ void __launch_bounds__(256) tdc_act_grad_kernel(const ActGradJobs jobs) {
    __shared__ float lds[256][9];
    const int k = (blockIdx.x >= jobs.end[0]) + (blockIdx.x >= jobs.end[1]);
    const ActGradArgs &a = jobs.job[k];
    const unsigned block = blockIdx.x - (k ? jobs.end[k - 1] : 0);
    if (a.act == TDC_ACT_RELU) act_grad<DT, TDC_ACT_RELU>(a, block, lds);
    else if (a.act == TDC_ACT_SILU) act_grad<DT, TDC_ACT_SILU>(a, block, lds);
    else act_grad<DT, TDC_ACT_NONE>(a, block, lds);
}
// The chunks' sums, 64 columns a workgroup, sixteen threads a column.
template <int OUT>
__global__ void __launch_bounds__(1024) tdc_column_sums_kernel(const float *part, void *out, long long N, int chunks) {
    __shared__ double lds[16][64];
    const long long n = (long long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int k = threadIdx.x >> 6;
    double s = 0;
    if (n < N) {
#pragma unroll 8
        for (int i = k; i < chunks; i += 16) s += part[i * N + n];
    }
    lds[k][threadIdx.x & 63] = s;
    __syncthreads();
    if (k || n >= N) return;
    for (int i = 1; i < 16; ++i) s += lds[i][threadIdx.x];
    reinterpret_cast<typename Num<OUT>::type *>(out)[n] = Num<OUT>::down((float)s);
}
int launch_column_sums(const float *part, void *out, long long N, int chunks, int out_dtype, void *stream) {
    const unsigned blocks = (unsigned)((N + 63) / 64);
    const hipStream_t s = (hipStream_t)stream;
    if (out_dtype == TDC_F32) tdc_column_sums_kernel<TDC_F32><<<blocks, 1024, 0, s>>>(part, out, N, chunks);
    else if (out_dtype == TDC_F16) tdc_column_sums_kernel<TDC_F16><<<blocks, 1024, 0, s>>>(part, out, N, chunks);
    else tdc_column_sums_kernel<TDC_BF16><<<blocks, 1024, 0, s>>>(part, out, N, chunks);
    return (int)hipGetLastError();
}

// Zeros of every type are the same bits.  (A fill, not a sum of no chunks: its 1024 threads for 64 numbers could not be launched for
// 2^28 of them.)
static __global__ void __launch_bounds__(256) tdc_zeros_kernel(unsigned short *out, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) out[i] = 0;
}
int launch_zeros(void *out, long long N, int dtype, void *stream) {
    const long long n = dtype == TDC_F32 ? 2 * N : N;
    tdc_zeros_kernel<<<(unsigned)std::min((n + 255) / 256, 16384ll), 256, 0, (hipStream_t)stream>>>((unsigned short *)out, n);
    return (int)hipGetLastError();
}

void act_grad_plan(ActGradArgs &a) {
    a.pitch = round_up(a.N, 8);
    const long long vectors = (a.N + 7) / 8;
    a.across = 1;
    while (a.across < 32 && a.across < vectors) a.across *= 2;
    a.tiles = (int)((vectors + a.across - 1) / a.across);
    // Some 2048 workgroups, of four rows a thread at least and 256 at most (a sum in fp32 is no longer than that); sixteen rows a thread
    // make one chunk, whose sums need no second launch.
    const long long down = 256 / a.across, want = std::max(1ll, 2048ll / a.tiles);
    a.chunk_rows = round_up(std::clamp((a.M + want - 1) / want, 4 * down, 256 * down), down);
    if (a.M <= 16 * down) a.chunk_rows = 16 * down;
    a.chunks = (int)((a.M + a.chunk_rows - 1) / a.chunk_rows);
}
long long act_grad_items(const ActGradArgs &a) {
    return std::max((long long)a.chunks * a.tiles * 256, (a.N + 63) / 64 * 1024);
}
int launch_act_grad(const ActGradArgs *jobs, int n, int dtype, void *stream) {
    if (!n) return 0;
    ActGradJobs all{};
    unsigned blocks = 0;
    for (int k = 0; k < 3; ++k) {
        if (k < n) {
            all.job[k] = jobs[k];
            blocks += (unsigned)jobs[k].chunks * (unsigned)jobs[k].tiles;
        }
        all.end[k] = blocks;
    }
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == TDC_F16) tdc_act_grad_kernel<TDC_F16><<<blocks, 256, 0, s>>>(all);
    else tdc_act_grad_kernel<TDC_BF16><<<blocks, 256, 0, s>>>(all);
    if (hipError_t e = hipGetLastError()) return (int)e;
    for (int k = 0; k < n; ++k)
        if (jobs[k].sums && jobs[k].chunks > 1)
            if (int e = launch_column_sums(jobs[k].part, jobs[k].sums, jobs[k].N, jobs[k].chunks, jobs[k].sums_dtype, stream)) return e;
    return 0;
}

}  // namespace tdc
