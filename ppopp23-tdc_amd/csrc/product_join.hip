// What surrounds the products in 16 and 8 bits: how one is dealt out, the join of a sum's parts, and what the gradients need
// before their products: dz = dy act'(z), its sums over the rows, copies of rows that no request could take as they lie.
#include <algorithm>

#include "ops_device.hpp"

namespace tdc {

// ---- how a product is dealt out ----

TilePlan tile_plan(long long M, long long N, long long K, int in_dtype) {
    TilePlan p{};
    const long long step = in_dtype == TDC_MX8 ? 64 : 32;
    p.steps = (int)((K + step - 1) / step);
    auto tiles = [&](long long m, long long n) { return ((M + m - 1) / m) * ((N + n - 1) / n); };
    p.kernel = M <= 32 ? kTile32 : p.steps >= 64 && tiles(256, 256) >= 192 ? kTile256 : kTile128;
    const long long m = p.kernel == kTile256 ? 256 : p.kernel == kTile128 ? 128 : 32, n = p.kernel == kTile256 ? 256 : 128;
    p.tm = (int)((M + m - 1) / m);
    p.tn = (int)((N + n - 1) / n);
    const long long all = (long long)p.tm * p.tn;
    p.blocks = round_up(all, 8);
    p.splits = 1;
    p.split_steps = p.steps;
    if (all < 256 && p.steps >= 16) {
        const long long splits = std::min<long long>(p.steps / 8, (512 + all - 1) / all);
        p.split_steps = (int)round_up((p.steps + splits - 1) / splits, 8);
        p.splits = (p.steps + p.split_steps - 1) / p.split_steps;
    }
    p.part_stride = round_up(N, 4);
    p.part_bytes = p.splits > 1 ? p.splits * M * p.part_stride * 4 : 0;
    p.items = std::max(p.blocks * p.splits * 256, p.splits > 1 ? (M * (p.part_stride / 4) + 255) / 256 * 256 : 0);
    return p;
}

// ---- the join ----

// Four neighbouring outputs a thread: the parts in their order, then what a tile does with its sums.
template <int DT, int ACT>
__global__ void __launch_bounds__(256) tdc_product_join_kernel(const TileArgs a, int across) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x, m = id / across, n = (id - m * across) * 4;
    if (m >= a.M) return;
    using T = typename Num<DT>::type;
    const float *const from = a.part + m * a.part_stride + n;
    const long long part = a.M * a.part_stride;
    float4 v = *reinterpret_cast<const float4 *>(from);
    for (int s = 1; s < a.splits; ++s) {
        const float4 w = *reinterpret_cast<const float4 *>(from + s * part);
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    }
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
template <int DT>
static int launch_join_of(const TileArgs &a, hipStream_t s) {
    const int across = (int)(a.part_stride / 4);
    const unsigned blocks = (unsigned)((a.M * across + 255) / 256);
    if (a.act == TDC_ACT_RELU) tdc_product_join_kernel<DT, TDC_ACT_RELU><<<blocks, 256, 0, s>>>(a, across);
    else if (a.act == TDC_ACT_SILU) tdc_product_join_kernel<DT, TDC_ACT_SILU><<<blocks, 256, 0, s>>>(a, across);
    else tdc_product_join_kernel<DT, TDC_ACT_NONE><<<blocks, 256, 0, s>>>(a, across);
    return (int)hipGetLastError();
}
int launch_join(const TileArgs &a, int y_dtype, void *stream) {
    return y_dtype == TDC_F16 ? launch_join_of<TDC_F16>(a, (hipStream_t)stream) : launch_join_of<TDC_BF16>(a, (hipStream_t)stream);
}

// ---- dz ----

// A workgroup of 256 owns `across` vectors of eight columns and `chunk_rows` rows.  Sums over the rows: a thread's own rows in fp32 (those of
// a chunk: see act_grad_plan), then over threads and chunks in 64 bits, in a fixed order.  (Sums are of dz before its rounding.)
template <int DT, int ACT>
__global__ void __launch_bounds__(256) tdc_act_grad_kernel(const ActGradArgs a) {
    using P = Pack<DT, 8>;
    using T = typename Num<DT>::type;
    __shared__ float lds[256][9];
    const unsigned chunk = blockIdx.x / (unsigned)a.tiles, tile = blockIdx.x - chunk * a.tiles;
    const int down = 256 / a.across, c = threadIdx.x % a.across, r = threadIdx.x / a.across;
    const long long n = ((long long)tile * a.across + c) * 8, row0 = chunk * a.chunk_rows, rows = min(a.chunk_rows, a.M - row0);
    float sum[8] = {};
    auto load = [&](const void *base, long long at) {
        if (n + 8 <= a.N) return P::load(base, at);
        typename P::type v = {};
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (n + i < a.N) v[i] = reinterpret_cast<const T *>(base)[at + i];
        return v;
    };
    if (n < a.N) {
        for (long long i = r; i < rows; i += down) {
            const long long m = row0 + i;
            float v[8], z[8];
            P::up(load(a.dy, m * a.dy_stride + n), v);
            if constexpr (ACT != TDC_ACT_NONE) {
                P::up(load(a.kept, m * a.N + n), z);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= act_slope<ACT>(z[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += v[j];
            if (a.dz) P::store(a.dz, m * a.pitch + n, P::down(v));
        }
    }
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
        a.part[chunk * a.N + at] = (float)s;
    }
}
// The chunks' sums, 64 columns a workgroup, sixteen threads a column.
template <int OUT>
__global__ void __launch_bounds__(1024) tdc_column_sums_kernel(const float *part, void *out, long long N, int chunks) {
    __shared__ double lds[16][64];
    const long long n = (long long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int k = threadIdx.x >> 6;
    double s = 0;
    if (n < N)
        for (int i = k; i < chunks; i += 16) s += part[i * N + n];
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

void act_grad_plan(ActGradArgs &a) {
    a.pitch = round_up(a.N, 8);
    const long long vectors = (a.N + 7) / 8;
    a.across = 1;
    while (a.across < 32 && a.across < vectors) a.across *= 2;
    a.tiles = (int)((vectors + a.across - 1) / a.across);
    // Some 2048 workgroups, of four rows a thread at least and 256 at most (a sum in fp32 is no longer than that).
    const long long down = 256 / a.across, want = std::max(1ll, 2048ll / a.tiles);
    a.chunk_rows = round_up(std::clamp((a.M + want - 1) / want, 4 * down, 256 * down), down);
    a.chunks = (int)((a.M + a.chunk_rows - 1) / a.chunk_rows);
}
long long act_grad_items(const ActGradArgs &a) {
    return std::max((long long)a.chunks * a.tiles * 256, (a.N + 63) / 64 * 1024);
}
template <int DT>
static int launch_act_grad_of(const ActGradArgs &a, hipStream_t s) {
    const unsigned blocks = (unsigned)a.chunks * (unsigned)a.tiles;
    if (a.act == TDC_ACT_RELU) tdc_act_grad_kernel<DT, TDC_ACT_RELU><<<blocks, 256, 0, s>>>(a);
    else if (a.act == TDC_ACT_SILU) tdc_act_grad_kernel<DT, TDC_ACT_SILU><<<blocks, 256, 0, s>>>(a);
    else tdc_act_grad_kernel<DT, TDC_ACT_NONE><<<blocks, 256, 0, s>>>(a);
    if (hipError_t e = hipGetLastError()) return (int)e;
    return a.sums ? launch_column_sums(a.part, a.sums, a.N, a.chunks, a.sums_dtype, s) : 0;
}
int launch_act_grad(const ActGradArgs &a, int dtype, void *stream) {
    return dtype == TDC_F16 ? launch_act_grad_of<TDC_F16>(a, (hipStream_t)stream) : launch_act_grad_of<TDC_BF16>(a, (hipStream_t)stream);
}

}  // namespace tdc
