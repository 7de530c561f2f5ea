// Product of two matrices in microscaled 4-bit floating point: y = act(x w^T + bias + residual).
//
// v_mfma_scale_f32_32x32x64: a lane holds one block of 32 numbers of its row (lane mod 32), the lower or the upper half of the 64
// (lane / 32), with that block's scale; products and sums are fp32.  The weights are the first operand, so that a lane ends up with
// neighbouring outputs of one row.  (16x16x128 does as much per instruction but takes the matrix unit 35 cycles where 32x32x64, with
// twice the work, takes 36: registers only, one wave a SIMD, 4.6 against 8.9 PFLOP/s, 6.4 on random numbers for their power.)
#include <type_traits>

#include "ops_device.hpp"

namespace tdc {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i8_t __attribute__((ext_vector_type(8)));
typedef float f16_t __attribute__((ext_vector_type(16)));

// One matrix instruction; the low bytes of the scale words are this step's.
static __device__ __forceinline__ f16_t mfma4(i4_t a, i4_t b, f16_t c, int sa, int sb) {
    const i8_t wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

// Eight neighbouring outputs of a row (those before N): sums with the bias in `v`; residual, activation, store.
template <int DT, int ACT>
static __device__ __forceinline__ void finish8(const ProductArgs &a, long long m, long long n, float (&v)[8]) {
    using T = typename Num<DT>::type;
    typedef T vec_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    T *const to = reinterpret_cast<T *>(a.y) + m * a.y_stride + n;
    const int count = (int)min(8ll, a.N - n);
    if (a.residual) {
        const T *const add = reinterpret_cast<const T *>(a.residual) + m * a.r_stride + n;
        vec_t r = {};
        if (count == 8) r = *reinterpret_cast<const vec_t *>(add);
        else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < count) r[i] = add[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += Num<DT>::up(r[i]);
    }
    vec_t out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = Num<DT>::down(act_of<ACT>(v[i]));
    if (count == 8) *reinterpret_cast<vec_t *>(to) = out;
    else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < count) to[i] = out[i];
    }
}
template <int DT>
static __device__ __forceinline__ void bias8(const ProductArgs &a, long long n, float (&bias)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bias[i] = a.bias && n + i < a.N ? param<DT>(a.bias, n + i, a.bias_dtype) : 0.0f;
}

// ---- tiles ----
//
// A workgroup of four waves owns 64 MB rows of x and 64 NB of w, a wave a quarter of it: MB x NB blocks of 32 x 32.  A step is
// 128 numbers of each row.  Codes go from global memory through registers into LDS buffers, a step each: asked for four steps
// ahead of their use, stored two ahead; scales do so for four steps at a time.  A wave's step has a part for each two blocks of
// weights; each part starts the LDS reads of the next part's weights and of the next step's x, stores what global memory has
// brought, and asks for more, so that one wave to a SIMD keeps the matrix unit fed across its one barrier a step.
//
// LDS holds 32 rows by their places: place p of row i, 16 bytes, at 512 p + 16 (i ^ 4 p).  Reads take a place of 32 rows, 512 bytes in
// a row; stores take four places of sixteen rows, and the twist spreads them over the banks.
// The row of w that is row r of a block: bits 2 and 3 change places, which makes a lane's outputs 8 i .. 8 i + 7 neighbours.
static __device__ __forceinline__ int weight_row(int r) { return (r & 19) | (r & 4) << 1 | (r & 8) >> 1; }

template <int MB, int NB>
struct Tile {
    static constexpr int M = 64 * MB, N = 64 * NB;
    static constexpr int kBuffer = (M + N) * 64;              // bytes of a step's codes: x, then w
    static constexpr int kScales = (M + N) * 16;              // bytes of four steps' scales
    static constexpr int kLds = 4 * kBuffer + 2 * kScales;
    static constexpr int kX = MB, kChunks = MB + NB;          // requests of 16 bytes a thread and step: of x, in all
    static constexpr int kParts = NB / 2;
};

template <int DT, int MB, int NB>
__global__ void __launch_bounds__(256, MB * NB > 8 ? 1 : 2) tdc_mx4_product_tile_kernel(const ProductArgs a, int tiles_m, int tiles_n) {
    using L = Tile<MB, NB>;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 31, q = lane >> 5;
    const int wm = wave & 1, wn = wave >> 1;

    // Neighbouring workgroups of a die take tiles of eight rows by as many columns as run at once: they share operands in its L2.
    const int total = tiles_m * tiles_n, per_die = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per_die + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per_die || id >= total) return;
    const int group = id / (8 * tiles_n), rest = id - group * 8 * tiles_n, high = min(8, tiles_m - group * 8);
    const long long m0 = (long long)(group * 8 + rest % high) * L::M, n0 = (long long)(rest / high) * L::N;

    const int last = a.ksteps - 1, last_m = (int)min((long long)L::M, a.M - m0) - 1, last_n = (int)min((long long)L::N, a.N - n0) - 1;
    const unsigned char *const xc = a.x_codes + m0 * 64, *const wc = a.w_codes + n0 * 64;
    const int place = t & 3;
    unsigned from[L::kChunks];          // (rows past the last repeat it: their products go nowhere)
#pragma unroll
    for (int i = 0; i < L::kChunks; ++i) {
        const int row = (i < L::kX ? i : i - L::kX) * 64 + (t >> 2);
        from[i] = min(row, i < L::kX ? last_m : last_n) * 64 + place * 16;
    }
    i4_t chunk[2][L::kChunks];
    auto fetch = [&](int set, int i, int step) {
        const long long k = min(step, last);
        chunk[set][i] = *reinterpret_cast<const i4_t *>((i < L::kX ? xc + k * a.M * 64 : wc + k * a.N * 64) + from[i]);
    };
    const int to = (t >> 7) * 2048 + place * 512 + ((t >> 2 & 31) ^ 4 * place) * 16;
    auto park = [&](int set, int i, int buffer) { *reinterpret_cast<i4_t *>(lds + buffer + i * 4096 + to) = chunk[set][i]; };

    // Scales of four steps: thread t brings row t of x and row t of w.
    i4_t sx_in, sw_in;
    const int groups = (a.ksteps + 3) / 4;
    auto fetch_scales = [&](int g) {
        const long long at = min(g, groups - 1);
        sx_in = *reinterpret_cast<const i4_t *>(a.x_scales + (at * a.M + m0 + min(t, last_m)) * 16);
        sw_in = *reinterpret_cast<const i4_t *>(a.w_scales + (at * a.N + n0 + min(t, last_n)) * 16);
    };
    unsigned char *const lds_scales = lds + 4 * L::kBuffer;
    auto park_scales = [&](int g) {
        unsigned char *const to = lds_scales + (g & 1) * L::kScales + t * 16;
        if (L::M == 256 || t < L::M) *reinterpret_cast<i4_t *>(to) = sx_in;
        if (L::N == 256 || t < L::N) *reinterpret_cast<i4_t *>(to + L::M * 16) = sw_in;
    };

    // Places q and 2 + q (`half`) of row r of a block.
    const int x_row = wm * 32 * MB + r, w_row = wn * 32 * NB + weight_row(r);
    const int x_at = wm * MB * 2048 + q * 512, w_at = L::M * 64 + wn * NB * 2048 + q * 512;
    int x_in[2], w_in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        x_in[h] = x_at + h * 1024 + (r ^ 4 * (2 * h + q)) * 16;
        w_in[h] = w_at + h * 1024 + (weight_row(r) ^ 4 * (2 * h + q)) * 16;
    }
    auto x_frag = [&](int i, int half, int buffer) { return *reinterpret_cast<const i4_t *>(lds + buffer + x_in[half] + i * 2048); };
    auto w_frag = [&](int j, int half, int buffer) { return *reinterpret_cast<const i4_t *>(lds + buffer + w_in[half] + j * 2048); };
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
    auto meet = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    f16_t acc[NB][MB];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.0f;

    // (each set's requests in order: the waits of the loop count them)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < L::kChunks; ++i) fetch(s, i, s);
        __builtin_amdgcn_sched_barrier(0);
    }
    fetch_scales(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < L::kChunks; ++i) {
            park(s, i, s * L::kBuffer);
            fetch(s, i, 2 + s);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    park_scales(0);
    fetch_scales(1);
    meet();
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
        const int now = (step & 3) * L::kBuffer, next = (step + 1 & 3) * L::kBuffer, fill = (step + 2 & 3) * L::kBuffer;
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
                for (int i = slot * L::kChunks / kSlots; i < (slot + 1) * L::kChunks / kSlots; ++i) {
                    park(S, i, fill);
                    fetch(S, i, step + 4);
                }
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
        meet();
    };
    // (an odd number of steps is rounded up: the scales past the last are zero, and so is what that step adds)
    int step = 0;
    const int steps = (a.ksteps + 1) / 2 * 2;
    for (int g = 0; g < groups; ++g) {
        // Four steps: their scales are in registers; those of the next four are stored here and read when these are done.
        park_scales(g + 1);
        fetch_scales(g + 2);
        for (const int end = min(step + 4, steps); step < end; step += 2) {
            run(std::integral_constant<int, 0>{}, step);
            run(std::integral_constant<int, 1>{}, step + 1);
        }
        read_scales(g + 1, sx, sw);
    }

    // A lane's outputs of a block: row r of x, and of w 16 u + 8 q .. 16 u + 8 q + 7, u = 0, 1.
    auto finish = [&](auto act) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const long long n = n0 + wn * 32 * NB + j * 32 + u * 16 + q * 8;
                if (n >= a.N) continue;
                float bias[8];
                bias8<DT>(a, n, bias);
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    const long long m = m0 + wm * 32 * MB + i * 32 + r;
                    if (m >= a.M) continue;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = acc[j][i][8 * u + e] + bias[e];
                    finish8<DT, decltype(act)::value>(a, m, n, v);
                    __builtin_amdgcn_sched_barrier(0);      // (or the rows' residuals are all requested first, and spill)
                }
            }
    };
    if (a.act == TDC_ACT_RELU) finish(std::integral_constant<int, TDC_ACT_RELU>{});
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
static int launch_product(const ProductArgs &a, hipStream_t s) {
    const long long big = ((a.M + 255) / 256) * ((a.N + 255) / 256);
    if (big >= 192) return launch_tile<DT, 4, 4>(a, s);
    return launch_tile<DT, 2, 2>(a, s);
}

int launch_mx4_product(const ProductArgs &a, int y_dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (y_dtype == TDC_F32) return launch_product<TDC_F32>(a, s);
    if (y_dtype == TDC_F16) return launch_product<TDC_F16>(a, s);
    return launch_product<TDC_BF16>(a, s);
}

}  // namespace tdc
