// Product of two matrices in microscaled 4-bit floating point: y = act(x w^T + bias + residual).
//
// v_mfma_scale_f32_16x16x128: a lane holds one block of 32 numbers of its row (lane mod 16), place lane / 16 of the four of
// a step, with that block's scale; products and sums are fp32.  The weights are the first operand, so that a lane ends
// up with neighbouring outputs of one row.
#include "ops_device.hpp"

namespace tdc {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// One matrix instruction; the low bytes of the scale words are this step's.
static __device__ __forceinline__ f4_t mfma4(i4_t a, i4_t b, f4_t c, int sa, int sb) {
    const i8_t wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

// Eight neighbouring outputs of a row (those before `n_end`): bias, residual, activation, store.
template <int DT>
static __device__ __forceinline__ void finish8(const ProductArgs &a, long long m, long long n, float (&v)[8], const float (&bias)[8]) {
    using T = typename Num<DT>::type;
    typedef T vec_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    T *const to = reinterpret_cast<T *>(a.y) + m * a.y_stride + n;
    const T *const add = reinterpret_cast<const T *>(a.residual) + m * a.r_stride + n;
    const int count = (int)min(8ll, a.N - n);
    vec_t r = {};
    if (a.residual) {
        if (count == 8) r = *reinterpret_cast<const vec_t *>(add);
        else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < count) r[i] = add[i];
        }
    }
    vec_t out;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float u = v[i] + bias[i] + Num<DT>::up(r[i]);
        if (a.act == TDC_ACT_RELU) u = act_of<TDC_ACT_RELU>(u);
        if (a.act == TDC_ACT_SILU) u = act_of<TDC_ACT_SILU>(u);
        out[i] = Num<DT>::down(u);
    }
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
// A workgroup of four waves owns 32 MF rows of x and 32 NF of w, a wave a quarter of it: MF x NF blocks of 16 x 16.  A step is
// 128 numbers of each row.  Codes go from global memory through registers into four LDS buffers, a step each, two steps ahead of
// their use; scales do so for four steps at a time.  A wave's step has NF parts of MF matrix instructions; each part starts the
// LDS reads of the weights two parts ahead (the last part those of the next step's x), stores what global memory has brought for
// the step after the next, and asks for the step behind it, so that one wave to a SIMD keeps the matrix unit fed across its
// one barrier a step.
//
// LDS holds a row's 64 bytes as four places of 16, place p of row i at p ^ fold(i): neither the stores (four lanes a row)
// nor the reads (eight rows at one place) meet on a bank.
static __device__ __forceinline__ int fold(int row) { return (row >> 1 & 3) ^ (row >> 3 & 1) << 1; }

// The row of w that is row r of a wave's block j: two blocks together hold 32 neighbouring rows, such that a lane's eight outputs
// from them are neighbours.
static __device__ __forceinline__ int weight_row(int j, int r) { return j / 2 * 32 + r / 4 * 8 + j % 2 * 4 + r % 4; }

template <int MF, int NF>
struct Tile {
    static constexpr int M = 32 * MF, N = 32 * NF;
    static constexpr int kBuffer = (M + N) * 64;              // bytes of a step's codes: x, then w
    static constexpr int kScales = (M + N) * 16;              // bytes of four steps' scales
    static constexpr int kLds = 4 * kBuffer + 2 * kScales;
    static constexpr int kX = MF / 2, kW = NF / 2, kChunks = kX + kW;   // requests of 16 bytes a thread and step
};

template <int DT, int MF, int NF>
__global__ void __launch_bounds__(256, MF * NF > 32 ? 1 : 2) tdc_mx4_product_tile_kernel(const ProductArgs a, int tiles_m, int tiles_n) {
    using L = Tile<MF, NF>;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 15, q = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;

    // Neighbouring workgroups of a die take tiles of eight rows by as many columns as run at once: they share operands in its L2.
    const int total = tiles_m * tiles_n, per_die = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per_die + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per_die || id >= total) return;
    const int group = id / (8 * tiles_n), rest = id - group * 8 * tiles_n, high = min(8, tiles_m - group * 8);
    const long long m0 = (long long)(group * 8 + rest % high) * L::M, n0 = (long long)(rest / high) * L::N;

    const long long pitch = (long long)a.ksteps * 64;
    const int last = a.ksteps - 1, last_m = (int)min((long long)L::M, a.M - m0) - 1, last_n = (int)min((long long)L::N, a.N - n0) - 1;
    const unsigned char *const xc = a.x_codes + m0 * pitch, *const wc = a.w_codes + n0 * pitch;
    const int q_in = (t & 3) ^ fold(t >> 2);
    unsigned from[L::kChunks];          // (rows past the last repeat it: their products go nowhere)
#pragma unroll
    for (int i = 0; i < L::kChunks; ++i) {
        const int row = (i < L::kX ? i : i - L::kX) * 64 + (t >> 2);
        from[i] = (unsigned)(min(row, i < L::kX ? last_m : last_n) * pitch) + q_in * 16;
    }
    i4_t chunk[L::kChunks];
    auto fetch = [&](int i, int step) {
        const long long k = (long long)min(step, last) * 64;
        chunk[i] = *reinterpret_cast<const i4_t *>((i < L::kX ? xc : wc) + k + from[i]);
    };
    auto park = [&](int i, int buffer) { *reinterpret_cast<i4_t *>(lds + buffer + i * 4096 + t * 16) = chunk[i]; };

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

    const int x_row = wm * 16 * MF + r, w_row = wn * 16 * NF + weight_row(0, r);
    const int x_at = x_row * 64 + (q ^ fold(x_row)) * 16, w_even = L::M * 64 + w_row * 64 + (q ^ fold(w_row)) * 16,
              w_odd = L::M * 64 + (w_row + 4) * 64 + (q ^ fold(w_row + 4)) * 16;
    auto x_frag = [&](int i, int buffer) { return *reinterpret_cast<const i4_t *>(lds + buffer + x_at + i * 1024); };
    auto w_frag = [&](int j, int buffer) { return *reinterpret_cast<const i4_t *>(lds + buffer + (j & 1 ? w_odd : w_even) + j / 2 * 2048); };
    auto read_scales = [&](int g, int (&sx)[MF], int (&sw)[NF]) {
        const unsigned char *const at = lds_scales + (g & 1) * L::kScales + q * 4;
#pragma unroll
        for (int i = 0; i < MF; ++i) sx[i] = *reinterpret_cast<const int *>(at + (x_row + i * 16) * 16);
#pragma unroll
        for (int j = 0; j < NF; ++j) sw[j] = *reinterpret_cast<const int *>(at + (L::M + wn * 16 * NF + weight_row(j, r)) * 16);
    };
    auto meet = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    f4_t acc[NF][MF];
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 0; i < MF; ++i) acc[j][i] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < L::kChunks; ++i) fetch(i, s);
        fetch_scales(s);
#pragma unroll
        for (int i = 0; i < L::kChunks; ++i) park(i, s * L::kBuffer);
        park_scales(s);
    }
#pragma unroll
    for (int i = 0; i < L::kChunks; ++i) fetch(i, 2);
    fetch_scales(2);
    meet();
    i4_t x[MF], w[4];
    int sx[MF], sw[NF];
#pragma unroll
    for (int i = 0; i < MF; ++i) x[i] = x_frag(i, 0);
    w[0] = w_frag(0, 0);
    w[1] = w_frag(1, 0);
    read_scales(0, sx, sw);
    meet();       // (the first group of steps overwrites the buffer that this read)

    int step = 0;
    for (int g = 0; g < groups; ++g) {
        // Four steps: their scales are in registers, those of the next four in LDS, the next but one on their way.
        int next_sx[MF], next_sw[NF];
        read_scales(g + 1, next_sx, next_sw);
        park_scales(g + 2);
        fetch_scales(g + 3);
        for (const int end = min(step + 4, a.ksteps); step < end; ++step) {
            const int now = (step & 3) * L::kBuffer, next = (step + 1 & 3) * L::kBuffer, fill = (step + 2 & 3) * L::kBuffer;
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                w[(j + 2) & 3] = j + 2 < NF ? w_frag(j + 2, now) : w_frag(j + 2 - NF, next);
#pragma unroll
                for (int i = j * L::kChunks / NF; i < (j + 1) * L::kChunks / NF; ++i) {
                    park(i, fill);
                    fetch(i, step + 3);
                }
#pragma unroll
                for (int i = 0; i < MF; ++i) {
                    acc[j][i] = mfma4(w[j & 3], x[i], acc[j][i], sw[j], sx[i]);
                    if (j == NF - 1) x[i] = x_frag(i, next);      // (its last use in this step)
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < MF; ++i) sx[i] = (int)((unsigned)sx[i] >> 8);
#pragma unroll
            for (int j = 0; j < NF; ++j) sw[j] = (int)((unsigned)sw[j] >> 8);
            meet();
        }
#pragma unroll
        for (int i = 0; i < MF; ++i) sx[i] = next_sx[i];
#pragma unroll
        for (int j = 0; j < NF; ++j) sw[j] = next_sw[j];
    }

#pragma unroll
    for (int p = 0; p < NF / 2; ++p) {
        const long long n = n0 + wn * 16 * NF + p * 32 + q * 8;
        if (n >= a.N) continue;
        float bias[8];
        bias8<DT>(a, n, bias);
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            const long long m = m0 + wm * 16 * MF + i * 16 + r;
            if (m >= a.M) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = acc[2 * p][i][e];
                v[4 + e] = acc[2 * p + 1][i][e];
            }
            finish8<DT>(a, m, n, v, bias);
            __builtin_amdgcn_sched_barrier(0);      // (or the rows' residuals are all requested first, and spill)
        }
    }
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

template <int DT, int MF, int NF>
static int launch_tile(const ProductArgs &a, hipStream_t s) {
    using L = Tile<MF, NF>;
    static unsigned long long done = 0;
    auto *const fn = &tdc_mx4_product_tile_kernel<DT, MF, NF>;
    if (int e = allow_lds((const void *)fn, L::kLds, done)) return e;
    const int tm = (int)((a.M + L::M - 1) / L::M), tn = (int)((a.N + L::N - 1) / L::N);
    const unsigned grid = (unsigned)(((long long)tm * tn + 7) / 8 * 8);
    fn<<<grid, 256, L::kLds, s>>>(a, tm, tn);
    return (int)hipGetLastError();
}
template <int DT>
static int launch_product(const ProductArgs &a, hipStream_t s) {
    const long long big = ((a.M + 255) / 256) * ((a.N + 255) / 256);
    if (big >= 192) return launch_tile<DT, 8, 8>(a, s);
    return launch_tile<DT, 4, 4>(a, s);
}

int launch_mx4_product(const ProductArgs &a, int y_dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (y_dtype == TDC_F32) return launch_product<TDC_F32>(a, s);
    if (y_dtype == TDC_F16) return launch_product<TDC_F16>(a, s);
    return launch_product<TDC_BF16>(a, s);
}

}  // namespace tdc
