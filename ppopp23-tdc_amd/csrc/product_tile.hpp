// Product of two matrices in 16 or 8 bits on the matrix cores, tile by tile: sums over a long axis of x[m, k] w[n, k], either
// operand with the sum's axis or with the other one as the neighbours in memory.
#pragma once
#include "product_device.hpp"

namespace tdc {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef short s4_t __attribute__((ext_vector_type(4)));

// A workgroup of four waves, WM x WN of them, owns 32 MB WM rows of x and 32 NB WN of w (below: outputs), a wave MB x NB blocks
// of 32 x 32.  A step is 64 bytes of each: 32 numbers of 16 bits, 64 of 8.
// LDS holds B steps.
template <int WM, int WN, int MB, int NB, int B>
struct Shape {
    static constexpr int M = 32 * MB * WM, N = 32 * NB * WN, kBuffers = B;
    static constexpr int kPerUnit = MB * NB <= 2 ? 2 : MB * NB <= 4 && B <= 3 ? 3 : 1;      // workgroups of a compute unit that the registers are for
    static constexpr int kBuffer = (M + N) * 64;                     // bytes of a step: x, then w
    static constexpr int kRequests = (M + N) / 16, kChunks = (kRequests + 3) / 4;   // of a step, of 1 KiB each: in all, of a wave
    static constexpr int kScaleX = (M + 63) / 64 * 64;               // (8 bits: rows of x among those whose scales are requested)
    static constexpr int kScales = (kScaleX + N) * 16;               // bytes of the scales of 512 numbers
    static constexpr int kScaleRequests = (kScaleX + N) / 64, kScaleChunks = (kScaleRequests + 3) / 4;
    static constexpr int kLds16 = kBuffers * kBuffer + N * 4, kLds8 = kBuffers * kBuffer + 2 * kScales + N * 4;
    static_assert(kBuffers * kBuffer >= 4 * NB * 4096, "what the outputs pass through");
};

// Which tile a workgroup has, if any: neighbouring workgroups of a die take tiles of eight rows by as many columns as run at once, which
// share operands in its L2.
static __device__ __forceinline__ bool tile_at(unsigned block, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int total = tiles_m * tiles_n, per_die = (total + 7) / 8;
    const int id = (block & 7) * per_die + (block >> 3);
    if ((int)(block >> 3) >= per_die || id >= total) return false;
    const int group = id / (8 * tiles_n), rest = id - group * 8 * tiles_n, high = min(8, tiles_m - group * 8);
    tm = group * 8 + rest % high;
    tn = rest / high;
    return true;
}

// The place of the 16-byte piece `piece` of row `row` in LDS, from the operand's start on.
//   Rows along the sum (T = false): a row is 64 bytes, four pieces, which change places by two bits of the row, so that the sixteen lanes whose
// 256 bytes LDS reads at once (which four fours of neighbours these are does not matter then) meet no bank twice; with those of the eight
// rows of neighbouring lanes alone (bits 1 and 2) half of the LDS cycles were conflicts.
//   Rows across it (T = true): `R` numbers of one place of the sum; its pieces change places by the row, so that 64 bytes of each of four rows,
// which 32 lanes read for a transposition, lie on different banks.
static __device__ __forceinline__ int turn_along(int row) { return row >> 2 & 3; }
template <int R>
static __device__ __forceinline__ int turn_across(int k) { return R >= 128 ? (k & 3) * 4 : R == 64 ? (k & 2) * 2 : 0; }

// How a wave brings one operand: rows `stride` bytes apart in memory; `outer` runs over what is not summed, and `outer_left` of that are there
// from the tile's first on (what lies past them repeats the last: its outputs go nowhere).
template <int IN, bool T, int R>
struct Source {
    static constexpr int kBytes = IN == TDC_MX8 ? 1 : 2, kStep = 64 / kBytes, kSlots = R * 2 / 16;
    // Of request c: this lane's offset from the step's start, and its place in the step's sum.
    static __device__ __forceinline__ void place(int c, int lane, int outer_left, int stride, int &at, int &k) {
        if constexpr (T) {
            const int row = c * (64 / kSlots) + lane / kSlots, piece = (lane % kSlots) ^ turn_across<R>(row);
            at = row * stride + min(piece * 8, outer_left - 8) * 2;
            k = row;
        } else {
            const int row = c * 16 + lane / 4, piece = (lane & 3) ^ turn_along(row);
            at = min(row, outer_left - 1) * stride + piece * 16;
            k = piece * 16 / kBytes;
        }
    }
    static __device__ __forceinline__ const unsigned char *start(const unsigned char *base, long long outer, long long stride, long long step) {
        return T ? base + outer * 2 + step * kStep * stride : base + outer * stride + step * 64;
    }
    static __device__ __forceinline__ long long advance(long long stride) { return T ? kStep * stride : 64; }
};

// Eight bytes a lane from LDS, transposed among sixteen lanes: of the four places of the sum that they point at, 32 bytes each, a lane gets
// its number of each.  (`__restrict` says nothing about so short a life that is not so, but gives the read a name for the compiler, which
// else waits for all requests into LDS before it: 1046 us for 8192 x 8192 x 8192 with both operands across the sum, 845 without that wait.)
typedef __attribute__((address_space(3))) s4_t lds_s4_t;
static __device__ __forceinline__ s4_t read_transposed(lds_s4_t *__restrict from) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(from); }

// A wave's reads of one operand from LDS: block i (32 rows from `first` on, a multiple of 32), its two halves.
template <bool T, int R, bool W, int BLOCKS>
struct Fragments {
    static constexpr int kReads = T ? 2 : 1;       // LDS reads of a half
    int at[T ? BLOCKS : 2];
    __device__ __forceinline__ void init(int lane, int first) {
        const int r = lane & 31, q = lane >> 5;
        if constexpr (T) {
            // Sixteen lanes get a number each of four places of the sum; of those that they point at lane 4 j + t holds the place j.
            const int half = lane >> 4 & 1, j = lane >> 2 & 3, t = lane & 3;
            const int column = half * 16 + (W ? (t & 1) << 3 | (t & 2) << 1 : t * 4);
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) {
                const int c = first + i * 32 + column;
                at[i] = (q * 8 + j) * R * 2 + ((c >> 3) ^ turn_across<R>(j)) * 16 + (c & 7) * 2;
            }
        } else {
            const int row = first + (W ? weight_row(r) : r), turn = turn_along(row);
#pragma unroll
            for (int p = 0; p < 2; ++p) at[p] = row * 64 + ((2 * p + q) ^ turn) * 16;
        }
    }
    // Read `part` (below kReads) of half `h` of block i, from the buffer's start for this operand on.
    __device__ __forceinline__ void read(const unsigned char *lds, int buffer, int i, int h, int part, i4_t &to) const {
        if constexpr (T) {
            const unsigned char *const from = lds + (buffer + at[i]) + (h * 16 + part * 4) * R * 2;
            const s4_t v = read_transposed((lds_s4_t *)(from));
            typedef int i2_t __attribute__((ext_vector_type(2)));
            const i2_t w = __builtin_bit_cast(i2_t, v);
            to[2 * part] = w[0];
            to[2 * part + 1] = w[1];
        } else {
            to = *reinterpret_cast<const i4_t *>(lds + (buffer + at[h]) + i * 2048);
        }
    }
};

template <int IN>
static __device__ __forceinline__ f16_t mfma16(i4_t a, i4_t b, f16_t c) {
    if constexpr (IN == TDC_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
// 8 bits: the lane's two pieces of a row's 64 numbers belong to its two blocks of 32 in turn, whose scales the lanes q = 0 and 1 hold.
static __device__ __forceinline__ f16_t mfma8(const i4_t (&a)[2], const i4_t (&b)[2], f16_t c, int sa, int sb) {
    const i8_t wa = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
    const i8_t wb = {b[0][0], b[0][1], b[0][2], b[0][3], b[1][0], b[1][1], b[1][2], b[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 0, 0, 0, sa, 0, sb);
}

// v_mfma_f32_32x32x16 and, in 8 bits, the scaled 32x32x64, sums in fp32.  The weights are the first operand, so that a lane ends up with neighbouring
// outputs of one row.  Operands come straight from global memory into LDS, `kBuffers` steps ahead, and a step's fragments from there into a
// second set of registers while the last step's are multiplied: one barrier a step, at which nothing is waited for but the requests of the
// step after the next.
//
// Measured, tiles of 256, 8192 x 8192 x 8192, in runs of a hundred: on random numbers 856 us in bf16 (1.28 PFLOP/s; w across the sum 847, both
// across it 837) and 420 to 440 in 8 bits (2.5 to 2.6), on zeros, which leave the clock up, 692 and 331; the first twenty launches behind other work take up
// to 930 and 480.  Without new requests 693 and 510 on zeros, when every tile asks for the same bytes 587 on zeros, from registers
// alone 610 and 503: a fifth of the time is operands on their way, and on numbers that are not all alike the power that these bytes take costs as much
// again.  That is not the card's limit: the library's product takes 670, 487 on zeros.  LDS is busy for 275000 of 1.5 million cycles, without conflicts; 0.8 GB come from
// beyond the L2.
//
// IN: type of the operands (TDC_F16, TDC_BF16, TDC_MX8).  XT, WT: x or w lies across the sum.  OUT: type of y, or TDC_F32 for the sums of one of
// `splits` parts of the axis, which a launch of its own joins.
template <int IN, bool XT, bool WT, int OUT, bool Z, int WM, int WN, int MB, int NB, int B>
__global__ void __launch_bounds__(256, (Shape<WM, WN, MB, NB, B>::kPerUnit)) tdc_product_tile_kernel(const TileArgs a) {
    using L = Shape<WM, WN, MB, NB, B>;
    using SX = Source<IN, XT, L::M>;
    using SW = Source<IN, WT, L::N>;
    constexpr bool kPart = OUT == TDC_F32, k8 = IN == TDC_MX8;
    constexpr int kLeft = (L::kBuffers - 2) * L::kChunks;       // requests that may be on their way when a step's numbers but one have to be there
    constexpr int kRX = L::M / 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), q = lane >> 5;
    const int wm = wave % WM, wn = wave / WM;

    int tm, tn;
    const int split = kPart ? blockIdx.x / a.blocks : 0;
    if (!tile_at(kPart ? blockIdx.x - split * a.blocks : blockIdx.x, a.tiles_m, a.tiles_n, tm, tn)) return;
    const long long m0 = (long long)tm * L::M, n0 = (long long)tn * L::N;
    const float b = kPart ? 0.0f : bias_of<kPart ? TDC_BF16 : OUT>(a, n0 + t, t < L::N);

    // Requests: what a wave's i-th one brings.
    const int first_step = split * a.split_steps, steps_here = min(a.split_steps, a.steps - first_step);
    const int x_left = (int)min((long long)L::M, a.x_outer - m0), w_left = (int)min((long long)L::N, a.w_outer - n0);
    int from[L::kChunks], place[L::kChunks];
#pragma unroll
    for (int i = 0; i < L::kChunks; ++i) {
        const int c = min(i * 4 + wave, L::kRequests - 1);
        if (c < kRX) SX::place(c, lane, x_left, (int)a.x_stride, from[i], place[i]);
        else SW::place(c - kRX, lane, w_left, (int)a.w_stride, from[i], place[i]);
    }
    const unsigned char *x_at = SX::start(a.x, m0, a.x_stride, first_step), *w_at = SW::start(a.w, n0, a.w_stride, first_step);
    const long long x_on = SX::advance(a.x_stride), w_on = SW::advance(a.w_stride);
    // Numbers of the sum that are there, from the step on that is requested next.
    int x_there = (int)min(a.x_limit - (long long)first_step * SX::kStep, (long long)steps_here * SX::kStep);
    int w_there = (int)min(a.w_limit - (long long)first_step * SW::kStep, (long long)steps_here * SW::kStep);
    auto fetch = [&](int i, int buffer) {
        const int c = min(i * 4 + wave, L::kRequests - 1);
        const bool of_x = c < kRX;
        // (an offset past the descriptor's 2 GiB brings zeros)
        const int at = place[i] < (of_x ? x_there : w_there) ? from[i] : (int)0x80000000;
        bring(of_x ? x_at : w_at, at, 0, lds + buffer + c * 1024);
    };
    auto fetched = [&] {
        x_at += x_on;
        w_at += w_on;
        x_there -= SX::kStep;
        w_there -= SW::kStep;
    };
    // 8 bits: the scales of 512 numbers, a row a lane.
    unsigned char *const lds_scales = lds + L::kBuffers * L::kBuffer;
    const int groups = (a.steps + 7) / 8;
    auto fetch_scales = [&](int g) {
        const long long at = min(first_step / 8 + g, groups - 1);
#pragma unroll
        for (int i = 0; i < L::kScaleChunks; ++i) {
            const int c = min(i * 4 + wave, L::kScaleRequests - 1);
            const bool of_x = c * 64 < L::kScaleX;
            const unsigned char *const base = of_x ? a.x_scales + (at * a.M + m0) * 16 : a.w_scales + (at * a.N + n0) * 16;
            const int row = c * 64 + lane, in = of_x ? min(row, x_left - 1) : min(row - L::kScaleX, w_left - 1);
            bring(base, in * 16, 0, lds_scales + (g & 1) * L::kScales + c * 1024);
        }
    };
    auto read_scales = [&](int g, int (&sx)[MB][2], int (&sw)[NB][2]) {
        const unsigned char *const at = lds_scales + (g & 1) * L::kScales + q * 4;
        const int r = lane & 31;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MB; ++i) sx[i][h] = *reinterpret_cast<const int *>(at + ((wm * MB + i) * 32 + r) * 16 + h * 8);
#pragma unroll
            for (int j = 0; j < NB; ++j) sw[j][h] = *reinterpret_cast<const int *>(at + (L::kScaleX + (wn * NB + j) * 32 + weight_row(r)) * 16 + h * 8);
        }
    };

    Fragments<XT, L::M, false, MB> xf;
    Fragments<WT, L::N, true, NB> wf;
    xf.init(lane, wm * MB * 32);
    wf.init(lane, wn * NB * 32);
    constexpr int kXReads = MB * xf.kReads, kWReads = NB * wf.kReads, kReads = 2 * (kXReads + kWReads);
    i4_t x[2][MB][2], w[2][NB][2];
    // LDS read n of a step's operands into register set S: all of half 0 before half 1.
    auto read = [&](auto set, int n, int buffer) {
        constexpr int S = decltype(set)::value;
        const int h = n / (kXReads + kWReads), in = n % (kXReads + kWReads);
        if (in < kWReads) wf.read(lds + L::M * 64, buffer, in / wf.kReads, h, in % wf.kReads, w[S][in / wf.kReads][h]);
        else xf.read(lds, buffer, (in - kWReads) / xf.kReads, h, (in - kWReads) % xf.kReads, x[S][(in - kWReads) / xf.kReads][h]);
    };
    f16_t acc[NB][MB];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.0f;

    float *const bias = reinterpret_cast<float *>(lds_scales + (k8 ? 2 * L::kScales : 0));
    int sx[MB][2], sw[NB][2];
    if constexpr (k8) fetch_scales(0);
#pragma unroll
    for (int s = 0; s < L::kBuffers; ++s) {
#pragma unroll
        for (int i = 0; i < L::kChunks; ++i) fetch(i, s * L::kBuffer);
        fetched();
    }
    if (t < L::N) bias[t] = b;
    meet<kLeft>();
#pragma unroll
    for (int n = 0; n < kReads; ++n) read(std::integral_constant<int, 0>{}, n, 0);
    if constexpr (k8) read_scales(0, sx, sw);
    meet<kLeft>();      // (the first step's requests go where these reads come from)

    // A step, the S-th of two: its numbers are in register set S.  Between its matrix instructions stand the
    // LDS reads of the next step and the requests of the step `kBuffers` on, one at a time, so that none of them keeps the matrix unit waiting.
    int now = 0, next = L::kBuffer;
    auto run = [&](auto parity) {
        constexpr int S = decltype(parity)::value, kMfma = (k8 ? 1 : 2) * MB * NB, kEarly = (kMfma * 3 + 3) / 4;
        const std::integral_constant<int, S ^ 1> other;
#pragma unroll
        for (int n = 0; n < kMfma; ++n) {
            const int h = n / (MB * NB), j = n % (MB * NB) / MB, i = n % MB;
            if constexpr (k8) acc[j][i] = mfma8(w[S][j], x[S][i], acc[j][i], sw[j][S], sx[i][S]);
            else acc[j][i] = mfma16<IN>(w[S][j][h], x[S][i][h], acc[j][i]);
            // (the requests evenly: four waves that ask at once would wait for the address unit, and the matrix unit with them.  The
            // reads in the first three quarters, so that none is out when the waves meet)
#pragma unroll
            for (int o = min(n * kReads / kEarly, kReads); o < min((n + 1) * kReads / kEarly, kReads); ++o) read(other, o, next);
#pragma unroll
            for (int o = n * L::kChunks / kMfma; o < (n + 1) * L::kChunks / kMfma; ++o) fetch(o, now);
            __builtin_amdgcn_sched_barrier(0);
        }
        fetched();
        now = next;
        next = next == (L::kBuffers - 1) * L::kBuffer ? 0 : next + L::kBuffer;
        if constexpr (k8 && S == 1) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < MB; ++i) sx[i][h] = (int)((unsigned)sx[i][h] >> 8);
#pragma unroll
                for (int j = 0; j < NB; ++j) sw[j][h] = (int)((unsigned)sw[j][h] >> 8);
            }
        }
        meet<kLeft>();
    };
    // (an odd number of steps is rounded up: what lies past the last number is zeros)
    const int steps = (steps_here + 1) / 2 * 2;
    int step = 0;
    if constexpr (k8) {
        for (int g = 0; step < steps; ++g) {
            fetch_scales(g + 1);
            for (const int end = min(step + 8, steps); step < end; step += 2) {
                run(std::integral_constant<int, 0>{});
                run(std::integral_constant<int, 1>{});
            }
            read_scales(g + 1, sx, sw);
        }
    } else {
        for (; step < steps; step += 2) {
            run(std::integral_constant<int, 0>{});
            run(std::integral_constant<int, 1>{});
        }
    }
    meet<0>();       // (nothing may still be on its way into LDS when the outputs pass through it, or the workgroup ends)

    unsigned char *const stage = lds + wave * NB * 4096;
    const long long m = m0 + wm * 32 * MB, n = n0 + wn * 32 * NB;
    if constexpr (kPart) {
        ProductOut o{};
        o.y = a.part + (long long)split * a.M * a.part_stride;
        o.M = a.M;
        o.N = a.N;
        o.y_stride = a.part_stride;
        finish_tile<TDC_F32, MB, NB, false, true>(o, acc, m, n, bias + wn * 32 * NB, stage);
    } else finish_tile<OUT, MB, NB, Z>(a, acc, m, n, bias + wn * 32 * NB, stage);
}

template <int IN, bool XT, bool WT, int OUT, bool Z, int WM, int WN, int MB, int NB, int B>
static int launch_tile(TileArgs &a, const TilePlan &p, hipStream_t s) {
    using L = Shape<WM, WN, MB, NB, B>;
    constexpr int kLds = IN == TDC_MX8 ? L::kLds8 : L::kLds16;
    static unsigned long long done = 0;
    auto *const fn = &tdc_product_tile_kernel<IN, XT, WT, OUT, Z, WM, WN, MB, NB, B>;
    if (int e = allow_lds((const void *)fn, kLds, done)) return e;
    fn<<<(unsigned)(p.blocks * p.splits), 256, kLds, s>>>(a);
    return (int)hipGetLastError();
}
template <int IN, bool XT, bool WT, int OUT, bool Z>
static int launch_shape(TileArgs &a, const TilePlan &p, hipStream_t s) {
    switch (p.kernel) {
        case kTile256: return launch_tile<IN, XT, WT, OUT, Z, 2, 2, 4, 4, 4>(a, p, s);
        case kTile256x128: return launch_tile<IN, XT, WT, OUT, Z, 2, 2, 4, 2, 6>(a, p, s);
        case kTile128Deep: return launch_tile<IN, XT, WT, OUT, Z, 2, 2, 2, 2, 8>(a, p, s);
        case kTile128: return launch_tile<IN, XT, WT, OUT, Z, 2, 2, 2, 2, 3>(a, p, s);
        case kTile64: return launch_tile<IN, XT, WT, OUT, Z, 2, 2, 1, 2, 6>(a, p, s);
        default: return launch_tile<IN, XT, WT, OUT, Z, 1, 4, 1, 1, 7>(a, p, s);
    }
}
// One launch, or one for the parts of the sum and one that joins them.
template <int IN, bool XT, bool WT, int OUT>
static int launch_product_of(TileArgs &a, const TilePlan &p, hipStream_t s) {
    if constexpr (!XT && !WT)
        if (p.kernel == kFewRows) return launch_product_few(a, IN, OUT, s);
    a.steps = p.steps;
    a.split_steps = p.split_steps;
    a.splits = p.splits;
    a.tiles_m = p.tm;
    a.tiles_n = p.tn;
    a.blocks = (unsigned)p.blocks;
    a.part_stride = p.part_stride;
    if (p.splits > 1) {
        if (int e = launch_shape<IN, XT, WT, TDC_F32, false>(a, p, s)) return e;
        return launch_join(a, OUT, s);
    }
    if constexpr (IN != TDC_MX8 && !XT && !WT)
        if (a.z) return launch_shape<IN, XT, WT, OUT, true>(a, p, s);
    return launch_shape<IN, XT, WT, OUT, false>(a, p, s);
}

}  // namespace tdc
