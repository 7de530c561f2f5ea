// C entry points of the channels-last operators: argument checks, plans, workspaces.
#include <algorithm>
#include <cmath>
#include <numeric>
#include <string>

#include "ops_internal.hpp"
#include "tdc_internal.hpp"

namespace tdc {
namespace {

int invalid(const std::string &what) { return api_fail(TDC_ERR_INVALID, what); }
int launched(const char *what, int err) {
    return err ? api_fail(TDC_ERR_HIP, std::string(what) + ": " + hipGetErrorString((hipError_t)err)) : (int)TDC_OK;
}
bool number(int dtype) { return dtype == TDC_F32 || dtype == TDC_F16 || dtype == TDC_BF16; }
constexpr long long kMostItems = (1ll << 32) - 1;      // of a launch
bool aligned(const void *p, int bytes) { return ((uintptr_t)p & (unsigned)(bytes - 1)) == 0; }

// ---- group norm ----

// `quantised`: tiles end at multiples of 32 channels, the blocks of the result, which is written in one launch only where rows end
// there too.  `grad`: x and dy are held side by side.
Divisor divisor(long long by) { return {(unsigned)by, by == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / by)}; }

NormPlan norm_plan(const tdc_group_norm_desc &d, bool quantised, bool grad) {
    NormPlan n{};
    const int Cg = d.C / d.groups, size = dtype_bytes(d.dtype), widest = 16 / size;
    const long long pixels = std::max<long long>(d.pixels, 1), batch = std::max(d.batch, 1);
    n.vec = d.C % widest == 0 ? widest : d.C % 2 == 0 ? 2 : 1;
    n.places = n.vec / std::gcd(n.vec, Cg);
    // Threads: the kernels' launch bounds (256 where a workgroup does not have all pixels), and at most 2048 sums in LDS.
    const int across = 256;      // vectors of a pixel
    const int most = std::min(grad ? 512 : 1024, 2048 / (grad ? 1 : n.places));
    const int whole = (int)std::min((long long)d.C, std::lcm((long long)Cg, std::lcm((long long)n.vec, quantised ? 32ll : 1ll)));
    // A tile of whole groups and vectors, of some `bytes` a pixel; groups that are too wide are shared.
    auto tile = [&](int bytes) {
        if (whole > across * n.vec) return across * n.vec;
        const int unit = std::max(1, (bytes / size + whole - 1) / whole) * whole;
        return std::min(std::min(unit, across * n.vec / whole * whole), d.C);
    };
    const bool blocks = quantised && n.vec != widest;
    n.round = quantised && !blocks && d.C % 32 ? 31 : 0;
    auto vectors = [&](int width) { return ((width + n.round) & ~n.round) / n.vec; };
    auto fits = [&](int unit) { return !blocks && unit % Cg == 0 && pixels <= (long long)(most / vectors(unit)) * 16; };
    // One launch pays where a workgroup has little to do, or every compute unit something (bf16, silu, us, one launch against two):
    // forward, 25 Ki numbers a workgroup 9.4 against 10.7; 51 Ki, 8 workgroups 12.5 against 11.0, 256 18.5 against 22.6; 100 Ki, 16 workgroups
    // 17.8 against 11.3 (28 against 12.5 into 4 bits), 128 23.1 against 22.7, 256 34.2 against 36.5 (fp32, with twice the bytes, goes by the
    // same counts, untimed).  Gradient, where the parameters need
    // a second launch in either case: 6 Ki 10.4 against 11.9; 25 Ki, 8 workgroups 16.3 against 12.0, 256 21.8 against 23.1; 51 Ki, 256 36
    // against 32.
    auto pays = [&](int unit) {
        const long long numbers = unit * pixels, workgroups = batch * ((d.C + unit - 1) / unit);
        return numbers <= (grad ? 8192 : 32768) || (workgroups >= 256 && (!grad || numbers <= 32768));
    };
    // Whole cache lines where that leaves two workgroups for every compute unit, half ones else: their neighbours come to the same
    // die.
    n.unit = tile(128);
    n.whole = fits(n.unit) && batch * ((d.C + n.unit - 1) / n.unit) >= 512 && pays(n.unit);
    if (!n.whole && fits(tile(64)) && pays(tile(64))) {
        n.unit = tile(64);
        n.whole = true;
    }
    n.tiles = (d.C + n.unit - 1) / n.unit;
    n.tiles_per_group = n.unit % Cg == 0 ? 1 : std::min(n.tiles, (Cg + n.unit - 2) / n.unit + 1);
    const int vecs = vectors(n.unit);
    const long long dealt = n.tiles * batch;
    n.threads = most;
    if (n.whole) {
        // Few workgroups: many threads with few requests each.  Many: few threads, so that several workgroups share a compute unit,
        // but two waves for each of its vector units (32 x 14 x 14 x 1024 in 16 bits: 13.5 us, 16.5 with one; 32 x 28 x 28 x 512: 19.2, 20.6
        // with four, 26.5 with eight).
        const bool many = dealt >= 512;
        while (n.threads > 64 && n.threads / 2 >= vecs && (long long)(n.threads / 2 / vecs) * (many ? 16 : 4) >= pixels &&
               (!many || dealt * n.threads >= 512 * 512)) n.threads /= 2;
        n.chunk_rows = (int)pixels;
    } else {
        // Workgroups of 256: two to a compute unit, as long as each thread has four pixels to move, and at most 256 (a sum in fp32 is no
        // longer than that before it meets others).
        n.threads = std::min(most, 256);
        const int rows = n.threads / vecs;
        const long long want = std::max(1ll, 512 / dealt);
        n.chunk_rows = (int)std::min(round_up(pixels, rows), round_up(std::clamp((pixels + want - 1) / want, 4ll * rows, 256ll * rows), rows));
    }
    n.chunks = (int)((pixels + n.chunk_rows - 1) / n.chunk_rows);
    n.held = n.vec == widest && (n.chunk_rows + n.threads / vecs - 1) / (n.threads / vecs) <= 4 ? 4 : 16;
    n.slots = n.chunks * n.tiles_per_group;
    n.run_shift = __builtin_ctz(n.vec / n.places);
    n.by_tiles = divisor(n.tiles);
    n.by_chunks = divisor(n.chunks);
    n.by_group = divisor(Cg);
    n.by_rows[0] = divisor(n.threads / vecs);
    n.by_rows[1] = divisor(n.threads / vectors(d.C - (n.tiles - 1) * n.unit));
    const int groups = std::min(n.unit, (n.unit - 1) / Cg + 2);
    n.lds = grad ? 8 * (n.threads * n.vec + groups) : 12 * n.threads * n.places + 8 * groups + 16 * (n.threads / 64);
    return n;
}
size_t stat_bytes(const tdc_group_norm_desc &d, const NormPlan &n) { return sizeof(NormStat) * d.batch * d.groups * n.slots; }
size_t part_bytes(const tdc_group_norm_desc &d, const NormPlan &n) {
    return (size_t)round_up((long long)sizeof(float2) * d.batch * d.groups * n.slots, 16);
}
size_t chan_bytes(const tdc_group_norm_desc &d, const NormPlan &n) { return (size_t)8 * d.batch * n.chunks * d.C; }

// Normalised copy of the descriptor with every stride filled in; an error code if it makes no sense.
int norm_check(const tdc_group_norm_desc *desc, tdc_group_norm_desc &d) {
    if (!desc) return invalid("group norm: null descriptor");
    d = *desc;
    if (d.batch < 0 || d.pixels < 0 || d.C < 1) return invalid("group norm: batch, pixels and C have to be 0, 0 and 1 at least");
    if (d.pixels >= (1ll << 31) || d.C >= (1 << 24)) return invalid("group norm: pixels has to be below 2^31, C below 2^24");
    if (d.groups < 1 || d.C % d.groups)
        return invalid("group norm: " + std::to_string(d.groups) + " groups do not divide " + std::to_string(d.C) + " channels");
    if (!number(d.dtype)) return invalid("group norm: dtype has to be TDC_F32, TDC_F16 or TDC_BF16");
    if (d.param_dtype != TDC_F32 && d.param_dtype != d.dtype) return invalid("group norm: param_dtype has to be TDC_F32 or dtype");
    if (d.act < TDC_ACT_NONE || d.act > TDC_ACT_SILU) return invalid("group norm: unknown activation");
    if (!(d.eps >= 0.0f) || !std::isfinite(d.eps)) return invalid("group norm: eps has to be finite and not negative");
    if (d.reserved) return invalid("group norm: reserved has to be 0");
    for (auto pair : {std::make_pair(&d.x_pixel_stride, &d.x_image_stride), std::make_pair(&d.y_pixel_stride, &d.y_image_stride)}) {
        if (*pair.first == 0) *pair.first = d.C;
        if (*pair.first < d.C) return invalid("group norm: a pixel stride below C");
        const long long image = d.pixels ? (d.pixels - 1) * *pair.first + d.C : 0;
        if (*pair.second == 0) *pair.second = d.pixels * *pair.first;
        if (d.batch > 1 && *pair.second < image) return invalid("group norm: an image stride below one image");
    }
    return TDC_OK;
}
// Whether the plan's launches can be made.  (The gradient has workgroups of 256 for the parameters: in its second launch, or by themselves.)
int plan_check(const tdc_group_norm_desc &d, const NormPlan &n, bool grad) {
    const double items = (double)d.batch * n.tiles * n.chunks * n.threads, params = grad ? (2.0 * d.C + 3) / 4 * 256 : 0.0;
    if ((n.whole ? std::max(items, params) : items + params) > kMostItems || (double)n.chunks * n.tiles_per_group > (1 << 24))
        return invalid("group norm: too large, a launch has fewer than 2^32 work items");
    return TDC_OK;
}

size_t forward_ws(const tdc_group_norm_desc &d, const NormPlan &n) { return n.whole ? 0 : stat_bytes(d, n); }
size_t backward_ws(const tdc_group_norm_desc &d, const NormPlan &n) { return part_bytes(d, n) + chan_bytes(d, n); }
NormArgs norm_args(const tdc_group_norm_desc &d, const void *x, const void *gamma, const void *beta) {
    NormArgs a{};
    a.x = x;
    a.gamma = gamma;
    a.beta = beta;
    a.x_ps = d.x_pixel_stride;
    a.x_is = d.x_image_stride;
    a.rows = d.batch * d.pixels;
    a.batch = d.batch;
    a.pixels = (int)d.pixels;
    a.C = d.C;
    a.groups = d.groups;
    a.Cg = d.C / d.groups;
    a.act = d.act;
    a.param_dtype = d.param_dtype;
    a.eps = d.eps;
    return a;
}
int ws_check(const char *what, const void *ws, size_t have, size_t need) {
    if (!need) return TDC_OK;
    if (!ws || have < need)
        return invalid(std::string(what) + ": the workspace has " + std::to_string(ws ? have : 0) + " bytes, needs " + std::to_string(need));
    if (!aligned(ws, 16)) return invalid(std::string(what) + ": the workspace is not 16-byte aligned");
    return TDC_OK;
}

// ---- 4-bit numbers ----

int mx4_range(const char *what, long long rows, long long K) {
    if (rows < 0 || K < 1) return invalid(std::string(what) + ": rows has to be 0 and K 1 at least");
    if (K > (1ll << 30) || rows > (1ll << 35) / mx4_padded(K) * 32) return invalid(std::string(what) + ": more numbers than 2^40");
    if (mx4_work_items(rows, K) > kMostItems) return invalid(std::string(what) + ": too many rows, a launch has fewer than 2^32 work items");
    return TDC_OK;
}
int mx4_check(const char *what, long long rows, long long K, const void *codes, const void *scales) {
    if (int st = mx4_range(what, rows, K)) return st;
    if (rows && (!codes || !scales)) return invalid(std::string(what) + ": null codes or scales");
    if (rows && (!aligned(codes, 16) || !aligned(scales, 16)))
        return invalid(std::string(what) + ": codes and scales have to be 16-byte aligned");
    return TDC_OK;
}

// ---- product ----

int linear_check(const tdc_mx4_linear_desc *desc, tdc_mx4_linear_desc &d) {
    if (!desc) return invalid("4-bit product: null descriptor");
    d = *desc;
    if (d.M < 0 || d.N < 0 || d.K < 1) return invalid("4-bit product: M, N and K have to be 0, 0 and 1 at least");
    if (d.K > (1ll << 24) || d.M > (1ll << 34) || d.N > (1ll << 34) || d.M > (1ll << 40) / std::max<long long>(d.N, 1))
        return invalid("4-bit product: K above 2^24 or M * N above 2^40");
    if (d.x_dtype != TDC_MX4 && !number(d.x_dtype)) return invalid("4-bit product: unknown x_dtype");
    if (!number(d.y_dtype)) return invalid("4-bit product: y_dtype has to be TDC_F32, TDC_F16 or TDC_BF16");
    if (d.bias_dtype != TDC_F32 && d.bias_dtype != d.y_dtype) return invalid("4-bit product: bias_dtype has to be TDC_F32 or y_dtype");
    if (d.act < TDC_ACT_NONE || d.act > TDC_ACT_SILU) return invalid("4-bit product: unknown activation");
    if (!d.x_stride) d.x_stride = d.K;
    if (!d.y_stride) d.y_stride = d.N;
    if (!d.residual_stride) d.residual_stride = d.N;
    if (d.x_dtype != TDC_MX4 && d.M > 1 && d.x_stride < d.K) return invalid("4-bit product: a row stride of x below K");
    if (d.M > 1 && (d.y_stride < d.N || d.residual_stride < d.N)) return invalid("4-bit product: a row stride below N");
    const bool numbers = d.x_dtype != TDC_MX4;
    if (product_work_items(d.M, d.N, d.K, numbers) > kMostItems ||
        (numbers && !product_takes_numbers(d.M, d.N, d.K) && mx4_work_items(d.M, d.K) > kMostItems))
        return invalid("4-bit product: too large, a launch has fewer than 2^32 work items");
    return TDC_OK;
}
size_t linear_codes(const tdc_mx4_linear_desc &d) { return (size_t)mx4_code_bytes(d.M, d.K); }
size_t linear_ws(const tdc_mx4_linear_desc &d) {
    return d.x_dtype == TDC_MX4 || product_takes_numbers(d.M, d.N, d.K) ? 0 : linear_codes(d) + (size_t)(d.M * mx4_scale_bytes(d.K));
}

}  // namespace
}  // namespace tdc

using namespace tdc;

// (an error message is the only thing here that allocates: no exception leaves a C entry)
#define TDC_ENTRY try
#define TDC_ENTRY_END                 \
    catch (...) {                     \
        return (int)TDC_ERR_NOMEM;    \
    }

extern "C" {

int tdc_group_norm_workspace(const tdc_group_norm_desc *desc, size_t *forward_bytes, size_t *backward_bytes) TDC_ENTRY {
    tdc_group_norm_desc d;
    if (int st = norm_check(desc, d)) return st;
    const NormPlan forward = norm_plan(d, false, false), backward = norm_plan(d, false, true);
    if (int st = plan_check(d, forward, false)) return st;
    if (int st = plan_check(d, backward, true)) return st;
    if (forward_bytes) *forward_bytes = forward_ws(d, forward);
    if (backward_bytes) *backward_bytes = backward_ws(d, backward);
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_group_norm_mx4_workspace(const tdc_group_norm_desc *desc, size_t *bytes) TDC_ENTRY {
    tdc_group_norm_desc d;
    if (int st = norm_check(desc, d)) return st;
    if (!bytes) return invalid("group norm: null argument");
    const NormPlan plan = norm_plan(d, true, false);
    if (int st = plan_check(d, plan, false)) return st;
    *bytes = forward_ws(d, plan);
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_group_norm_forward(const tdc_group_norm_desc *desc, const void *x, const void *gamma, const void *beta, void *y,
                           float *mean, float *rstd, void *ws, size_t ws_bytes, void *stream) TDC_ENTRY {
    tdc_group_norm_desc d;
    if (int st = norm_check(desc, d)) return st;
    if (!d.batch || !d.pixels) return TDC_OK;
    if (!x || !y) return invalid("group norm: null x or y");
    const NormPlan plan = norm_plan(d, false, false);
    if (int st = plan_check(d, plan, false)) return st;
    if (int st = ws_check("group norm", ws, ws_bytes, forward_ws(d, plan))) return st;
    NormArgs a = norm_args(d, x, gamma, beta);
    a.out = y;
    a.o_ps = d.y_pixel_stride;
    a.o_is = d.y_image_stride;
    a.mean = mean;
    a.rstd = rstd;
    a.stat = (NormStat *)ws;
    a.plan = plan;
    a.per_number = 1.0 / ((double)std::max<long long>(d.pixels, 1) * (d.C / d.groups));
    return launched("group norm", launch_norm_forward(a, d.dtype, stream));
}
TDC_ENTRY_END

int tdc_group_norm_forward_mx4(const tdc_group_norm_desc *desc, const void *x, const void *gamma, const void *beta, void *codes,
                               void *scales, void *ws, size_t ws_bytes, void *stream) TDC_ENTRY {
    tdc_group_norm_desc d;
    if (int st = norm_check(desc, d)) return st;
    if (!d.batch || !d.pixels) return TDC_OK;
    if (!x) return invalid("group norm: null x");
    const NormPlan plan = norm_plan(d, true, false);
    if (int st = plan_check(d, plan, false)) return st;
    if (int st = mx4_check("group norm", d.batch * d.pixels, d.C, codes, scales)) return st;
    if (int st = ws_check("group norm", ws, ws_bytes, forward_ws(d, plan))) return st;
    NormArgs a = norm_args(d, x, gamma, beta);
    a.codes = (unsigned char *)codes;
    a.scales = (unsigned char *)scales;
    a.stat = (NormStat *)ws;
    a.plan = plan;
    a.per_number = 1.0 / ((double)std::max<long long>(d.pixels, 1) * (d.C / d.groups));
    return launched("group norm", launch_norm_forward(a, d.dtype, stream));
}
TDC_ENTRY_END

int tdc_group_norm_backward(const tdc_group_norm_desc *desc, const void *x, const void *dy, const void *gamma, const void *beta,
                            const float *mean, const float *rstd, void *dx, float *dgamma, float *dbeta, void *ws,
                            size_t ws_bytes, void *stream) TDC_ENTRY {
    tdc_group_norm_desc d;
    if (int st = norm_check(desc, d)) return st;
    if (!dx && !dgamma && !dbeta) return TDC_OK;
    if (!d.batch || !d.pixels) {
        // no numbers: the parameters' gradients are sums of nothing
        if (dgamma)
            if (int e = launch_zero_words((unsigned *)dgamma, d.C, stream)) return launched("group norm", e);
        if (dbeta)
            if (int e = launch_zero_words((unsigned *)dbeta, d.C, stream)) return launched("group norm", e);
        return TDC_OK;
    }
    if (!x || !dy || !mean || !rstd) return invalid("group norm: null x, dy, mean or rstd");
    const NormPlan plan = norm_plan(d, false, true);
    if (int st = plan_check(d, plan, true)) return st;
    if (int st = ws_check("group norm", ws, ws_bytes, backward_ws(d, plan))) return st;
    NormArgs a = norm_args(d, x, gamma, beta);
    a.dy = dy;
    a.d_ps = d.y_pixel_stride;
    a.d_is = d.y_image_stride;
    a.out = dx;
    a.o_ps = d.C;
    a.o_is = d.pixels * d.C;
    a.mean = const_cast<float *>(mean);
    a.rstd = const_cast<float *>(rstd);
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    a.plan = plan;
    a.per_number = 1.0 / ((double)std::max<long long>(d.pixels, 1) * (d.C / d.groups));
    a.part = (float2 *)ws;
    a.chan = (float *)((char *)ws + part_bytes(d, a.plan));
    return launched("group norm", launch_norm_backward(a, d.dtype, stream));
}
TDC_ENTRY_END

int tdc_mx4_sizes(int64_t rows, int64_t K, size_t *code_bytes, size_t *scale_bytes) TDC_ENTRY {
    if (int st = mx4_range("4-bit numbers", rows, K)) return st;
    if (code_bytes) *code_bytes = (size_t)mx4_code_bytes(rows, K);
    if (scale_bytes) *scale_bytes = (size_t)(rows * mx4_scale_bytes(K));
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_mx4_quantize(const void *x, int32_t dtype, int64_t rows, int64_t K, int64_t row_stride, void *codes, void *scales, void *stream) TDC_ENTRY {
    if (!number(dtype)) return invalid("4-bit numbers: dtype has to be TDC_F32, TDC_F16 or TDC_BF16");
    if (int st = mx4_check("4-bit numbers", rows, K, codes, scales)) return st;
    if (!rows) return TDC_OK;
    if (!x) return invalid("4-bit numbers: null x");
    if (!row_stride) row_stride = K;
    if (rows > 1 && row_stride < K) return invalid("4-bit numbers: a row stride below K");
    return launched("4-bit numbers", launch_mx4_quantize(x, dtype, rows, K, row_stride, codes, scales, stream));
}
TDC_ENTRY_END

int tdc_mx4_dequantize(const void *codes, const void *scales, int64_t rows, int64_t K, void *y, int32_t dtype, int64_t row_stride,
                       void *stream) TDC_ENTRY {
    if (!number(dtype)) return invalid("4-bit numbers: dtype has to be TDC_F32, TDC_F16 or TDC_BF16");
    if (int st = mx4_check("4-bit numbers", rows, K, codes, scales)) return st;
    if (!rows) return TDC_OK;
    if (!y) return invalid("4-bit numbers: null y");
    if (!row_stride) row_stride = K;
    if (rows > 1 && row_stride < K) return invalid("4-bit numbers: a row stride below K");
    return launched("4-bit numbers", launch_mx4_dequantize(codes, scales, rows, K, y, dtype, row_stride, stream));
}
TDC_ENTRY_END

int tdc_mx4_linear_workspace(const tdc_mx4_linear_desc *desc, size_t *bytes) TDC_ENTRY {
    tdc_mx4_linear_desc d;
    if (int st = linear_check(desc, d)) return st;
    if (!bytes) return invalid("4-bit product: null argument");
    *bytes = linear_ws(d);
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_mx4_linear(const tdc_mx4_linear_desc *desc, const void *x, const void *x_scales, const void *w_codes, const void *w_scales,
                   const void *bias, const void *residual, void *y, void *ws, size_t ws_bytes, void *stream) TDC_ENTRY {
    tdc_mx4_linear_desc d;
    if (int st = linear_check(desc, d)) return st;
    if (!d.M || !d.N) return TDC_OK;
    if (!x || !y) return invalid("4-bit product: null x or y");
    if (int st = mx4_check("4-bit product", d.N, d.K, w_codes, w_scales)) return st;
    ProductArgs a{};
    if (d.x_dtype == TDC_MX4) {
        if (int st = mx4_check("4-bit product", d.M, d.K, x, x_scales)) return st;
        a.x_codes = (const unsigned char *)x;
        a.x_scales = (const unsigned char *)x_scales;
    } else if (product_takes_numbers(d.M, d.N, d.K)) {
        a.x = x;
        a.x_dtype = d.x_dtype;
        a.x_stride = d.x_stride;
    } else {
        if (int st = ws_check("4-bit product", ws, ws_bytes, linear_ws(d))) return st;
        a.x_codes = (const unsigned char *)ws;
        a.x_scales = a.x_codes + linear_codes(d);
        if (int e = launch_mx4_quantize(x, d.x_dtype, d.M, d.K, d.x_stride, ws, (char *)ws + linear_codes(d), stream))
            return launched("4-bit product", e);
    }
    a.w_codes = (const unsigned char *)w_codes;
    a.w_scales = (const unsigned char *)w_scales;
    a.bias = bias;
    a.residual = residual;
    a.y = y;
    a.M = d.M;
    a.N = d.N;
    a.K = d.K;
    a.y_stride = d.y_stride;
    a.r_stride = d.residual_stride;
    a.ksteps = (int)(mx4_padded(d.K) / 128);
    a.bias_dtype = d.bias_dtype;
    a.act = d.act;
    return launched("4-bit product", launch_mx4_product(a, d.y_dtype, stream));
}
TDC_ENTRY_END

}  // extern "C"
