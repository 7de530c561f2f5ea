// C entry points of the products in 16 and 8 bits and of RMS norm: argument checks, plans, workspaces.
#include <algorithm>
#include <cmath>

#include "ops_checks.hpp"

namespace tdc {
namespace {

constexpr long long kMostAlong = 1ll << 21, kMostStride = 1ll << 22;      // numbers of a row, between rows (requests have 32-bit offsets)
bool half(int dtype) { return dtype == TDC_F16 || dtype == TDC_BF16; }

int plan_fits(const char *what, const TilePlan &p) {
    if (p.items > kMostItems) return invalid(std::string(what) + ": too large, a launch has fewer than 2^32 work items");
    return TDC_OK;
}
// The sizes of a product: M rows by N outputs.
int sizes_check(const char *what, long long M, long long N, long long K) {
    if (M < 0 || N < 0 || K < 1) return invalid(std::string(what) + ": M, N and K have to be 0, 0 and 1 at least");
    if (K > kMostAlong || N > kMostAlong || M >= (1ll << 31)) return invalid(std::string(what) + ": N or K above 2^21, or M not below 2^31");
    return TDC_OK;
}

// ---- 16 bits ----

// Whether rows of n numbers have to be copied before a tile can request them, 16 bytes at a time.
bool must_pack(long long rows, long long n, long long stride) {
    return n % 8 != 0 || (rows > 1 && (stride % 8 != 0 || stride >= kMostStride));
}
size_t packed_bytes(long long rows, long long n) { return (size_t)(rows * round_up(n, 8) * 2); }
size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

int linear_check(const tdc_linear_desc *desc, tdc_linear_desc &d) {
    if (!desc) return invalid("product: null descriptor");
    d = *desc;
    if (int st = sizes_check("product", d.M, d.N, d.K)) return st;
    if (!half(d.dtype)) return invalid("product: dtype has to be TDC_F16 or TDC_BF16");
    if (d.bias_dtype != TDC_F32 && d.bias_dtype != d.dtype) return invalid("product: bias_dtype has to be TDC_F32 or dtype");
    if (d.kept_dtype != TDC_MX8 && d.kept_dtype != d.dtype) return invalid("product: kept_dtype has to be dtype or TDC_MX8");
    if (d.act < TDC_ACT_NONE || d.act > TDC_ACT_SILU) return invalid("product: unknown activation");
    if (!d.x_stride) d.x_stride = d.K;
    if (!d.w_stride) d.w_stride = d.K;
    if (!d.y_stride) d.y_stride = d.N;
    if (!d.residual_stride) d.residual_stride = d.N;
    if ((d.M > 1 && (d.x_stride < d.K || d.y_stride < d.N || d.residual_stride < d.N)) || (d.N > 1 && d.w_stride < d.K))
        return invalid("product: a row stride below the row");
    return TDC_OK;
}
ActGradArgs copy_args(const void *from, long long rows, long long n, long long stride, void *to) {
    ActGradArgs a{};
    a.dy = from;
    a.dz = to;
    a.M = rows;
    a.N = n;
    a.dy_stride = stride;
    act_grad_plan(a);
    return a;
}
// Copies and the gradient's first pass are one launch.
struct Copies {
    long long items = 0;
    void add(long long rows, long long n) { items += act_grad_items(copy_args(nullptr, rows, n, n, nullptr)); }
    int fit() const { return items > kMostItems ? invalid("product: too large, a launch has fewer than 2^32 work items") : (int)TDC_OK; }
};

// What a pass does, and where its scratch lies.
struct Forward {
    TilePlan plan;
    size_t x = 0, w = 0, part = 0, all = 0;
    bool pack_x, pack_w;
};
int forward_plan(const tdc_linear_desc &d, Forward &f) {
    f.plan = tile_plan(d.M, d.N, d.K, d.dtype, kAlong);
    if (int st = plan_fits("product", f.plan)) return st;
    Copies copies;
    if ((f.pack_x = must_pack(d.M, d.K, d.x_stride))) copies.add(d.M, d.K);
    if ((f.pack_w = must_pack(d.N, d.K, d.w_stride))) copies.add(d.N, d.K);
    if (int st = copies.fit()) return st;
    f.w = f.x + (f.pack_x ? padded(packed_bytes(d.M, d.K)) : 0);
    f.part = f.w + (f.pack_w ? padded(packed_bytes(d.N, d.K)) : 0);
    f.all = f.part + (size_t)f.plan.part_bytes;
    return TDC_OK;
}
struct Backward {
    TilePlan dx, dw;
    size_t dz = 0, sums = 0, x = 0, w = 0, part = 0, all = 0;
    bool make_dz, pack_x, pack_w;       // (make_dz: dy is not dz as it lies)
    ActGradArgs grad;
};
// (dz_given: the caller takes dz as a result, and there it lies)
int backward_plan(const tdc_linear_desc &d, bool dz_given, Backward &b) {
    b.dx = tile_plan(d.M, d.K, d.N, d.dtype, kWAcross);
    b.dw = tile_plan(d.N, d.K, d.M, d.dtype, kAcross);
    if (int st = plan_fits("product's gradient", b.dx)) return st;
    if (int st = plan_fits("product's gradient", b.dw)) return st;
    b.make_dz = d.act != TDC_ACT_NONE || must_pack(d.M, d.N, d.y_stride);
    b.pack_x = d.kept_dtype == TDC_MX8 || must_pack(d.M, d.K, d.x_stride);
    b.pack_w = must_pack(d.N, d.K, d.w_stride);
    Copies copies;
    copies.add(d.M, d.N);
    if (b.pack_x && d.kept_dtype != TDC_MX8) copies.add(d.M, d.K);
    if (b.pack_w) copies.add(d.N, d.K);
    if (int st = copies.fit()) return st;
    if (d.kept_dtype == TDC_MX8)
        if (int st = mx_range("product's gradient", d.M, d.K)) return st;
    b.grad = copy_args(nullptr, d.M, d.N, d.y_stride, nullptr);
    b.sums = b.dz + (b.make_dz && !dz_given ? padded(packed_bytes(d.M, d.N)) : 0);
    b.x = b.sums + padded((size_t)b.grad.chunks * d.N * 4);
    b.w = b.x + (b.pack_x ? padded(packed_bytes(d.M, d.K)) : 0);
    b.part = b.w + (b.pack_w ? padded(packed_bytes(d.N, d.K)) : 0);
    b.all = b.part + (size_t)std::max(b.dx.part_bytes, b.dw.part_bytes);
    return TDC_OK;
}
int launch_16(const TileArgs &a, const TilePlan &p, int layout, int dtype, void *stream) {
    return dtype == TDC_F16 ? launch_product_f16(a, p, layout, stream) : launch_product_bf16(a, p, layout, stream);
}
// An operand as it lies, or copied to `at` where it must be.
struct Lying {
    const unsigned char *at;
    long long stride, width;      // bytes between rows, numbers of a row
};
Lying lying(const void *p, long long rows, long long n, long long stride, bool packed) {
    const long long width = packed ? round_up(n, 8) : n;
    return {(const unsigned char *)p, (packed || rows <= 1 ? round_up(n, 8) : stride) * 2, width};
}

// ---- 8 bits ----

int linear8_check(const tdc_mx4_linear_desc *desc, tdc_mx4_linear_desc &d, TilePlan &p) {
    if (!desc) return invalid("8-bit product: null descriptor");
    d = *desc;
    if (int st = sizes_check("8-bit product", d.M, d.N, d.K)) return st;
    if (d.x_dtype != TDC_MX8 && !number(d.x_dtype)) return invalid("8-bit product: unknown x_dtype");
    if (!half(d.y_dtype)) return invalid("8-bit product: y_dtype has to be TDC_F16 or TDC_BF16");
    if (d.bias_dtype != TDC_F32 && d.bias_dtype != d.y_dtype) return invalid("8-bit product: bias_dtype has to be TDC_F32 or y_dtype");
    if (d.act < TDC_ACT_NONE || d.act > TDC_ACT_SILU) return invalid("8-bit product: unknown activation");
    if (!d.x_stride) d.x_stride = d.K;
    if (!d.y_stride) d.y_stride = d.N;
    if (!d.residual_stride) d.residual_stride = d.N;
    if (d.x_dtype != TDC_MX8 && d.M > 1 && d.x_stride < d.K) return invalid("8-bit product: a row stride of x below K");
    if (d.M > 1 && (d.y_stride < d.N || d.residual_stride < d.N)) return invalid("8-bit product: a row stride below N");
    p = tile_plan(std::max<long long>(d.M, 1), std::max<long long>(d.N, 1), d.K, TDC_MX8, kAlong);
    if (int st = plan_fits("8-bit product", p)) return st;
    return d.x_dtype == TDC_MX8 ? (int)TDC_OK : mx_range("8-bit product", d.M, d.K);
}
size_t x8_codes(const tdc_mx4_linear_desc &d) { return (size_t)(d.M * mx8_pitch(d.K)); }
size_t x8_bytes(const tdc_mx4_linear_desc &d) {
    return d.x_dtype == TDC_MX8 ? 0 : padded(x8_codes(d) + (size_t)(d.M * mx4_scale_bytes(d.K)));
}

// ---- RMS norm ----

int rms_check(const tdc_rms_norm_desc *desc, tdc_rms_norm_desc &d) {
    if (!desc) return invalid("RMS norm: null descriptor");
    d = *desc;
    if (d.rows < 0 || d.C < 1) return invalid("RMS norm: rows and C have to be 0 and 1 at least");
    if (d.C > 8192 || d.rows > (1ll << 40) / d.C) return invalid("RMS norm: C above 8192, or more than 2^40 numbers");
    if (!number(d.dtype)) return invalid("RMS norm: dtype has to be TDC_F32, TDC_F16 or TDC_BF16");
    if (d.weight_dtype != TDC_F32 && d.weight_dtype != d.dtype) return invalid("RMS norm: weight_dtype has to be TDC_F32 or dtype");
    if (!(d.eps >= 0.0f) || !std::isfinite(d.eps)) return invalid("RMS norm: eps has to be finite and not negative");
    for (int64_t *s : {&d.x_stride, &d.residual_stride, &d.dy_stride, &d.dh_stride}) {
        if (!*s) *s = d.C;
        if (d.rows > 1 && *s < d.C) return invalid("RMS norm: a row stride below C");
    }
    return TDC_OK;
}
// The launch's arguments, with its plan.
int rms_args(const tdc_rms_norm_desc &d, const void *weight, bool grad, RmsArgs &a) {
    a = RmsArgs{};
    a.weight = weight;
    a.rows = d.rows;
    a.C = d.C;
    a.weight_dtype = d.weight_dtype;
    a.eps = d.eps;
    a.x_stride = d.x_stride;
    a.r_stride = d.residual_stride;
    a.dy_stride = d.dy_stride;
    a.dh_stride = d.dh_stride;
    rms_plan(a, grad);
    if (rms_items(a, grad) > kMostItems) return invalid("RMS norm: too large, a launch has fewer than 2^32 work items");
    return TDC_OK;
}

}  // namespace
}  // namespace tdc

using namespace tdc;

extern "C" {

int tdc_linear_workspace(const tdc_linear_desc *desc, size_t *forward_bytes, size_t *backward_bytes) TDC_ENTRY {
    tdc_linear_desc d;
    if (int st = linear_check(desc, d)) return st;
    Forward f;
    Backward b;
    const bool some = d.M && d.N;      // (nothing has no plan)
    if (forward_bytes) {
        if (int st = some ? forward_plan(d, f) : TDC_OK) return st;
        *forward_bytes = f.all;
    }
    if (backward_bytes) {
        if (int st = some ? backward_plan(d, false, b) : TDC_OK) return st;
        *backward_bytes = b.all;
    }
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_linear_backward_workspace(const tdc_linear_desc *desc, int32_t dz_given, size_t *bytes) TDC_ENTRY {
    tdc_linear_desc d;
    if (int st = linear_check(desc, d)) return st;
    if (!bytes) return invalid("product's gradient: null argument");
    Backward b;
    if (int st = d.M && d.N ? backward_plan(d, dz_given != 0, b) : TDC_OK) return st;
    *bytes = b.all;
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_linear_forward(const tdc_linear_desc *desc, const void *x, const void *w, const void *bias, const void *residual, void *y, void *z,
                       void *ws, size_t ws_bytes, void *stream) TDC_ENTRY {
    tdc_linear_desc d;
    if (int st = linear_check(desc, d)) return st;
    if (!d.M || !d.N) return TDC_OK;
    if (!x || !w || !y) return invalid("product: null x, w or y");
    if (!aligned(x, 16) || !aligned(w, 16)) return invalid("product: x and w have to be 16-byte aligned");
    Forward f;
    if (int st = forward_plan(d, f)) return st;
    if (int st = ws_check("product", ws, ws_bytes, f.all)) return st;
    char *const scratch = (char *)ws;
    ActGradArgs jobs[2];
    int n = 0;
    if (f.pack_x) {
        jobs[n++] = copy_args(x, d.M, d.K, d.x_stride, scratch + f.x);
        x = scratch + f.x;
    }
    if (f.pack_w) {
        jobs[n++] = copy_args(w, d.N, d.K, d.w_stride, scratch + f.w);
        w = scratch + f.w;
    }
    if (int e = launch_act_grad(jobs, n, d.dtype, stream)) return launched("product", e);
    const Lying lx = lying(x, d.M, d.K, d.x_stride, f.pack_x), lw = lying(w, d.N, d.K, d.w_stride, f.pack_w);
    TileArgs a{};
    a.x = lx.at;
    a.w = lw.at;
    a.x_stride = lx.stride;
    a.w_stride = lw.stride;
    a.x_outer = d.M;
    a.w_outer = d.N;
    a.x_limit = lx.width;
    a.w_limit = lw.width;
    a.bias = bias;
    a.residual = residual;
    a.y = y;
    a.z = z;
    a.M = d.M;
    a.N = d.N;
    a.y_stride = d.y_stride;
    a.r_stride = d.residual_stride;
    a.z_stride = d.N;
    a.bias_dtype = d.bias_dtype;
    a.act = d.act;
    a.part = (float *)(scratch + f.part);
    return launched("product", launch_16(a, f.plan, kAlong, d.dtype, stream));
}
TDC_ENTRY_END

int tdc_linear_backward(const tdc_linear_desc *desc, const void *x, const void *x_scales, const void *w, const void *kept, const void *dy,
                        void *dx, void *dw, void *dbias, void *dz, void *ws, size_t ws_bytes, void *stream) TDC_ENTRY {
    const char *const what = "product's gradient";
    tdc_linear_desc d;
    if (int st = linear_check(desc, d)) return st;
    if (!dx && !dw && !dbias && !dz) return TDC_OK;
    if (!d.M || !d.N) {
        // sums of nothing
        if (dw && d.N)
            if (int e = launch_zeros(dw, d.N * d.K, d.dtype, stream)) return launched(what, e);
        if (dbias && d.N)
            if (int e = launch_zeros(dbias, d.N, d.bias_dtype, stream)) return launched(what, e);
        if (dx && d.M)
            if (int e = launch_zeros(dx, d.M * d.K, d.dtype, stream)) return launched(what, e);
        return TDC_OK;
    }
    Backward b;
    if (int st = backward_plan(d, dz != nullptr, b)) return st;
    if (!dy || (dw && !x) || (dx && !w)) return invalid("product's gradient: null x, w or dy");
    if (dw && (d.kept_dtype == TDC_MX8) != (x_scales != nullptr)) return invalid("product's gradient: scales go with x in 8 bits");
    if (d.act != TDC_ACT_NONE && !kept) return invalid("product's gradient: an activation's gradient needs what it was taken of");
    if (!aligned(dy, 16) || (dw && !aligned(x, 16)) || (dw && x_scales && !aligned(x_scales, 16)) || (dx && !aligned(w, 16)) || (dz && !aligned(dz, 16)))
        return invalid("product's gradient: x, w, dy and dz have to be 16-byte aligned");
    if (int st = ws_check(what, ws, ws_bytes, b.all)) return st;
    char *const scratch = (char *)ws;
    // dz, and its sums
    void *made = dz ? dz : b.make_dz && (dx || dw) ? scratch + b.dz : nullptr;
    ActGradArgs jobs[3];
    int n = 0;
    if (made || dbias) {
        ActGradArgs &g = jobs[n++] = b.grad;
        g.dy = dy;
        g.kept = kept;
        g.dz = made;
        g.sums = dbias;
        g.part = (float *)(scratch + b.sums);
        g.act = d.act;
        g.sums_dtype = d.bias_dtype;
    }
    // (and what no tile can take as it lies)
    if (dx && b.pack_w) {
        jobs[n++] = copy_args(w, d.N, d.K, d.w_stride, scratch + b.w);
        w = scratch + b.w;
    }
    if (dw && b.pack_x && d.kept_dtype != TDC_MX8) {
        jobs[n++] = copy_args(x, d.M, d.K, d.x_stride, scratch + b.x);
        x = scratch + b.x;
    }
    if (int e = launch_act_grad(jobs, n, d.dtype, stream)) return launched(what, e);
    const Lying lz = made ? lying(made, d.M, d.N, 0, true) : lying(dy, d.M, d.N, d.y_stride, false);
    TileArgs a{};
    a.x = lz.at;
    a.x_stride = lz.stride;
    a.part = (float *)(scratch + b.part);
    a.act = TDC_ACT_NONE;
    if (dx) {
        const Lying lw = lying(w, d.N, d.K, d.w_stride, b.pack_w);
        a.w = lw.at;
        a.w_stride = lw.stride;
        a.x_outer = d.M;
        a.w_outer = lw.width;
        a.x_limit = lz.width;
        a.w_limit = d.N;
        a.y = dx;
        a.M = d.M;
        a.N = a.y_stride = d.K;
        if (int e = launch_16(a, b.dx, kWAcross, d.dtype, stream)) return launched(what, e);
    }
    if (dw) {
        if (d.kept_dtype == TDC_MX8) {
            if (int e = launch_mx8_dequantize(x, x_scales, d.M, d.K, scratch + b.x, d.dtype, round_up(d.K, 8), stream)) return launched(what, e);
            x = scratch + b.x;
        }
        const Lying lx = lying(x, d.M, d.K, d.x_stride, b.pack_x);
        a.w = lx.at;
        a.w_stride = lx.stride;
        a.x_outer = lz.width;
        a.w_outer = lx.width;
        a.x_limit = a.w_limit = d.M;
        a.y = dw;
        a.M = d.N;
        a.N = a.y_stride = d.K;
        if (int e = launch_16(a, b.dw, kAcross, d.dtype, stream)) return launched(what, e);
    }
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_mx8_sizes(int64_t rows, int64_t K, size_t *code_bytes, size_t *scale_bytes) TDC_ENTRY {
    if (int st = mx_range("8-bit numbers", rows, K)) return st;
    if (code_bytes) *code_bytes = (size_t)(rows * mx8_pitch(K));
    if (scale_bytes) *scale_bytes = (size_t)(rows * mx4_scale_bytes(K));
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_mx8_quantize(const void *x, int32_t dtype, int64_t rows, int64_t K, int64_t row_stride, void *codes, void *scales, void *stream) TDC_ENTRY {
    if (!number(dtype)) return invalid("8-bit numbers: dtype has to be TDC_F32, TDC_F16 or TDC_BF16");
    if (int st = mx_check("8-bit numbers", rows, K, codes, scales)) return st;
    if (!rows) return TDC_OK;
    if (!x) return invalid("8-bit numbers: null x");
    if (!row_stride) row_stride = K;
    if (rows > 1 && row_stride < K) return invalid("8-bit numbers: a row stride below K");
    return launched("8-bit numbers", launch_mx8_quantize(x, dtype, rows, K, row_stride, codes, scales, stream));
}
TDC_ENTRY_END

int tdc_mx8_dequantize(const void *codes, const void *scales, int64_t rows, int64_t K, void *y, int32_t dtype, int64_t row_stride,
                       void *stream) TDC_ENTRY {
    if (!number(dtype)) return invalid("8-bit numbers: dtype has to be TDC_F32, TDC_F16 or TDC_BF16");
    if (int st = mx_check("8-bit numbers", rows, K, codes, scales)) return st;
    if (!rows) return TDC_OK;
    if (!y) return invalid("8-bit numbers: null y");
    if (!row_stride) row_stride = K;
    if (rows > 1 && row_stride < K) return invalid("8-bit numbers: a row stride below K");
    return launched("8-bit numbers", launch_mx8_dequantize(codes, scales, rows, K, y, dtype, row_stride, stream));
}
TDC_ENTRY_END

int tdc_mx8_linear_workspace(const tdc_mx4_linear_desc *desc, size_t *bytes) TDC_ENTRY {
    tdc_mx4_linear_desc d;
    TilePlan p;
    if (int st = linear8_check(desc, d, p)) return st;
    if (!bytes) return invalid("8-bit product: null argument");
    *bytes = x8_bytes(d) + (size_t)p.part_bytes;
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_mx8_linear(const tdc_mx4_linear_desc *desc, const void *x, const void *x_scales, const void *w_codes, const void *w_scales,
                   const void *bias, const void *residual, void *y, void *ws, size_t ws_bytes, void *stream) TDC_ENTRY {
    tdc_mx4_linear_desc d;
    TilePlan p;
    if (int st = linear8_check(desc, d, p)) return st;
    if (!d.M || !d.N) return TDC_OK;
    if (!x || !y) return invalid("8-bit product: null x or y");
    if (int st = mx_check("8-bit product", d.N, d.K, w_codes, w_scales)) return st;
    if (d.x_dtype == TDC_MX8)
        if (int st = mx_check("8-bit product", d.M, d.K, x, x_scales)) return st;
    if (int st = ws_check("8-bit product", ws, ws_bytes, x8_bytes(d) + (size_t)p.part_bytes)) return st;
    TileArgs a{};
    if (d.x_dtype == TDC_MX8) {
        a.x = (const unsigned char *)x;
        a.x_scales = (const unsigned char *)x_scales;
    } else {
        a.x = (const unsigned char *)ws;
        a.x_scales = a.x + x8_codes(d);
        if (int e = launch_mx8_quantize(x, d.x_dtype, d.M, d.K, d.x_stride, ws, (char *)ws + x8_codes(d), stream))
            return launched("8-bit product", e);
    }
    a.w = (const unsigned char *)w_codes;
    a.w_scales = (const unsigned char *)w_scales;
    a.x_stride = a.w_stride = a.x_limit = a.w_limit = mx8_pitch(d.K);
    a.x_outer = a.M = d.M;
    a.w_outer = a.N = d.N;
    a.bias = bias;
    a.residual = residual;
    a.y = y;
    a.y_stride = d.y_stride;
    a.r_stride = d.residual_stride;
    a.bias_dtype = d.bias_dtype;
    a.act = d.act;
    a.part = (float *)((char *)ws + x8_bytes(d));
    return launched("8-bit product", launch_product_mx8(a, p, d.y_dtype, stream));
}
TDC_ENTRY_END

int tdc_rms_norm_workspace(const tdc_rms_norm_desc *desc, size_t *backward_bytes) TDC_ENTRY {
    tdc_rms_norm_desc d;
    if (int st = rms_check(desc, d)) return st;
    if (!backward_bytes) return invalid("RMS norm: null argument");
    RmsArgs a;
    if (int st = rms_args(d, nullptr, true, a)) return st;
    *backward_bytes = d.rows ? (size_t)a.blocks * d.C * 4 : 0;
    return TDC_OK;
}
TDC_ENTRY_END

int tdc_rms_norm_forward(const tdc_rms_norm_desc *desc, const void *x, const void *residual, const void *weight, void *y, void *h, float *rstd,
                         void *kept_codes, void *kept_scales, void *stream) TDC_ENTRY {
    tdc_rms_norm_desc d;
    if (int st = rms_check(desc, d)) return st;
    if (!d.rows) return TDC_OK;
    if (!x || !y) return invalid("RMS norm: null x or y");
    if (!residual != !h) return invalid("RMS norm: residual and h go together");
    if (!kept_codes != !kept_scales) return invalid("RMS norm: codes and scales go together");
    if (kept_codes)
        if (int st = mx_check("RMS norm", d.rows, d.C, kept_codes, kept_scales)) return st;
    RmsArgs a;
    if (int st = rms_args(d, weight, false, a)) return st;
    a.x = x;
    a.residual = residual;
    a.y = y;
    a.h = h;
    a.rstd = rstd;
    a.codes = (unsigned char *)kept_codes;
    a.scales = (unsigned char *)kept_scales;
    return launched("RMS norm", launch_rms_forward(a, d.dtype, kept_codes ? kRmsKeptMx8 : kRmsPlain, stream));
}
TDC_ENTRY_END

int tdc_rms_norm_forward_mx8(const tdc_rms_norm_desc *desc, const void *x, const void *residual, const void *weight, void *codes, void *scales,
                             void *h, void *stream) TDC_ENTRY {
    tdc_rms_norm_desc d;
    if (int st = rms_check(desc, d)) return st;
    if (!d.rows) return TDC_OK;
    if (!x) return invalid("RMS norm: null x");
    if (!residual != !h) return invalid("RMS norm: residual and h go together");
    if (int st = mx_check("RMS norm", d.rows, d.C, codes, scales)) return st;
    RmsArgs a;
    if (int st = rms_args(d, weight, false, a)) return st;
    a.x = x;
    a.residual = residual;
    a.h = h;
    a.codes = (unsigned char *)codes;
    a.scales = (unsigned char *)scales;
    return launched("RMS norm", launch_rms_forward(a, d.dtype, kRmsOutputMx8, stream));
}
TDC_ENTRY_END

int tdc_rms_norm_backward(const tdc_rms_norm_desc *desc, const void *h, const void *h_scales, const void *weight, const void *dy, const void *dh,
                          const float *rstd, void *dx, void *dweight, void *ws, size_t ws_bytes, void *stream) TDC_ENTRY {
    tdc_rms_norm_desc d;
    if (int st = rms_check(desc, d)) return st;
    if (!dx && !dweight) return TDC_OK;
    if (!d.rows) {
        if (!dweight) return TDC_OK;      // (a sum of nothing)
        return launched("RMS norm's gradient", launch_zeros(dweight, d.C, d.weight_dtype, stream));
    }
    if (!h || !dy || !rstd) return invalid("RMS norm's gradient: null h, dy or rstd");
    if (h_scales)
        if (int st = mx_check("RMS norm's gradient", d.rows, d.C, h, h_scales)) return st;
    RmsArgs a;
    if (int st = rms_args(d, weight, true, a)) return st;
    if (int st = ws_check("RMS norm's gradient", ws, ws_bytes, dweight ? (size_t)a.blocks * d.C * 4 : 0)) return st;
    if (h_scales) {
        a.codes = (unsigned char *)h;
        a.scales = (unsigned char *)h_scales;
    } else a.h = const_cast<void *>(h);
    a.dy = dy;
    a.dh = dh;
    a.rstd = const_cast<float *>(rstd);
    a.dx = dx;
    a.dweight = dweight;
    a.part = (float *)ws;
    return launched("RMS norm's gradient", launch_rms_backward(a, d.dtype, h_scales != nullptr, stream));
}
TDC_ENTRY_END

}  // extern "C"
