"""Channels-last operators: group norm with an activation, numbers in microscaled 4-bit floating point (MXFP4), and the
product of two such operands.

With a tensor's channels neighbours in memory a 1x1 (Tucker factor) convolution is a matrix product over its pixels, and
these are the operators that stand around it: ``group_norm_act`` (with its gradient) normalises what batch norm folding cannot,
``mx4_quantize`` / ``Mx4Tensor`` hold factors and activations in 4 bits with a power-of-two scale per block of 32 channels,
``mx4_linear`` / ``mx4_conv1x1`` multiply them on the matrix cores, and ``group_norm_act_mx4`` hands a normalised
tensor to such a product without writing it out in 16 bits.  All work is queued on the current stream of the
tensors' device; scratch comes from torch's allocator, call by call.
"""
from __future__ import annotations

import ctypes
import warnings
from ctypes import byref

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, lib
from .conv import _device, _raw_stream

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MX4 = 3
_ACTS = {"none": 0, "relu": 1, "silu": 2}
_empty, _empty_strided, _u8, _f32 = torch.empty, torch.empty_strided, torch.uint8, torch.float32
_calls = {}


def _call(name):
    """The library's entry point of that name (looked up once)."""
    fn = _calls.get(name)
    if fn is None:
        fn = _calls[name] = getattr(lib(), name)
    return fn


def _act(name):
    try:
        return _ACTS[name]
    except (KeyError, TypeError):
        raise ValueError(f"act has to be one of {', '.join(_ACTS)}: got {name!r}") from None


def _number_tensor(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} has to be a tensor: got {type(t).__name__}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{what} has to be float32, float16 or bfloat16: got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a device tensor")


def _vector(t, n, dtype, device, what):
    """A parameter vector (or None): [n], float32 or the tensor's type."""
    if t is None:
        return
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise ValueError(f"{what} must be a tensor on {device}")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected ({n},)")
    if t.dtype != torch.float32 and t.dtype != dtype:
        raise TypeError(f"{what} has to be float32 or {dtype}: got {t.dtype}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{what} must be contiguous")


def _wants(t):
    """Whether a gradient would have to reach t."""
    return t is not None and getattr(t, "requires_grad", False) and torch.is_grad_enabled()


def _no_tangent(what, *tensors):
    """Refuses dual tensors of forward mode: they need not require a gradient, and their tangents would be lost."""
    if getattr(forward_ad, "_current_level", 0) < 0:      # (no level is open: the usual call)
        return
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no derivative in forward mode")


def _no_gradient(what, name):
    raise RuntimeError(f"{what} has no gradient, and {name} requires one: call it under torch.no_grad(), or on {name}.detach()")


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Cache(dict):
    """What a shape's calls have in common (descriptor, sizes): no data, and a bounded number of shapes."""
    MOST = 512

    def keep(self, key, value):
        if len(self) >= self.MOST:
            self.clear()
        self[key] = value
        return value


# ---- group norm ---------------------------------------------------------------------------------------------------------

def _pixel_strides(shape, stride):
    """(pixels, pixel stride, image stride) of a channels-last [B, C, ...] tensor, or None if it is none."""
    B, C = shape[0], shape[1]
    pixels, step, run = 1, None, None
    for n, s in zip(reversed(shape[2:]), reversed(stride[2:])):
        pixels *= n
        if n <= 1:
            continue
        if step is None:
            step = s
        elif s != run:
            return None
        run = s * n
    if pixels == 0 or B == 0:
        return pixels, C, pixels * C
    if (C > 1 and stride[1] != 1) or (step is not None and step < C):
        return None
    step = C if step is None else step
    image = stride[0] if B > 1 else pixels * step
    if image < (pixels - 1) * step + C:
        return None
    return pixels, step, image


def _dense_strides(shape):
    """Channels-last strides of [B, C, ...]."""
    strides, run = [], shape[1]
    for n in reversed(shape[2:]):
        strides.append(run)
        run *= n
    return (run, 1, *reversed(strides))


class _Norm:
    """A norm's descriptor and sizes, for one shape of x (and of y or dy)."""
    __slots__ = ("desc", "ref", "forward_ws", "backward_ws", "mx4_ws", "y_strides", "stats_shape", "stats_bytes", "mx4_shape", "dense")

    def __init__(self, x_shape, x_stride, y_stride, dtype, param_dtype, groups, eps, act):
        x = _pixel_strides(x_shape, x_stride)
        if x is None:
            raise ValueError("x has to be channels last, the channels of a pixel neighbours in memory and its pixels evenly spaced: "
                             "x.contiguous(memory_format=torch.channels_last)")
        self.y_strides = _dense_strides(x_shape)
        y = _pixel_strides(x_shape, y_stride) if y_stride is not None else (x[0], x_shape[1], x[0] * x_shape[1])
        self.dense = y is None      # dy in another order: copied first
        y = y or (x[0], x_shape[1], x[0] * x_shape[1])
        self.desc = _lib.GroupNormDesc(x_shape[0], x_shape[1], groups, act, _DTYPES[dtype], _DTYPES[param_dtype], eps, 0,
                                       x[0], x[1], x[2], y[1], y[2])
        self.ref = byref(self.desc)
        fwd, bwd, mx4 = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
        check(lib().tdc_group_norm_workspace(self.ref, byref(fwd), byref(bwd)))
        check(lib().tdc_group_norm_mx4_workspace(self.ref, byref(mx4)))
        self.forward_ws, self.backward_ws, self.mx4_ws = fwd.value, bwd.value, mx4.value
        self.stats_shape = (2, x_shape[0], groups)
        self.stats_bytes = 4 * x_shape[0] * groups
        self.mx4_shape = (x_shape[0], *x_shape[2:], x_shape[1])


_norms = _Cache()


def _norm_for(x, groups, weight, bias, eps, act, y_stride=None):
    given = weight if weight is not None else bias
    wd = getattr(given, "dtype", None)
    key = (x.shape, x.stride(), y_stride, x.dtype, x.device, wd, weight is None, bias is None, groups, eps, act)
    plan = _norms.get(key)
    if plan is None:
        _number_tensor(x, "x")
        if x.dim() < 2:
            raise ValueError(f"expected x [batch, channels, ...], got {tuple(x.shape)}")
        C = x.shape[1]
        if isinstance(groups, bool) or not isinstance(groups, int) or groups < 1 or C % groups:
            raise ValueError(f"groups has to be a whole number that divides the {C} channels: got {groups!r}")
        _vector(weight, C, x.dtype, x.device, "weight")
        _vector(bias, C, x.dtype, x.device, "bias")
        plan = _norms.keep(key, _Norm(tuple(x.shape), x.stride(), y_stride, x.dtype, wd or torch.float32, groups, float(eps), _act(act)))
    if weight is not None or bias is not None:
        for t, what in ((weight, "weight"), (bias, "bias")):
            if t is not None and (getattr(t, "dtype", None) != wd or wd is None or t.dim() != 1 or t.shape[0] != x.shape[1] or t.device != x.device or not t.is_contiguous()):
                _vector(t, x.shape[1], x.dtype, x.device, what)
                raise TypeError("weight and bias have to be of one type")
        if wd != torch.float32 and wd != x.dtype:
            raise TypeError(f"weight and bias have to be float32 or {x.dtype}: got {wd}")
    return plan


def _norm_forward(x, groups, weight, bias, eps, act, stats):
    plan = _norm_for(x, groups, weight, bias, eps, act)
    dev = x.device
    y = _empty_strided(x.shape, plan.y_strides, dtype=x.dtype, device=dev)
    need = plan.forward_ws
    ws = _empty(need, dtype=_u8, device=dev) if need else None
    kept = mean = rstd = None
    if stats:
        kept = _empty(plan.stats_shape, dtype=_f32, device=dev)
        mean = kept.data_ptr()
        rstd = mean + plan.stats_bytes if mean else None
    status = _call("tdc_group_norm_forward")(plan.ref, x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), mean, rstd, _ptr(ws), need,
                                             _raw_stream(x.get_device()))
    if status:
        check(status)
    return y, kept


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, stats = _norm_forward(x, groups, weight, bias, eps, act, True)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.how = (groups, eps, act)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        _no_tangent("the gradient of group_norm_act", dy)
        groups, eps, act = ctx.how
        plan = _norm_for(x, groups, weight, bias, eps, act, dy.stride())
        dev, C = x.device, x.shape[1]
        if plan.dense:
            dy = _empty_strided(x.shape, plan.y_strides, dtype=x.dtype, device=dev).copy_(dy)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = _empty_strided(x.shape, plan.y_strides, dtype=x.dtype, device=dev) if need_x else None
        dw = _empty(C, dtype=_f32, device=dev) if need_w else None
        db = _empty(C, dtype=_f32, device=dev) if need_b else None
        ws = _empty(plan.backward_ws, dtype=_u8, device=dev)
        mean = stats.data_ptr()
        status = _call("tdc_group_norm_backward")(plan.ref, x.data_ptr(), dy.data_ptr(), _ptr(weight), _ptr(bias), mean,
                                                  mean + plan.stats_bytes, _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(),
                                                  plan.backward_ws, _raw_stream(x.get_device()))
        if status:
            check(status)
        if need_w and weight.dtype != _f32:
            dw = dw.to(weight.dtype)
        if need_b and bias.dtype != _f32:
            db = db.to(bias.dtype)
        return dx, dw, db, None, None, None


def _on(t, call, *args):
    """`call` with the tensor's device as the current one."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() != _device():
        with torch.cuda.device(t.device):
            return call(*args)
    return call(*args)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="none"):
    """``act(group_norm(x, groups) * weight + bias)`` for a channels-last ``x`` [batch, channels, ...].

    Mean and variance are those of one image and group of channels, in 32 bits; ``act`` is "none", "relu" or "silu".  ``x``
    may be float32, float16 or bfloat16 and a channel slice of a wider tensor; ``weight`` and ``bias`` [channels] float32 or
    of x's type.  The result is dense channels last, of x's type.  Differentiable once, backwards, in x, weight and bias."""
    _no_tangent("group_norm_act", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or getattr(weight, "requires_grad", False) or getattr(bias, "requires_grad", False)):
        return _on(x, _GroupNormAct.apply, x, weight, bias, groups, eps, act)
    return _on(x, _norm_forward, x, groups, weight, bias, eps, act, False)[0]


# ---- 4-bit numbers --------------------------------------------------------------------------------------------------------

class Mx4Tensor:
    """Numbers in microscaled 4-bit floating point, in blocks of 32 along the last axis.

    ``shape`` is that of the numbers, ``codes`` [ceil(K / 128), ceil(rows / 32), 4, 32, 16] and ``scales``
    [ceil(K / 512), rows, 16] are bytes (the layout is that of include/tdc.h)."""
    __slots__ = ("shape", "rows", "K", "device", "index", "_held", "_codes_at", "_scales_at")

    def __init__(self, codes, scales, shape):
        shape = tuple(int(n) for n in shape)
        if not shape or shape[-1] < 1:
            raise ValueError(f"the last axis has to hold a number at least: got {shape}")
        self.shape, self.K, self.rows = shape, shape[-1], _product(shape[:-1])
        for t, want, what in zip((codes, scales), self._byte_shapes(), ("codes", "scales")):
            if t.dtype != _u8 or tuple(t.shape) != want or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"{what} has to be a contiguous uint8 device tensor of shape {want}")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on one device")
        self.device, self.index, self._held = codes.device, codes.get_device(), (codes, scales)
        self._codes_at, self._scales_at = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _new(cls, rows, K, shape, device, index):
        t = cls.__new__(cls)
        codes = (K + 127) // 128 * ((rows + 31) // 32) * 2048
        t._held = _empty(codes + (K + 511) // 512 * rows * 16, dtype=_u8, device=device)
        t._codes_at = t._held.data_ptr()
        t._scales_at = t._codes_at + codes
        t.shape, t.rows, t.K, t.device, t.index = shape, rows, K, device, index
        return t

    def __reduce__(self):
        # (a copy, also one from a file, finds its addresses anew)
        return _mx4_again, (self.codes, self.scales, self.shape)

    def _byte_shapes(self):
        return ((self.K + 127) // 128, (self.rows + 31) // 32, 4, 32, 16), ((self.K + 511) // 512, self.rows, 16)

    def _bytes(self, which):
        if type(self._held) is tuple:
            return self._held[which]
        shapes = self._byte_shapes()
        split = _product(shapes[0])
        return (self._held[split:] if which else self._held[:split]).view(shapes[which])

    @property
    def codes(self):
        return self._bytes(0)

    @property
    def scales(self):
        return self._bytes(1)

    def dequantize(self, dtype=torch.float32):
        """The numbers that the codes and scales stand for (each is exact in float32 and bfloat16)."""
        kind = _DTYPES.get(dtype)
        if kind is None:
            raise TypeError(f"dtype has to be float32, float16 or bfloat16: got {dtype}")
        if self.index != _device():
            with torch.cuda.device(self.device):
                return self.dequantize(dtype)
        y = _empty(self.shape, dtype=dtype, device=self.device)
        status = _call("tdc_mx4_dequantize")(self._codes_at, self._scales_at, self.rows, self.K, y.data_ptr(), kind, self.K,
                                             _raw_stream(self.index))
        if status:
            check(status)
        return y

    def __repr__(self):
        return f"Mx4Tensor(shape={self.shape}, device={self.device})"


def _mx4_again(codes, scales, shape):
    t = Mx4Tensor.__new__(Mx4Tensor)
    t.shape, t.K, t.rows = shape, shape[-1], _product(shape[:-1])
    t.device, t.index, t._held = codes.device, codes.get_device(), (codes, scales)
    t._codes_at, t._scales_at = codes.data_ptr(), scales.data_ptr()
    return t


def _product(shape):
    n = 1
    for k in shape:
        n *= k
    return n


def _rows(t):
    """t as evenly spaced rows of neighbouring numbers (copied if it is not), and the distance between rows."""
    K = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(_product(t.shape[:-1]), K)
    step = t.stride(0) if t.shape[0] > 1 else K
    if (K > 1 and t.stride(1) != 1) or step < K:
        t = t.contiguous()
        step = K
    return t, step


def _quantize(x):
    flat, step = _rows(x)
    index = x.get_device()
    q = Mx4Tensor._new(flat.shape[0], flat.shape[1], tuple(x.shape), x.device, index)
    status = _call("tdc_mx4_quantize")(flat.data_ptr(), _DTYPES[x.dtype], q.rows, q.K, step, q._codes_at, q._scales_at, _raw_stream(index))
    if status:
        check(status)
    return q


def mx4_quantize(x):
    """``x`` [..., K] in microscaled 4-bit floating point: each block of 32 along the last axis is scaled by the power of two that
    takes its largest magnitude into [4, 8) and rounded to nearest (halfway to the even code, saturating at 6).  A block with
    an infinity or a NaN stands for NaNs.  Has no gradient: weights that train are put into 4 bits under ``torch.no_grad()``."""
    _number_tensor(x, "x")
    _no_tangent("mx4_quantize", x)
    if _wants(x):
        _no_gradient("mx4_quantize", "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected x [..., K] with K at least 1, got {tuple(x.shape)}")
    return _on(x, _quantize, x)


def group_norm_act_mx4(x, groups, weight=None, bias=None, eps=1e-5, act="none"):
    """``group_norm_act`` with its result in 4 bits, quantised from the 32-bit values: an ``Mx4Tensor`` of shape
    [batch, ..., channels] for ``mx4_conv1x1``.  Has no gradient: an ``x`` that requires one is refused, ``weight`` and ``bias`` that
    do are taken as they are, with a warning."""
    _no_tangent("group_norm_act_mx4", x, weight, bias)
    if _wants(x):
        raise RuntimeError("group_norm_act_mx4 has no gradient: call it under torch.no_grad(), or use group_norm_act")
    if _wants(weight) or _wants(bias):
        warnings.warn("group_norm_act_mx4 has no gradient: weight and bias get none from it (torch.no_grad() says that this is meant)", stacklevel=2)
    return _on(x, _norm_mx4, x, groups, weight, bias, eps, act)


def _norm_mx4(x, groups, weight, bias, eps, act):
    plan = _norm_for(x, groups, weight, bias, eps, act)
    d, index, need = plan.desc, x.get_device(), plan.mx4_ws
    q = Mx4Tensor._new(d.batch * d.pixels, d.C, plan.mx4_shape, x.device, index)
    ws = _empty(need, dtype=_u8, device=x.device) if need else None
    status = _call("tdc_group_norm_forward_mx4")(plan.ref, x.data_ptr(), _ptr(weight), _ptr(bias), q._codes_at, q._scales_at, _ptr(ws), need,
                                                 _raw_stream(index))
    if status:
        check(status)
    return q


# ---- product ----------------------------------------------------------------------------------------------------------------

_linears = _Cache()


def _linear(x, weight, bias, residual, act, out_dtype, pixels):
    """``pixels``: x [B, H, W, K] stands for a channels-last [B, K, H, W], as the result [B, N, H, W] does."""
    if type(weight) is not Mx4Tensor or len(weight.shape) != 2:
        raise TypeError("weight has to be an Mx4Tensor of shape [N, K]: mx4_quantize(weight)")
    index, dev, N = weight.index, weight.device, weight.rows
    quantised = type(x) is Mx4Tensor
    if not quantised:
        _number_tensor(x, "x")
        if _wants(x):
            _no_gradient("the 4-bit product", "x")
        if x.dim() < 1:
            raise ValueError("expected x [..., K]")
    _no_tangent("the 4-bit product", x, bias, residual)
    if _wants(bias):
        _no_gradient("the 4-bit product", "bias")
    if _wants(residual):
        _no_gradient("the 4-bit product", "residual")
    shape = x.shape
    if shape[-1] != weight.K:
        raise ValueError(f"x has {shape[-1]} numbers a row, weight {weight.K}")
    if x.device != dev:
        raise ValueError(f"x is on {x.device}, weight on {dev}")
    if index != _device():
        with torch.cuda.device(dev):
            return _linear(x, weight, bias, residual, act, out_dtype, pixels)
    if quantised:
        M, dtype, x_type, x_step = x.rows, out_dtype or torch.bfloat16, _MX4, 0
        x_at, x_scales = x._codes_at, x._scales_at
    else:
        flat, x_step = _rows(x)
        M, dtype, x_type = flat.shape[0], out_dtype or x.dtype, _DTYPES[x.dtype]
        x_at, x_scales = flat.data_ptr(), None
    r_step, r_at, bias_type, b_at = 0, None, _f32, None
    if residual is not None:
        if residual.dtype != dtype or residual.device != dev or residual.shape != (*shape[:-1], N):
            raise ValueError(f"residual has to be {dtype} of shape {(*shape[:-1], N)} on {dev}: got {residual.dtype} "
                             f"{tuple(residual.shape)} on {residual.device}")
        residual, r_step = _rows(residual)
        r_at = residual.data_ptr()
    if bias is not None:
        _vector(bias, N, dtype, dev, "bias")
        bias_type, b_at = bias.dtype, bias.data_ptr()
    key = (M, N, weight.K, x_type, dtype, bias_type, act, x_step, r_step)
    plan = _linears.get(key)
    if plan is None:
        if dtype not in _DTYPES:
            raise TypeError(f"out_dtype has to be float32, float16 or bfloat16: got {dtype}")
        desc = _lib.Mx4LinearDesc(M, N, weight.K, x_type, _DTYPES[dtype], _DTYPES[bias_type], _act(act), x_step, N, r_step)
        need = ctypes.c_size_t()
        check(lib().tdc_mx4_linear_workspace(byref(desc), byref(need)))
        plan = _linears.keep(key, (byref(desc), need.value))
    ref, need = plan
    if pixels:
        B, H, W = shape[:3]
        y = _empty_strided((B, N, H, W), (H * W * N, 1, W * N, N), dtype=dtype, device=dev)
    else:
        y = _empty((*shape[:-1], N), dtype=dtype, device=dev)
    ws = _empty(need, dtype=_u8, device=dev) if need else None
    status = _call("tdc_mx4_linear")(ref, x_at, x_scales, weight._codes_at, weight._scales_at, b_at, r_at, y.data_ptr(), _ptr(ws), need,
                                     _raw_stream(index))
    if status:
        check(status)
    return y


def mx4_linear(x, weight, bias=None, residual=None, act="none", out_dtype=None):
    """``act(x @ weight.T + bias + residual)`` with both operands in 4 bits, products and sums in 32.

    ``weight`` is an ``Mx4Tensor`` [N, K]; ``x`` [..., K] is numbers (float32, float16, bfloat16), quantised on the way, or an
    ``Mx4Tensor``.  ``out_dtype`` is x's type unless given (bfloat16 for an Mx4Tensor); ``residual`` [..., N] is of that type,
    ``bias`` [N] of it or float32.  Has no gradient: an ``x``, ``bias`` or ``residual`` that requires one is refused."""
    return _linear(x, weight, bias, residual, act, out_dtype, False)


def mx4_conv1x1(x, weight, bias=None, residual=None, act="none", out_dtype=None):
    """``mx4_linear`` over the pixels of a channels-last tensor: ``x`` [batch, C, H, W] (or an Mx4Tensor [batch, H, W, C], as
    ``group_norm_act_mx4`` gives it), ``weight`` an Mx4Tensor [N, C], ``residual`` [batch, N, H, W]; the result is channels
    last [batch, N, H, W]."""
    if type(x) is not Mx4Tensor:
        _number_tensor(x, "x")
        if x.dim() != 4:
            raise ValueError(f"expected x [batch, channels, height, width], got {tuple(x.shape)}")
        x = x.permute(0, 2, 3, 1)
    elif len(x.shape) != 4:
        raise ValueError(f"expected x [batch, height, width, channels] in 4 bits, got {x.shape}")
    if residual is not None:
        if residual.dim() != 4:
            raise ValueError(f"expected residual [batch, channels, height, width], got {tuple(residual.shape)}")
        residual = residual.permute(0, 2, 3, 1)
    return _linear(x, weight, bias, residual, act, out_dtype, True)
