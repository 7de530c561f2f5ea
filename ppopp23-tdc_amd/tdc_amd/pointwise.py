"""Operators around a 1x1 (Tucker factor) convolution in 16 and 8 bits, over rows of numbers: the pixels of a channels-last tensor,
or tokens.

``linear_act`` / ``conv1x1_act`` are the factor's product with bias, residual and activation in one pass, with its gradients;
``rms_norm`` normalises rows and takes the residual's addition along, with its gradients.  Both can keep what their gradient needs of
their input in microscaled 8-bit floating point (``checkpoint="mx8"``: 33/32 byte a number).  For inference
``mx8_quantize`` / ``Mx8Tensor`` hold numbers in that format, ``rms_norm_mx8`` hands a normalised tensor on in it, and ``mx8_linear``
/ ``mx8_conv1x1`` multiply two such operands on the matrix cores.  All work is queued on the current stream of the tensors' device;
scratch comes from torch's allocator, call by call.

Small training steps are the host's: most of one is handing the backward pass to autograd's thread and back.  A program with one device
can keep it on the calling thread, ``with torch.autograd.set_multithreading_enabled(False)`` around ``backward()``: 41 us in place of 103
for a norm of 663 x 1001 and its gradient, 63 in place of 135 for a product of 33 x 2001 by 1001.
"""
from __future__ import annotations

import ctypes
import warnings
from ctypes import byref

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, lib
from .channels_last import (_act, _Cache, _call, _DTYPES, _no_gradient, _no_tangent, _number_tensor, _on, _product, _ptr, _rows,
                            _vector, _wants)
from .conv import _device, _raw_stream

_MX8 = 4
_empty, _empty_like, _u8, _f32 = torch.empty, torch.empty_like, torch.uint8, torch.float32


def _checkpoint(how):
    if how is not None and how != "mx8":
        raise ValueError(f"checkpoint has to be None or 'mx8': got {how!r}")
    return how is not None


def _flat(t):
    """t as evenly spaced rows of neighbouring numbers: (what holds them, rows, distance between rows)."""
    K = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // K if K else _product(t.shape[:-1]), K
    t, step = _rows(t)
    return t, t.shape[0], step


def _like(t):
    """A dense tensor like t."""
    return _empty_like(t) if t.is_contiguous() else _empty(t.shape, dtype=t.dtype, device=t.device)


def _tile_rows(t):
    """`_flat` at an address that 16-byte requests can start from."""
    t, rows, step = _flat(t)
    if t.data_ptr() & 15:
        step = t.shape[-1]
        t = t.clone(memory_format=torch.contiguous_format)
    return t, rows, step


def _once(body):
    """A backward that refuses to be differentiated itself.  (The wrapper that does costs some microseconds: not where no graph is made.)"""
    refusing = once_differentiable(body)

    def backward(ctx, *grads):
        return refusing(ctx, *grads) if torch.is_grad_enabled() else body(ctx, *grads)
    return backward


# ---- 8-bit numbers --------------------------------------------------------------------------------------------------------

class Mx8Tensor:
    """Numbers in microscaled 8-bit floating point (E4M3), in blocks of 32 along the last axis.

    ``shape`` is that of the numbers, ``codes`` [rows, K rounded up to 128] and ``scales`` [ceil(K / 512), rows, 16] are bytes (the
    layout is that of include/tdc.h)."""
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
        return cls._of(_empty(rows * ((K + 127) // 128 * 128 + (K + 511) // 512 * 16), dtype=_u8, device=device), rows, K, shape, device, index)

    @classmethod
    def _of(cls, held, rows, K, shape, device, index):
        t = cls.__new__(cls)
        t._held = held
        t._codes_at = held.data_ptr()
        t._scales_at = t._codes_at + rows * ((K + 127) // 128 * 128)
        t.shape, t.rows, t.K, t.device, t.index = shape, rows, K, device, index
        return t

    def __reduce__(self):
        # (a copy, also one from a file, finds its addresses anew)
        return _mx8_again, (self.codes, self.scales, self.shape)

    def _byte_shapes(self):
        return (self.rows, (self.K + 127) // 128 * 128), ((self.K + 511) // 512, self.rows, 16)

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
        status = _call("tdc_mx8_dequantize")(self._codes_at, self._scales_at, self.rows, self.K, y.data_ptr(), kind, self.K,
                                             _raw_stream(self.index))
        if status:
            check(status)
        return y

    def __repr__(self):
        return f"Mx8Tensor(shape={self.shape}, device={self.device})"


def _mx8_again(codes, scales, shape):
    t = Mx8Tensor.__new__(Mx8Tensor)
    t.shape, t.K, t.rows = shape, shape[-1], _product(shape[:-1])
    t.device, t.index, t._held = codes.device, codes.get_device(), (codes, scales)
    t._codes_at, t._scales_at = codes.data_ptr(), scales.data_ptr()
    return t


def _quantize(x):
    flat, rows, step = _flat(x)
    index = x.get_device()
    q = Mx8Tensor._new(rows, x.shape[-1], tuple(x.shape), x.device, index)
    status = _call("tdc_mx8_quantize")(flat.data_ptr(), _DTYPES[x.dtype], q.rows, q.K, step, q._codes_at, q._scales_at, _raw_stream(index))
    if status:
        check(status)
    return q


def mx8_quantize(x):
    """``x`` [..., K] in microscaled 8-bit floating point: each block of 32 along the last axis is scaled by the power of two that
    takes its largest magnitude into [256, 512) and rounded to nearest in E4M3 (halfway to the even code, saturating at 448).  A
    block with an infinity or a NaN stands for NaNs.  Has no gradient: weights that train are put into 8 bits under
    ``torch.no_grad()``."""
    _number_tensor(x, "x")
    _no_tangent("mx8_quantize", x)
    if _wants(x):
        _no_gradient("mx8_quantize", "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected x [..., K] with K at least 1, got {tuple(x.shape)}")
    return _on(x, _quantize, x)


# ---- product of 8-bit numbers ---------------------------------------------------------------------------------------------

_plans8 = _Cache()


def _pixels_out(shape, N, dtype, device):
    """A result [..., N], or for pixels' [B, H, W] the channels-last [B, N, H, W]."""
    B, H, W = shape[:3]
    return torch.empty_strided((B, N, H, W), (H * W * N, 1, W * N, N), dtype=dtype, device=device)


def _residual(t, shape, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or tuple(t.shape) != shape:
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"residual has to be {dtype} of shape {shape} on {device}: got {got}")


def _mx8_linear(x, weight, bias, residual, act, out_dtype, pixels):
    if type(weight) is not Mx8Tensor or len(weight.shape) != 2:
        raise TypeError("weight has to be an Mx8Tensor of shape [N, K]: mx8_quantize(weight)")
    index, dev, N = weight.index, weight.device, weight.rows
    quantised = type(x) is Mx8Tensor
    if not quantised:
        _number_tensor(x, "x")
        if x.dim() < 1:
            raise ValueError("expected x [..., K]")
    _no_tangent("the 8-bit product", x, bias, residual)
    for t, name in ((x, "x"), (bias, "bias"), (residual, "residual")):
        if not (quantised and t is x) and _wants(t):
            _no_gradient("the 8-bit product", name)
    shape = tuple(x.shape)
    if shape[-1] != weight.K:
        raise ValueError(f"x has {shape[-1]} numbers a row, weight {weight.K}")
    if x.device != dev:
        raise ValueError(f"x is on {x.device}, weight on {dev}")
    if index != _device():
        with torch.cuda.device(dev):
            return _mx8_linear(x, weight, bias, residual, act, out_dtype, pixels)
    if quantised:
        M, dtype, x_type, x_step = x.rows, out_dtype or torch.bfloat16, _MX8, 0
        x_at, x_scales = x._codes_at, x._scales_at
    else:
        flat, M, x_step = _flat(x)
        dtype, x_type = out_dtype or x.dtype, _DTYPES[x.dtype]
        x_at, x_scales = flat.data_ptr(), None
    if dtype != torch.float16 and dtype != torch.bfloat16:
        raise TypeError(f"the 8-bit product's result is float16 or bfloat16 (out_dtype): got {dtype}")
    r_step, r_at, bias_type, b_at = 0, None, _f32, None
    if residual is not None:
        _residual(residual, (*shape[:-1], N), dtype, dev)
        residual, _, r_step = _flat(residual)
        r_at = residual.data_ptr()
    if bias is not None:
        _vector(bias, N, dtype, dev, "bias")
        bias_type, b_at = bias.dtype, bias.data_ptr()
    key = (M, N, weight.K, x_type, dtype, bias_type, act, x_step, r_step)
    plan = _plans8.get(key)
    if plan is None:
        desc = _lib.Mx4LinearDesc(M, N, weight.K, x_type, _DTYPES[dtype], _DTYPES[bias_type], _act(act), x_step, N, r_step)
        need = ctypes.c_size_t()
        check(lib().tdc_mx8_linear_workspace(byref(desc), byref(need)))
        plan = _plans8.keep(key, (byref(desc), need.value))
    ref, need = plan
    y = _pixels_out(shape, N, dtype, dev) if pixels else _empty((*shape[:-1], N), dtype=dtype, device=dev)
    ws = _empty(need, dtype=_u8, device=dev) if need else None
    status = _call("tdc_mx8_linear")(ref, x_at, x_scales, weight._codes_at, weight._scales_at, b_at, r_at, y.data_ptr(), _ptr(ws), need,
                                     _raw_stream(index))
    if status:
        check(status)
    return y


def mx8_linear(x, weight, bias=None, residual=None, act="none", out_dtype=None):
    """``act(x @ weight.T + bias + residual)`` with both operands in 8 bits and sums in 32.

    ``weight`` is an ``Mx8Tensor`` [N, K]; ``x`` [..., K] is numbers (float32, float16, bfloat16), quantised on the way, or an
    ``Mx8Tensor``.  The result is float16 or bfloat16: ``out_dtype``, else x's type (bfloat16 for an Mx8Tensor).  ``residual``
    [..., N] is of that type, ``bias`` [N] of it or float32.  Has no gradient: an ``x``, ``bias`` or ``residual`` that requires one is
    refused."""
    return _mx8_linear(x, weight, bias, residual, act, out_dtype, False)


def _images(x, what):
    _number_tensor(x, what)
    if x.dim() != 4:
        raise ValueError(f"expected {what} [batch, channels, height, width], got {tuple(x.shape)}")
    return x.permute(0, 2, 3, 1)


def mx8_conv1x1(x, weight, bias=None, residual=None, act="none", out_dtype=None):
    """``mx8_linear`` over the pixels of a channels-last tensor: ``x`` [batch, C, H, W] (or an Mx8Tensor [batch, H, W, C]), ``weight`` an
    Mx8Tensor [N, C], ``residual`` [batch, N, H, W]; the result is channels last [batch, N, H, W]."""
    if type(x) is not Mx8Tensor:
        x = _images(x, "x")
    elif len(x.shape) != 4:
        raise ValueError(f"expected x [batch, height, width, channels] in 8 bits, got {x.shape}")
    if residual is not None:
        residual = _images(residual, "residual")
    return _mx8_linear(x, weight, bias, residual, act, out_dtype, True)


# ---- product in 16 bits -----------------------------------------------------------------------------------------------------

_plans = _Cache()


def _linear_plan(M, N, K, dtype, bias_dtype, act, kept8, x_step, w_step, y_step, r_step, backward, dz_given=False):
    key = (M, N, K, dtype, bias_dtype, act, kept8, x_step, w_step, y_step, r_step, backward, dz_given)
    plan = _plans.get(key)
    if plan is None:
        kind = _DTYPES[dtype]
        desc = _lib.LinearDesc(M, N, K, kind, _DTYPES[bias_dtype], _act(act), _MX8 if kept8 else kind, x_step, w_step, y_step, r_step)
        need = ctypes.c_size_t()
        if backward:
            check(lib().tdc_linear_backward_workspace(byref(desc), dz_given, byref(need)))
        else:
            check(lib().tdc_linear_workspace(byref(desc), byref(need), None))
        plan = _plans.keep(key, (byref(desc), need.value))
    return plan


def _linear_forward(x, weight, bias, residual, act, want_z):
    """(y, z): rows [M, K] and so on, on the current device."""
    dev, dtype, N = x.device, x.dtype, weight.shape[0]
    flat, M, x_step = _tile_rows(x)
    w, _, w_step = _tile_rows(weight)
    K, r_step, r_at = weight.shape[1], 0, None
    if residual is not None:
        r, _, r_step = _flat(residual)
        r_at = r.data_ptr()
    ref, need = _linear_plan(M, N, K, dtype, _f32 if bias is None else bias.dtype, act, False, x_step, w_step, 0, r_step, False)
    y = _empty((*x.shape[:-1], N), dtype=dtype, device=dev)
    z = _empty((M, N), dtype=dtype, device=dev) if want_z else None
    ws = _empty(need, dtype=_u8, device=dev) if need else None
    status = _call("tdc_linear_forward")(ref, flat.data_ptr(), w.data_ptr(), _ptr(bias), r_at, y.data_ptr(), _ptr(z), _ptr(ws), need,
                                         _raw_stream(x.get_device()))
    if status:
        check(status)
    return y, z


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, kept8):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        y, z = _linear_forward(x, weight, bias, residual, act, act == "silu")
        ctx.how = (act, kept8 and need_w, tuple(x.shape), bias.dtype if bias is not None else _f32)
        held = None
        if need_w:
            held = _quantize(x)._held if kept8 else x
        # (x and weight each for the other's gradient; of the activation what its slope is taken at)
        ctx.save_for_backward(held, weight if need_x else None, y if act == "relu" else z)
        ctx.sizes = (weight.shape[0], weight.shape[1])
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        held, weight, kept = ctx.saved_tensors
        _no_tangent("the gradient of linear_act", dy)
        act, kept8, shape, bias_dtype = ctx.how
        (N, K), dev, dtype, index = ctx.sizes, dy.device, dy.dtype, dy.get_device()
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = _empty(shape, dtype=dtype, device=dev) if need_x else None
        dw = _empty((N, K), dtype=dtype, device=dev) if need_w else None
        db = _empty(N, dtype=bias_dtype, device=dev) if need_b else None
        flat, M, y_step = _tile_rows(dy)
        dz, dr = None, None
        if need_r:
            if act == "none":
                dr = dy
            else:
                wide = (N + 7) // 8 * 8
                dz = _empty((M, wide), dtype=dtype, device=dev)
                dr = dz.view(dy.shape) if wide == N else dz.as_strided(dy.shape, (*_leading(dy.shape, wide), 1))
        if need_x or need_w or need_b or dz is not None:
            x, x_step, x_at, x_scales = None, 0, None, None
            if need_w and kept8:
                q = Mx8Tensor._of(held, M, K, shape, dev, index)
                x_at, x_scales = q._codes_at, q._scales_at
            elif need_w:
                x, _, x_step = _tile_rows(held)
                x_at = x.data_ptr()
            w, _, w_step = _tile_rows(weight) if need_x else (None, 0, 0)
            ref, need = _linear_plan(M, N, K, dtype, bias_dtype, act, kept8, x_step, w_step, y_step, 0, True, dz is not None)
            ws = _empty(need, dtype=_u8, device=dev) if need else None
            status = _call("tdc_linear_backward")(ref, x_at, x_scales, _ptr(w), _ptr(kept), flat.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db),
                                                  _ptr(dz), _ptr(ws), need, _raw_stream(index))
            if status:
                check(status)
        return dx, dw, db, dr, None, None


def _leading(shape, run):
    """Strides of all axes but the last, of rows `run` apart."""
    strides = []
    for n in reversed(shape[:-1]):
        strides.append(run)
        run *= n
    return tuple(reversed(strides))


def _linear_act(x, weight, bias, residual, act, checkpoint):
    _number_tensor(x, "x")
    if x.dtype == _f32:
        raise TypeError("linear_act takes float16 and bfloat16 (32-bit 1x1 factors: Conv2dPlan, TKConv2dC)")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.dtype != x.dtype or weight.device != x.device:
        got = f"{weight.dtype} {tuple(weight.shape)} on {weight.device}" if isinstance(weight, torch.Tensor) else type(weight).__name__
        raise ValueError(f"weight has to be {x.dtype} of shape (N, K) on {x.device}: got {got}")
    N, K = weight.shape
    if x.dim() < 1 or x.shape[-1] != K or K < 1:
        raise ValueError(f"expected x [..., {K}] with at least one number a row, got {tuple(x.shape)}")
    _vector(bias, N, x.dtype, x.device, "bias")
    if residual is not None:
        _residual(residual, (*x.shape[:-1], N), x.dtype, x.device)
    _no_tangent("linear_act", x, weight, bias, residual)
    _act(act)
    kept8 = _checkpoint(checkpoint)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or getattr(bias, "requires_grad", False) or
                                    getattr(residual, "requires_grad", False)):
        return _on(x, _LinearAct.apply, x, weight, bias, residual, act, kept8)
    return _on(x, _linear_forward, x, weight, bias, residual, act, False)[0]


def linear_act(x, weight, bias=None, residual=None, act="none", checkpoint=None):
    """``act(x @ weight.T + bias + residual)`` in one pass, products and sums in 32 bits.

    ``x`` [..., K], ``weight`` [N, K] and ``residual`` [..., N] are float16 or bfloat16, as the result is; ``bias`` [N] is of that type or
    float32; ``act`` is "none", "relu" or "silu".  Differentiable once, backwards, in all four: the gradient of what the
    activation is taken of is rounded to x's type before it is multiplied, and so is, for "silu", that itself.
    ``checkpoint="mx8"`` keeps x for the weight's gradient in microscaled 8 bits in place of x (33/32 byte a number): that
    gradient is then the product with the rounded x."""
    return _linear_act(x, weight, bias, residual, act, checkpoint)


def conv1x1_act(x, weight, bias=None, residual=None, act="none", checkpoint=None):
    """``linear_act`` over the pixels of a channels-last tensor: ``x`` [batch, C, H, W], ``weight`` [N, C] or [N, C, 1, 1], ``residual``
    [batch, N, H, W]; the result is channels last [batch, N, H, W]."""
    x = _images(x, "x")
    if isinstance(weight, torch.Tensor) and weight.dim() == 4 and weight.shape[2:] == (1, 1):
        weight = weight.flatten(1)
    if residual is not None:
        residual = _images(residual, "residual")
    return _linear_act(x, weight, bias, residual, act, checkpoint).permute(0, 3, 1, 2)


# ---- RMS norm ---------------------------------------------------------------------------------------------------------------

_rms_plans = _Cache()


def _rms_plan(rows, C, dtype, weight_dtype, eps, x_step, r_step, dy_step, dh_step, backward):
    key = (rows, C, dtype, weight_dtype, eps, x_step, r_step, dy_step, dh_step, backward)
    plan = _rms_plans.get(key)
    if plan is None:
        desc = _lib.RmsNormDesc(rows, C, _DTYPES[dtype], _DTYPES[weight_dtype], eps, x_step, r_step, dy_step, dh_step)
        need = ctypes.c_size_t()
        check(lib().tdc_rms_norm_workspace(byref(desc), byref(need)))
        plan = _rms_plans.keep(key, (byref(desc), need.value if backward else 0))
    return plan


def _rms_forward(x, weight, residual, eps, output8, grad, kept8):
    """(y or an Mx8Tensor, h or None, rstd or None, h in 8 bits or None), on the current device."""
    dev, dtype, C, index = x.device, x.dtype, x.shape[-1], x.get_device()
    flat, M, x_step = _flat(x)
    r_step, r_at, h = 0, None, None
    if residual is not None:
        r, _, r_step = _flat(residual)
        r_at = r.data_ptr()
        h = _like(x)
    ref, _ = _rms_plan(M, C, dtype, _f32 if weight is None else weight.dtype, eps, x_step, r_step, 0, 0, False)
    if output8:
        q = Mx8Tensor._new(M, C, tuple(x.shape), dev, index)
        status = _call("tdc_rms_norm_forward_mx8")(ref, flat.data_ptr(), r_at, _ptr(weight), q._codes_at, q._scales_at, _ptr(h),
                                                   _raw_stream(index))
        if status:
            check(status)
        return q, h, None, None
    y = _like(x)
    rstd = _empty(M, dtype=_f32, device=dev) if grad else None
    kept = Mx8Tensor._new(M, C, tuple(x.shape), dev, index) if kept8 else None
    status = _call("tdc_rms_norm_forward")(ref, flat.data_ptr(), r_at, _ptr(weight), y.data_ptr(), _ptr(h), _ptr(rstd),
                                           kept._codes_at if kept8 else None, kept._scales_at if kept8 else None, _raw_stream(index))
    if status:
        check(status)
    return y, h, rstd, kept


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, kept8):
        y, h, rstd, kept = _rms_forward(x, weight, residual, eps, False, True, kept8)
        ctx.how = (eps, kept8, tuple(x.shape), x.dtype)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(kept._held if kept8 else x if residual is None else h, weight, rstd)
        return y if residual is None else (y, h)

    @staticmethod
    @_once
    def backward(ctx, dy, dh=None):
        held, weight, rstd = ctx.saved_tensors
        _no_tangent("the gradient of rms_norm", dy, dh)
        eps, kept8, shape, dtype = ctx.how
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if dy is None:      # (only h was used)
            return dh if need_x else None, torch.zeros_like(weight) if need_w and dh is not None else None, dh if need_r else None, None, None
        dev, C, index = dy.device, shape[-1], dy.get_device()
        g, M, dy_step = _flat(dy)
        h_step, dh_step, e = 0, 0, None
        if kept8:
            q = Mx8Tensor._of(held, M, C, shape, dev, index)
            h_at, h_scales = q._codes_at, q._scales_at
        else:
            flat, _, h_step = _flat(held)
            h_at, h_scales = flat.data_ptr(), None
        if dh is not None:
            e, _, dh_step = _flat(dh)
        ref, need = _rms_plan(M, C, dtype, _f32 if weight is None else weight.dtype, eps, h_step, 0, dy_step, dh_step, True)
        dx = _like(dy) if need_x or need_r else None
        dw = _empty_like(weight) if need_w else None
        need = need if need_w else 0
        ws = _empty(need, dtype=_u8, device=dev) if need else None
        status = _call("tdc_rms_norm_backward")(ref, h_at, h_scales, _ptr(weight), g.data_ptr(), _ptr(e), rstd.data_ptr(), _ptr(dx),
                                                _ptr(dw), _ptr(ws), need, _raw_stream(index))
        if status:
            check(status)
        return dx if need_x else None, dw, dx if need_r else None, None, None


def _rms_check(what, x, weight, residual, eps):
    _number_tensor(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        raise ValueError(f"expected x [..., C] with C from 1 to 8192, got {tuple(x.shape)}")
    _vector(weight, x.shape[-1], x.dtype, x.device, "weight")
    if residual is not None:
        _residual(residual, tuple(x.shape), x.dtype, x.device)
    _no_tangent(what, x, weight, residual)
    return float(eps)


def rms_norm(x, weight=None, residual=None, eps=1e-6, checkpoint=None):
    """``weight * h / sqrt(mean(h ** 2) + eps)`` over the last axis, ``h = x + residual``.

    ``x`` and ``residual`` [..., C] (C up to 8192) are float32, float16 or bfloat16; ``weight`` [C] is of that type or float32.  Without
    a residual h is x and the result is returned; with one ``(result, h)``, h rounded to x's type, which is what is normalised.
    Sums are in 32 bits (a row whose squares' sum passes 3.4e38 comes out as zeros).  Differentiable once, backwards, in all three.
    ``checkpoint="mx8"`` keeps h for the gradient in microscaled 8 bits in place of h
    (33/32 byte a number): the gradients are then those at the rounded h, with the unrounded one's root mean square."""
    eps = _rms_check("rms_norm", x, weight, residual, eps)
    kept8 = _checkpoint(checkpoint)
    if torch.is_grad_enabled() and (x.requires_grad or getattr(weight, "requires_grad", False) or getattr(residual, "requires_grad", False)):
        return _on(x, _RmsNorm.apply, x, weight, residual, eps, kept8)
    y, h, _, _ = _on(x, _rms_forward, x, weight, residual, eps, False, False, False)
    return y if residual is None else (y, h)


def rms_norm_mx8(x, weight=None, residual=None, eps=1e-6):
    """``rms_norm`` with its result in 8 bits, quantised from the 32-bit values: an ``Mx8Tensor`` of x's shape for ``mx8_linear``, with a
    residual ``(Mx8Tensor, h)``.  Has no gradient: an ``x`` or ``residual`` that requires one is refused, a ``weight`` that does is taken
    as it is, with a warning."""
    eps = _rms_check("rms_norm_mx8", x, weight, residual, eps)
    for t, name in ((x, "x"), (residual, "residual")):
        if _wants(t):
            _no_gradient("rms_norm_mx8", name)
    if _wants(weight):
        warnings.warn("rms_norm_mx8 has no gradient: weight gets none from it (torch.no_grad() says that this is meant)", stacklevel=2)
    q, h, _, _ = _on(x, _rms_forward, x, weight, residual, eps, True, False, False)
    return q if residual is None else (q, h)
