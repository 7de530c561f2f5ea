"""Timed cases of the channels-last operators: group norm with an activation (and its gradient), numbers in microscaled
4-bit floating point (E2M1 values in blocks of 32 with a power-of-two scale), the product of two such operands, and
group norm handed to that product in 4 bits.

Tensors are [batch, channels, height, width] in channels-last memory, as a 1x1 factor convolution wants them as a matrix
product, or [rows, K].  `run` computes each operator in plain torch operations where `own` is false and through the
library's entry points where it is true.  Sizes are those of the residual networks' stages (56/28/14/7 pixels, 64 to 2048
channels, 1000 classes), and generic square products.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5


def _package():
    at = os.path.join(os.getcwd(), "ppopp23-tdc_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tdc_amd
    return tdc_amd


def _norm(name, kind, batch, H, W, C, groups, act, dtype):
    c = {"kind": kind, "batch": batch, "H": H, "W": W, "C": C, "groups": groups, "act": act, "dtype": dtype}
    return {"name": name, **c} if name else c


def _quantize(name, rows, K, dtype):
    c = {"kind": "quantize", "rows": rows, "K": K, "dtype": dtype}
    return {"name": name, **c} if name else c


def _linear(name, rows, K, N, act, bias, residual, dtype):
    c = {"kind": "linear", "rows": rows, "K": K, "N": N, "act": act, "bias": bias, "residual": residual, "dtype": dtype}
    return {"name": name, **c} if name else c


def _block(name, batch, H, W, C, N, groups, act, residual, dtype):
    c = {"kind": "block", "batch": batch, "H": H, "W": W, "C": C, "N": N, "groups": groups, "act": act, "residual": residual,
         "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One image at the deepest stage of a residual network: nothing but launch and latency.
        _norm("norm_1x7x7x512_f32", "norm", 1, 7, 7, 512, 32, "silu", "f32"),
        # The output of a first-stage block for a serving batch.
        _norm("norm_32x56x56x256_bf16", "norm", 32, 56, 56, 256, 32, "relu", "bf16"),
        # A training step of no round size: 19 channels a group, pixels that start at no aligned address.
        _norm("norm_train_3x13x17x114_f16", "norm_train", 3, 13, 17, 114, 6, "silu", "f16"),
        # A training step over early, large feature maps: forward and gradients, all of it memory traffic.
        _norm("norm_train_32x112x112x128_bf16", "norm_train", 32, 112, 112, 128, 32, "silu", "bf16"),
        # The deepest feature map of one image, in and out of 4 bits.
        _quantize("quantize_49x2048_f32", 49, 2048, "f32"),
        # A serving batch of first-stage activations.
        _quantize("quantize_100352x256_bf16", 32 * 56 * 56, 256, "bf16"),
        # One token through a large layer: the weights' bytes are all there is.
        _linear("linear_1x4096x16384_bf16", 1, 4096, 16384, "none", False, False, "bf16"),
        # A classifier for a ragged batch, with a K that ends inside a block.
        _linear("linear_33x2000x1001_f32", 33, 2000, 1001, "relu", True, False, "f32"),
        # A bottleneck's last 1x1 factor with its residual, for a serving batch: activations in and out dominate.
        _linear("linear_25088x128x512_bf16", 32 * 28 * 28, 128, 512, "relu", True, True, "bf16"),
        # A product large enough to be held by the matrix cores alone.
        _linear("linear_8192x8192x8192_bf16", 8192, 8192, 8192, "none", False, False, "bf16"),
        # norm -> activation -> 1x1 factor of one image.
        _block("block_1x14x14x1024x256_bf16", 1, 14, 14, 1024, 256, 32, "silu", False, "bf16"),
        # The same for a serving batch of the second stage.
        _block("block_32x28x28x512x128_bf16", 32, 28, 28, 512, 128, 32, "silu", True, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


_MAX_VALUES = 32 * 112 * 112 * 128


def draw(rng):
    kind = rng.choice(("norm", "norm_train", "quantize", "linear", "linear", "block"))
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    act = rng.choice(("none", "relu", "silu"))
    if kind in ("norm", "norm_train"):
        while True:
            groups = rng.choice((1, 2, 4, 6, 8, 16, 32, 32))
            C = groups * _log(rng, 1, 64)
            c = _norm(None, kind, _log(rng, 1, 64), _log(rng, 3, 112), _log(rng, 3, 112), C, groups, act, dtype)
            values = c["batch"] * c["H"] * c["W"] * C
            if 16 <= C <= 2048 and 4096 <= values <= _MAX_VALUES // (2 if dtype == "f32" else 1):
                return c
    if kind == "quantize":
        while True:
            rows, K = _log(rng, 1, 200000), _log(rng, 32, 8192)
            if 2048 <= rows * K <= _MAX_VALUES // 2:
                return _quantize(None, rows, K, dtype)
    if kind == "linear":
        M = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 64, 8192)
        K, N = _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.5:
            K, N = (K + 31) // 32 * 32, (N + 15) // 16 * 16
        return _linear(None, M, K, N, act, rng.random() < 0.5, rng.random() < 0.3, dtype)
    while True:
        groups = rng.choice((8, 16, 32))
        C = groups * _log(rng, 4, 64)
        c = _block(None, _log(rng, 1, 32), _log(rng, 7, 56), _log(rng, 7, 56), C, _log(rng, 32, 1024), groups, act,
                   rng.random() < 0.5, rng.choice(("f16", "bf16")))     # a serving path: 16 bits in and out
        if 256 <= C <= 2048 and c["batch"] * c["H"] * c["W"] * max(C, c["N"]) <= _MAX_VALUES // 2:
            return c


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, shape, dtype):
    """What a layer hands on: every channel (the last axis) with a spread and an offset of its own, a few of them large."""
    x = torch.randn(shape, generator=g, device="cuda")
    C = shape[-1]
    spread = torch.rand(C, generator=g, device="cuda") + 0.5
    spread = torch.where(torch.rand(C, generator=g, device="cuda") < 0.01, spread * 16, spread)
    return x.mul_(spread).add_(torch.randn(C, generator=g, device="cuda") * 0.5).to(_DTYPES[dtype])


def _norm_inputs(case, g):
    B, H, W, C = case["batch"], case["H"], case["W"], case["C"]
    return {"x": _activations(g, (B, H, W, C), case["dtype"]).permute(0, 3, 1, 2),
            "gamma": torch.randn(C, generator=g, device="cuda") * 0.2 + 1, "beta": torch.randn(C, generator=g, device="cuda") * 0.2}


def _inputs(case, seed):
    """All inputs of a case as numbers."""
    g, kind = _generator(seed), case["kind"]
    if kind in ("norm", "norm_train"):
        s = _norm_inputs(case, g)
        if kind == "norm_train":
            s["dy"] = torch.randn((case["batch"], case["H"], case["W"], case["C"]), generator=g,
                                  device="cuda").to(_DTYPES[case["dtype"]]).permute(0, 3, 1, 2)
        return s
    if kind == "quantize":
        return {"x": _activations(g, (case["rows"], case["K"]), case["dtype"])}
    if kind == "linear":
        s, K, out = {"x": _activations(g, (case["rows"], case["K"]), case["dtype"])}, case["K"], (case["rows"], case["N"])
    else:
        s, K, out = _norm_inputs(case, g), case["C"], (case["batch"], case["H"], case["W"], case["N"])
    s["weight"] = torch.randn((case["N"], K), generator=g, device="cuda") / math.sqrt(K)
    s["bias"] = torch.randn(case["N"], generator=g, device="cuda") * 0.1 if case.get("bias", True) else None
    s["residual"] = torch.randn(out, generator=g, device="cuda").to(_DTYPES[case["dtype"]]) if case["residual"] else None
    if kind == "block" and case["residual"]:
        s["residual"] = s["residual"].permute(0, 3, 1, 2)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "norm_train":
        for name in ("x", "gamma", "beta"):
            s[name].requires_grad_()
    if "weight" in s:
        # The layer's weights are kept in 4 bits: as the library's handle, or as the values that those bits stand for.
        s["weight"] = _package().mx4_quantize(s["weight"]) if own else _rounded_plain(s["weight"])
    return case, s


# ---- the plain form ----------------------------------------------------------------------------------------------------

def _act_plain(z, act):
    return z.clamp(min=0) if act == "relu" else z / (1 + torch.exp(-z)) if act == "silu" else z


def _norm_plain(x, gamma, beta, groups):
    """(x hat, z, r) over [batch, pixels, groups, channels of a group], in 32 bits."""
    B, C, H, W = x.shape
    x = x.permute(0, 2, 3, 1).reshape(B, H * W, groups, C // groups).float()
    x = x - x.mean((1, 3), keepdim=True)
    r = torch.rsqrt((x * x).mean((1, 3), keepdim=True) + _EPS)
    xh = x * r
    return xh, xh * gamma.view(groups, -1) + beta.view(groups, -1), r


def _like(v, x):
    """[batch, pixels, ...] back to the shape, memory order and type of x."""
    B, C, H, W = x.shape
    return v.reshape(B, H, W, -1).permute(0, 3, 1, 2).to(x.dtype)


def _norm_train_plain(x, gamma, beta, groups, act, dy):
    xh, z, r = _norm_plain(x, gamma, beta, groups)
    y = _like(_act_plain(z, act), x)
    dz = dy.permute(0, 2, 3, 1).reshape(z.shape).float()
    if act == "relu":
        dz = dz * (z > 0)
    elif act == "silu":
        s = 1 / (1 + torch.exp(-z))
        dz = dz * (s * (1 + z * (1 - s)))
    dgamma, dbeta = (dz * xh).sum((0, 1)).view(-1), dz.sum((0, 1)).view(-1)
    dxh = dz * gamma.view(groups, -1)
    dx = r * (dxh - dxh.mean((1, 3), keepdim=True) - xh * (dxh * xh).mean((1, 3), keepdim=True))
    return y, _like(dx, x), dgamma, dbeta


def _rounded_plain(x):
    """The values that 4 bits a number and a scale a block of 32 along the last axis hold of x, in 32 bits."""
    K = x.shape[-1]
    v = x.float()
    if K % 32:
        v = torch.cat((v, v.new_zeros((*v.shape[:-1], -K % 32))), -1)
    v = v.reshape(*v.shape[:-1], -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)     # floor(log2(top)) - 2: the largest power below 6 goes to 4
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    v = torch.ldexp(v, -e)
    a = v.abs()
    a = torch.where(a < 2, (a * 2).round() / 2, torch.where(a < 4, a.round(), ((a / 2).round() * 2).clamp(max=6)))
    v = torch.ldexp(torch.copysign(a, v), e)
    return v.reshape(*x.shape[:-1], -1)[..., :K]


def _linear_plain(x, weight, bias, residual, act):
    """x: numbers in 32 bits, [..., K]."""
    y = _rounded_plain(x) @ weight.t()
    if bias is not None:
        y = y + bias
    if residual is not None:
        y = y + residual.float()
    return _act_plain(y, act)


def _plain(case, s):
    kind, x = case["kind"], s["x"]
    if kind == "norm":
        return _like(_act_plain(_norm_plain(x, s["gamma"], s["beta"], case["groups"])[1], case["act"]), x)
    if kind == "norm_train":
        return _norm_train_plain(x, s["gamma"], s["beta"], case["groups"], case["act"], s["dy"])
    if kind == "quantize":
        return _rounded_plain(x).to(x.dtype)
    if kind == "linear":
        return _linear_plain(x, s["weight"], s["bias"], s["residual"], case["act"]).to(x.dtype)
    h = _act_plain(_norm_plain(x, s["gamma"], s["beta"], case["groups"])[1], case["act"])
    residual = s["residual"].permute(0, 2, 3, 1) if s["residual"] is not None else None
    h = h.reshape(case["batch"], case["H"], case["W"], -1)
    return _like(_linear_plain(h, s["weight"], s["bias"], residual, "none"), x)


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    case, s = state
    if not own:
        with torch.no_grad():
            return _plain(case, s)
    tdc, kind, x = _package(), case["kind"], s["x"]
    if kind == "norm":
        return tdc.group_norm_act(x, case["groups"], s["gamma"], s["beta"], eps=_EPS, act=case["act"])
    if kind == "norm_train":
        y = tdc.group_norm_act(x, case["groups"], s["gamma"], s["beta"], eps=_EPS, act=case["act"])
        return (y, *torch.autograd.grad(y, (x, s["gamma"], s["beta"]), s["dy"]))
    if kind == "quantize":
        return tdc.mx4_quantize(x).dequantize(x.dtype)
    if kind == "linear":
        return tdc.mx4_linear(x, s["weight"], s["bias"], s["residual"], act=case["act"])
    h = tdc.group_norm_act_mx4(x, case["groups"], s["gamma"], s["beta"], eps=_EPS, act=case["act"])
    return tdc.mx4_conv1x1(h, s["weight"], s["bias"], s["residual"], out_dtype=x.dtype)


def work(case):
    kind, size = case["kind"], _BYTES[case["dtype"]]
    if kind in ("norm", "norm_train"):
        n, C = case["batch"] * case["H"] * case["W"] * case["C"], case["C"]
        if kind == "norm":
            return {"bytes": 2 * n * size + 8 * C, "flops": 10 * n}
        return {"bytes": 4 * n * size + 16 * C, "flops": 40 * n}
    if kind == "quantize":
        n = case["rows"] * case["K"]
        return {"bytes": 2 * n * size, "flops": 8 * n}
    M, K, N = (case["rows"], case["K"], case["N"]) if kind == "linear" else (case["batch"] * case["H"] * case["W"], case["C"], case["N"])
    moved = M * K * size + N * -(-K // 32) * 17 + M * N * size * (2 if case["residual"] else 1)
    return {"bytes": moved + 4 * N * bool(case.get("bias", True)) + (8 * K if kind == "block" else 0), "flops": 2 * M * N * K}


# ---- in 64 bits, from the definitions ------------------------------------------------------------------------------------

def _rounded_exact(x):
    """Each block of 32: the power of two that takes its largest magnitude into [4, 8), then the nearest of 0, 0.5, 1, 1.5, 2,
    3, 4, 6, halfway between two to the one with an even place in that row."""
    x = x.double()
    K = x.shape[-1]
    out = torch.zeros_like(x)
    for k in range(0, K, 32):
        part = x[..., k:k + 32]
        scale = torch.exp2(torch.floor(torch.log2(part.abs().max(-1, keepdim=True).values)) - 2)
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))
        size = part.abs() / scale
        place = torch.zeros_like(size)
        for n, halfway in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
            place += (size >= halfway) if n % 2 else (size > halfway)
        row = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        out[..., k:k + 32] = row[place.long()] * scale * torch.sign(part)
    return out


def _norm_exact(x, gamma, beta, groups, act):
    """x: [batch, channels, height, width] in 64 bits."""
    B, C = x.shape[:2]
    rows = x.reshape(B * groups, -1)
    var, mean = torch.var_mean(rows, 1, unbiased=False, keepdim=True)
    z = ((rows - mean) / torch.sqrt(var + _EPS)).reshape(x.shape) * gamma.view(1, C, 1, 1) + beta.view(1, C, 1, 1)
    return torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    s = {k: v.double() if v is not None else None for k, v in s.items()}
    if kind == "norm":
        return _norm_exact(s["x"], s["gamma"], s["beta"], case["groups"], case["act"])
    if kind == "norm_train":
        wrt = [s[k].requires_grad_() for k in ("x", "gamma", "beta")]
        y = _norm_exact(*wrt, case["groups"], case["act"])
        return (y.detach(), *torch.autograd.grad(y, wrt, s["dy"]))
    if kind == "quantize":
        return _rounded_exact(s["x"])
    x, act = s["x"], case["act"]
    if kind == "block":
        x, act = _norm_exact(x, s["gamma"], s["beta"], case["groups"], act).permute(0, 2, 3, 1).contiguous(), "none"
    rows = _rounded_exact(x.reshape(-1, x.shape[-1]))
    y = torch.mm(rows, _rounded_exact(s["weight"]).t().contiguous())
    if s["bias"] is not None:
        y += s["bias"]
    if s["residual"] is not None:
        r = s["residual"]
        y += (r.permute(0, 2, 3, 1) if kind == "block" else r).reshape(y.shape)
    y = torch.relu(y) if act == "relu" else y * torch.sigmoid(y) if act == "silu" else y
    return y.reshape(case["batch"], case["H"], case["W"], -1).permute(0, 3, 1, 2) if kind == "block" else y
