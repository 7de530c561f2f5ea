"""Timed cases of the operators that stand around a 1x1 factor in 16 and 8 bits: the product with bias, residual and
activation and its gradients, RMS norm with the residual's addition and its gradients, checkpoints in microscaled 8-bit
floating point (E4M3 values in blocks of 32 with a power-of-two scale), the product of two such operands, and RMS norm
handed to that product in 8 bits.

Tensors are rows [rows, K]: the pixels of a channels-last image, or tokens.  `run` computes each operator in plain torch
operations where `own` is false and through the library's entry points where it is true.  Sizes are those of the residual
networks' stages (56/28/14/7 pixels, 64 to 2048 channels, 1000 classes), and generic products.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6


def _package():
    at = os.path.join(os.getcwd(), "ppopp23-tdc_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tdc_amd
    return tdc_amd


def _product(kind, name, rows, K, N, act, bias, residual, dtype, checkpoint="none"):
    c = {"kind": kind, "rows": rows, "K": K, "N": N, "act": act, "bias": bias, "residual": residual, "dtype": dtype,
         "checkpoint": checkpoint}
    return {"name": name, **c} if name else c


def _norm(kind, name, rows, C, residual, dtype, checkpoint="none"):
    c = {"kind": kind, "rows": rows, "C": C, "residual": residual, "dtype": dtype, "checkpoint": checkpoint}
    return {"name": name, **c} if name else c


def _block(name, rows, C, N, add, act, dtype):
    c = {"kind": "block", "rows": rows, "C": C, "N": N, "add": add, "act": act, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One token through a large layer: the weights' bytes are all there is.
        _product("linear", "linear_1x4096x16384_bf16", 1, 4096, 16384, "none", False, False, "bf16"),
        # A bottleneck's last 1x1 factor with its residual, for a serving batch: activations in and out dominate.
        _product("linear", "linear_25088x128x512_bf16", 32 * 28 * 28, 128, 512, "relu", True, True, "bf16"),
        # A product large enough to be held by the matrix cores alone.
        _product("linear", "linear_8192x8192x8192_bf16", 8192, 8192, 8192, "none", False, False, "bf16"),
        # A classifier's training step on a ragged batch, no size of which is round.
        _product("linear_train", "linear_train_33x2001x1001_f16", 33, 2001, 1001, "silu", True, False, "f16"),
        # A training step of a bottleneck's first factor: weights far smaller than the sums that make their gradient.
        _product("linear_train", "linear_train_25088x512x128_bf16", 32 * 28 * 28, 512, 128, "none", True, True, "bf16"),
        # A training step of a large layer that keeps its input in 8 bits for the backward pass.
        _product("linear_train", "linear_train_8192x4096x4096_bf16_mx8", 8192, 4096, 4096, "silu", True, False, "bf16", "mx8"),
        # One forward for a serving batch of first-stage pixels.
        _norm("rms", "rms_100352x256_bf16", 32 * 56 * 56, 256, True, "bf16"),
        # A training step of no round size: rows that start at no aligned address.
        _norm("rms_train", "rms_train_663x1001_f16", 663, 1001, False, "f16"),
        # A training step over a large feature map that keeps the sum in 8 bits for the backward pass.
        _norm("rms_train", "rms_train_100352x512_bf16_mx8", 32 * 56 * 56, 512, True, "bf16", "mx8"),
        # A ragged batch through a classifier in 8 bits, with a K that ends inside a block.
        _product("mx8_linear", "mx8_linear_33x2000x1001_f16", 33, 2000, 1001, "relu", True, False, "f16"),
        # A large product in 8 bits, its input quantised on the way.
        _product("mx8_linear", "mx8_linear_8192x8192x8192_bf16", 8192, 8192, 8192, "none", False, False, "bf16"),
        # residual -> norm -> product in 8 bits, for a serving batch of the second stage.
        _block("block_25088x512x128_bf16", 32 * 28 * 28, 512, 128, True, "silu", "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear_train", "linear_train", "rms", "rms_train", "mx8_linear", "block"))
    dtype, act = rng.choice(("f16", "bf16", "bf16")), rng.choice(("none", "relu", "silu"))
    if kind in ("linear", "linear_train", "mx8_linear"):
        train = kind == "linear_train"
        M = _log(rng, 1, 64) if rng.random() < 0.4 else _log(rng, 64, 32768)
        K, N = _log(rng, 32, 8192), _log(rng, 32, 8192)
        if rng.random() < 0.6:
            K, N = (K + 31) // 32 * 32, (N + 15) // 16 * 16
        while M * K * N > (8192 * 4096 * 4096 if train else 8192 ** 3):
            M //= 2
        if train and N < 64:
            act = "silu"        # (few outputs: one whose sign rounding decides would show in dx)
        return _product(kind, None, M, K, N, act, rng.random() < 0.5, rng.random() < 0.3,
                        dtype, "mx8" if train and rng.random() < 0.4 else "none")
    if kind in ("rms", "rms_train"):
        dtype = rng.choice((dtype, dtype, "f32"))
        while True:
            rows, C = _log(rng, 1, 100352), _log(rng, 16, 8192)
            if rng.random() < 0.5:
                C = (C + 31) // 32 * 32
            if 1024 <= rows * C <= 100352 * 512 // (2 if dtype == "f32" else 1):
                return _norm(kind, None, rows, C, rng.random() < 0.6, dtype,
                             "mx8" if kind == "rms_train" and rng.random() < 0.4 else "none")
    while True:
        rows, C, N = _log(rng, 1, 32768), _log(rng, 64, 4096), _log(rng, 32, 4096)
        if rows * max(C, N) <= 100352 * 256:
            return _block(None, rows, C, N, rng.random() < 0.6, act, dtype)


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, rows, C, dtype):
    """What a layer hands on: every channel with a spread and an offset of its own, a few of them large."""
    x = torch.randn((rows, C), generator=g, device="cuda")
    spread = torch.rand(C, generator=g, device="cuda") + 0.5
    spread = torch.where(torch.rand(C, generator=g, device="cuda") < 0.01, spread * 16, spread)
    return x.mul_(spread).add_(torch.randn(C, generator=g, device="cuda") * 0.5).to(_DTYPES[dtype])


def _normal(g, shape, dtype, by=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * by).to(_DTYPES[dtype])


def _inputs(case, seed):
    """All inputs of a case as numbers."""
    g, kind, M, dtype = _generator(seed), case["kind"], case["rows"], case["dtype"]
    if kind in ("rms", "rms_train", "block"):
        C = case["C"]
        s = {"x": _activations(g, M, C, dtype), "gamma": torch.randn(C, generator=g, device="cuda") * 0.2 + 1,
             "residual": _normal(g, (M, C), dtype) if case.get("residual", case.get("add")) else None}
        if kind == "rms_train":
            s["dy"] = _normal(g, (M, C), dtype)
            s["dh"] = _normal(g, (M, C), dtype) if case["residual"] else None
        if kind == "block":
            s["weight"] = _normal(g, (case["N"], C), "f32", 1 / math.sqrt(C))
            s["bias"] = _normal(g, case["N"], "f32", 0.1)
        return s
    K, N = case["K"], case["N"]
    params = "f32" if kind == "mx8_linear" else dtype      # (weights in 8 bits come from 32)
    s = {"x": _activations(g, M, K, dtype), "weight": _normal(g, (N, K), params, 1 / math.sqrt(K)),
         "bias": _normal(g, N, params, 0.1) if case["bias"] else None,
         "residual": _normal(g, (M, N), dtype) if case["residual"] else None}
    if kind == "linear_train":
        s["dy"] = _normal(g, (M, N), dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("linear_train", "rms_train"):
        for name in ("x", "weight", "bias", "gamma", "residual"):
            if s.get(name) is not None:
                s[name].requires_grad_()
    if case["kind"] in ("mx8_linear", "block"):
        # The layer's weights are kept in 8 bits: as the library's handle, or as the values that those bits stand for.
        s["weight"] = _package().mx8_quantize(s["weight"]) if own else _rounded_plain(s["weight"])
    return case, s


# ---- the plain form ----------------------------------------------------------------------------------------------------

def _act_plain(z, act):
    return z.clamp(min=0) if act == "relu" else z / (1 + torch.exp(-z)) if act == "silu" else z


def _slope_plain(z, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return (z > 0).float()


def _rounded_plain(x):
    """The values that 8 bits a number and a scale a block of 32 along the last axis hold of x, in 32 bits."""
    rows, K = x.shape
    v = x.float()
    if K % 32:
        v = torch.cat((v, v.new_zeros((rows, -K % 32))), -1)
    v = v.reshape(rows, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 9).clamp(-127, 127)     # floor(log2(top)) - 8: the largest power below 448 goes to 256
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    v = torch.ldexp(v, -e)
    step = (torch.frexp(v).exponent - 4).clamp(min=-9)       # three bits behind the leading one, 2^-9 at least
    v = torch.ldexp(torch.ldexp(v, -step).round(), step).clamp(-448, 448)
    return torch.ldexp(v, e).reshape(rows, -1)[:, :K]


def _product_plain(x, s, act):
    """x and the weight in 32 bits: (the sums with bias and residual, the activation of them)."""
    z = x @ s["weight"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if s.get("residual") is not None:
        z = z + s["residual"].float()
    return z, _act_plain(z, act)


def _train_plain(case, s):
    x, weight, act = s["x"].float(), s["weight"].float(), case["act"]
    z, y = _product_plain(x, s, act)
    dz = s["dy"].float()
    if act != "none":
        dz = dz * _slope_plain(z, act)
    kept = _rounded_plain(s["x"]) if case["checkpoint"] == "mx8" else x
    out = [y, dz @ weight, dz.t() @ kept]
    if case["bias"]:
        out.append(dz.sum(0))
    if case["residual"]:
        out.append(dz)
    return tuple(v.to(s["x"].dtype) for v in out)


def _norm_plain(s):
    """(h, h / its root mean square, that times gamma, 1 / the root), in 32 bits."""
    h = s["x"].float()
    if s["residual"] is not None:
        h = (h + s["residual"].float()).to(s["x"].dtype).float()
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)
    return h, h * r * s["gamma"], r


def _norm_train_plain(case, s):
    h, y, r = _norm_plain(s)
    kept = (_rounded_plain(h) if case["checkpoint"] == "mx8" else h) * r
    dy = s["dy"].float()
    g = dy * s["gamma"]
    dx = r * (g - kept * (g * kept).mean(-1, keepdim=True))
    dtype, dgamma = s["x"].dtype, (dy * kept).sum(0)
    if not case["residual"]:
        return y.to(dtype), dx.to(dtype), dgamma
    dx = (dx + s["dh"].float()).to(dtype)
    return y.to(dtype), h.to(dtype), dx, dx, dgamma


def _plain(case, s):
    kind, dtype = case["kind"], s["x"].dtype
    if kind == "linear":
        return _product_plain(s["x"].float(), s, case["act"])[1].to(dtype)
    if kind == "linear_train":
        return _train_plain(case, s)
    if kind == "mx8_linear":
        return _product_plain(_rounded_plain(s["x"]), s, case["act"])[1].to(dtype)
    if kind == "rms_train":
        return _norm_train_plain(case, s)
    h, y, _ = _norm_plain(s)
    if kind == "rms":
        return (y.to(dtype), h.to(dtype)) if case["residual"] else y.to(dtype)
    y = _product_plain(_rounded_plain(y), {"weight": s["weight"], "bias": s["bias"]}, case["act"])[1].to(dtype)
    return (y, h.to(dtype)) if case["add"] else y


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    case, s = state
    if not own:
        with torch.no_grad():
            return _plain(case, s)
    tdc, kind, x = _package(), case["kind"], s["x"]
    if kind == "linear":
        return tdc.linear_act(x, s["weight"], s["bias"], s["residual"], act=case["act"])
    if kind == "mx8_linear":
        return tdc.mx8_linear(x, s["weight"], s["bias"], s["residual"], act=case["act"])
    if kind == "linear_train":
        y = tdc.linear_act(x, s["weight"], s["bias"], s["residual"], act=case["act"],
                           checkpoint="mx8" if case["checkpoint"] == "mx8" else None)
        wrt = [t for t in (x, s["weight"], s["bias"], s["residual"]) if t is not None]
        return (y.detach(), *torch.autograd.grad(y, wrt, s["dy"]))
    if kind == "rms":
        return tdc.rms_norm(x, s["gamma"], s["residual"], eps=_EPS)
    if kind == "rms_train":
        out = tdc.rms_norm(x, s["gamma"], s["residual"], eps=_EPS, checkpoint="mx8" if case["checkpoint"] == "mx8" else None)
        if not case["residual"]:
            return (out.detach(), *torch.autograd.grad(out, (x, s["gamma"]), s["dy"]))
        y, h = out
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), (x, s["residual"], s["gamma"]), (s["dy"], s["dh"])))
    q = tdc.rms_norm_mx8(x, s["gamma"], s["residual"], eps=_EPS)
    q, h = q if case["add"] else (q, None)
    y = tdc.mx8_linear(q, s["weight"], s["bias"], act=case["act"], out_dtype=x.dtype)
    return (y, h) if case["add"] else y


def work(case):
    kind, size, M = case["kind"], _BYTES[case["dtype"]], case["rows"]
    if kind in ("rms", "rms_train"):
        n, C = M * case["C"], case["C"]
        passes = 4 if case["residual"] else 2      # x, residual, y, h
        if kind == "rms":
            return {"bytes": passes * n * size + 4 * C, "flops": 4 * n}
        # dy, dh and the two gradients (of a sum's two terms: one tensor), dgamma
        return {"bytes": (passes + (3 if case["residual"] else 2)) * n * size + 8 * C, "flops": 14 * n}
    if kind == "block":
        C, N = case["C"], case["N"]
        return {"bytes": M * C * size * (3 if case["add"] else 1) + N * -(-C // 32) * 33 + M * N * size + 4 * (N + C),
                "flops": 2 * M * N * C}
    K, N = case["K"], case["N"]
    weights, outputs = (N * -(-K // 32) * 33 if kind == "mx8_linear" else N * K * size), M * N * size
    moved = M * K * size + weights + outputs * (2 if case["residual"] else 1) + (4 if kind == "mx8_linear" else size) * N * case["bias"]
    if kind != "linear_train":
        return {"bytes": moved, "flops": 2 * M * N * K}
    moved += outputs * (2 if case["residual"] else 1) + M * K * size + weights + N * size * case["bias"]     # dy and the gradients
    return {"bytes": moved, "flops": 6 * M * N * K}


# ---- in 64 bits, from the definitions ------------------------------------------------------------------------------------

def _e4m3():
    """The magnitudes of E4M3, in the order of their codes: 2^-9 and its multiples, then eight to a power of two."""
    small = [n / 512 for n in range(8)]
    return small + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]


def _rounded_exact(x):
    """Each block of 32: the power of two that takes its largest magnitude into [256, 512), then the nearest of E4M3's values,
    halfway between two to the one with an even place in that row."""
    rows, K = x.shape
    row = torch.tensor(_e4m3(), dtype=torch.float64, device=x.device)
    halfway = (row[1:] + row[:-1]) / 2
    out = torch.empty_like(x, dtype=torch.float64)
    step = max(32, 2 ** 24 // max(rows, 1) // 32 * 32)
    for k in range(0, K, step):
        part = x[:, k:k + step].double()
        n = part.shape[1]
        part = torch.nn.functional.pad(part, (0, -n % 32)).view(rows, -1, 32)
        scale = torch.exp2(torch.floor(torch.log2(part.abs().max(-1, keepdim=True).values)) - 8)
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))
        size = (part.abs() / scale).contiguous()
        low, high = torch.bucketize(size, halfway), torch.bucketize(size, halfway, right=True)
        place = torch.where(low % 2 == 0, low, high)
        out[:, k:k + step] = (row[place] * scale * torch.sign(part)).view(rows, -1)[:, :n]
    return out


def _act_exact(z, act):
    return torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z


def _product_exact(x, weight, bias, residual, act):
    z = torch.mm(x, weight.t().contiguous())
    z = z if bias is None else z + bias
    return _act_exact(z if residual is None else z + residual, act)


def exact(case, seed):
    given, kind = _inputs(case, seed), case["kind"]
    dtype = given["x"].dtype
    s = {k: v.double() if v is not None else None for k, v in given.items()}
    x, residual = s["x"], s["residual"] if "residual" in s else None
    if kind in ("linear", "mx8_linear"):
        w = s["weight"]
        if kind == "mx8_linear":
            x, w = _rounded_exact(x), _rounded_exact(w)
        return _product_exact(x, w, s["bias"], residual, case["act"])
    if kind == "linear_train":
        wrt = [t.requires_grad_() for t in (x, s["weight"], s["bias"], residual) if t is not None]
        y = _product_exact(x, s["weight"], s["bias"], residual, case["act"])
        grads = list(torch.autograd.grad(y, wrt, s["dy"]))
        if case["checkpoint"] == "mx8":
            # the weight's gradient is linear in what is kept of x
            z = torch.mm(x, s["weight"].t().contiguous()).detach()
            z = z if s["bias"] is None else z + s["bias"].detach()
            z = (z if residual is None else z + residual.detach()).requires_grad_()
            dz, = torch.autograd.grad(_act_exact(z, case["act"]), z, s["dy"])
            grads[1] = torch.mm(dz.t().contiguous(), _rounded_exact(x.detach()))
        return (y.detach(), *grads)
    h = x if residual is None else (x + residual).to(dtype).double()
    root = torch.sqrt((h ** 2).mean(1, keepdim=True) + _EPS)
    y = h / root * s["gamma"]
    if kind == "rms":
        return (y, h) if residual is not None else y
    if kind == "block":
        y = _product_exact(_rounded_exact(y.float()), _rounded_exact(s["weight"]), s["bias"], None, case["act"])
        return (y, h) if residual is not None else y
    if case["checkpoint"] == "mx8":
        unit = _rounded_exact(h) / root
        along = (s["dy"] * s["gamma"] * unit).sum(1, keepdim=True) / h.shape[1]
        dx, dgamma = (s["dy"] * s["gamma"] - unit * along) / root, (s["dy"] * unit).sum(0)
    else:
        at, gamma = h.clone().requires_grad_(), s["gamma"].requires_grad_()
        out = at / torch.sqrt((at ** 2).mean(1, keepdim=True) + _EPS) * gamma
        dx, dgamma = torch.autograd.grad(out, (at, gamma), s["dy"])
        y = y.detach()
    if residual is None:
        return y, dx, dgamma
    dx = dx + s["dh"]
    return y, h, dx, dx, dgamma
