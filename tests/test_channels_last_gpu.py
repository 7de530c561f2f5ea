"""Group norm with an activation, 4-bit microscaled numbers and their product, against plain 64-bit forms.

Tolerances, from the arithmetic.  u is the unit roundoff of the output's type (2^-24, 2^-11, 2^-8), e = 2^-24.
Norm: x - mean, the scale, the shift and the activation are some ten fp32 operations, each good to e of the largest
magnitude in play, |gamma| (|x hat| + |mean| rstd) + |beta|: 16 e of that, then u |y|.  Its gradient: the same of
|gamma dy| (1 + |x hat|) rstd and of the two group means, whose terms it bounds: 64 e.  The parameters' gradients add
|dz| (1 + |x hat|) in trees of short chains: 64 e of the sum of the magnitudes.  4-bit numbers are exact.  The product adds exact
products in fp32: (16 + K / 64) e of the sum of the magnitudes, and 8 e for bias, residual and activation."""
import ctypes
import math

import numpy as np
import pytest
import torch

import tdc_amd
from oracle import channels_last_ref as ref
from util import seeded

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def close(got, want, bound, what):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound + 2.0 ** -149)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - want), 0)), got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside; at {i} got {got[i]!r} want {want[i]!r} bound {np.broadcast_to(bound, got.shape)[i]:.3g}")


def rows(t):
    """[B, C, ...] as [B, S, C] in 64 bits on the host."""
    t = t.detach().double().cpu()
    return t.reshape(t.shape[0], t.shape[1], -1).permute(0, 2, 1).numpy()


def norm_case(seed, shape, dtype, offset=0.5, wide=None):
    g = seeded(seed)
    B, C, *space = shape
    x = torch.randn(B, *space, wide or C, generator=g) * (torch.rand(wide or C, generator=g) + 0.5) + offset * torch.randn(wide or C, generator=g)
    x = x.to(dtype).cuda()
    if wide:
        x = x[..., (wide - C) // 2:(wide - C) // 2 + C]
    x = x.permute(0, x.dim() - 1, *range(1, x.dim() - 1))
    gamma, beta = torch.randn(C, generator=g) * 0.3 + 1, torch.randn(C, generator=g) * 0.3
    return x, gamma, beta


def check_forward(y, x, groups, gamma, beta, act, eps=1e-5, what=""):
    xh, z, mean, rstd = ref.norm_parts(rows(x), groups, gamma, beta, eps)
    want = ref.act(z, act)
    size = np.abs(gamma) * (np.abs(xh) + np.abs(mean) * rstd) + np.abs(beta)
    close(torch.from_numpy(rows(y)), want, U[y.dtype] * np.abs(want) + 16 * E * size + (2.0 ** -25 if y.dtype == F16 else 0), what)


NORMS = [  # shape, groups
    ((1, 1, 1, 1), 1), ((2, 7, 1, 1), 7), ((1, 512, 7, 7), 32), ((3, 114, 13, 17), 6), ((2, 64, 56, 56), 32),
    ((1, 33, 5, 9), 1), ((2, 24, 11, 3), 24), ((5, 40, 9, 8), 8), ((2, 2048, 3, 3), 32), ((1, 4104, 4, 5), 1),
    ((2, 2050, 3, 2), 1), ((1, 8008, 2, 3), 8), ((2, 3000, 2, 2), 3), ((40, 16, 6, 6), 4), ((1, 96, 150, 150), 3),
    ((2, 36, 1237), 4), ((3, 300), 10), ((1, 48, 3, 4, 5), 6), ((1, 2600, 1, 9), 1300),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", NORMS)
def test_norm_forward(shape, groups, dtype):
    for i, act in enumerate(("none", "relu", "silu")):
        x, gamma, beta = norm_case(100 + i, shape, dtype)
        y = tdc_amd.group_norm_act(x, groups, gamma.cuda(), beta.cuda(), act=act)
        assert y.dtype == dtype and y.shape == x.shape
        check_forward(y, x, groups, gamma.double().numpy(), beta.double().numpy(), act, what=f"{shape} {groups} {act}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups,wide", [((2, 64, 9, 9), 8, 96), ((3, 30, 5, 7), 5, 37), ((2, 2, 8, 8), 1, 7), ((1, 128, 31, 33), 4, 130)])
def test_norm_of_a_channel_slice_and_without_parameters(shape, groups, wide, dtype):
    x, gamma, beta = norm_case(7, shape, dtype, wide=wide)
    one, zero = np.ones(shape[1]), np.zeros(shape[1])
    y = tdc_amd.group_norm_act(x, groups, act="silu")
    check_forward(y, x, groups, one, zero, "silu")
    assert y.is_contiguous(memory_format=torch.channels_last)
    check_forward(tdc_amd.group_norm_act(x, groups, gamma.cuda()), x, groups, gamma.double().numpy(), zero, "none")
    check_forward(tdc_amd.group_norm_act(x, groups, bias=beta.cuda()), x, groups, one, beta.double().numpy(), "none")
    gd, bd = gamma.to(dtype), beta.to(dtype)
    check_forward(tdc_amd.group_norm_act(x, groups, gd.cuda(), bd.cuda(), eps=0.1), x, groups, gd.double().numpy(), bd.double().numpy(),
                  "none", eps=float(np.float32(0.1)))


@pytest.mark.parametrize("offset", [1e2, 1e4])
def test_norm_far_from_zero(offset):
    """Squares of the numbers themselves would leave nothing of the variance."""
    x, gamma, beta = norm_case(11, (2, 32, 40, 40), F32)
    x = x + offset
    y = tdc_amd.group_norm_act(x, 4, gamma.cuda(), beta.cuda())
    check_forward(y, x, 4, gamma.double().numpy(), beta.double().numpy(), "none")


def test_norm_of_nothing_and_of_constants():
    for shape in ((0, 8, 3, 3), (2, 8, 0, 3)):
        x = torch.empty(shape, device="cuda").contiguous(memory_format=torch.channels_last)
        assert tdc_amd.group_norm_act(x, 2).shape == shape
        w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
        x.requires_grad_()
        dx, dw, db = torch.autograd.grad(tdc_amd.group_norm_act(x, 2, w, b).sum(), (x, w, b))
        assert dx.shape == shape and not dw.any() and not db.any()
        assert tdc_amd.group_norm_act_mx4(x.detach(), 2).rows == 0
    x = torch.full((2, 8, 5, 5), 3.25, device="cuda").contiguous(memory_format=torch.channels_last)
    beta = torch.arange(8.0, device="cuda") - 3
    y = tdc_amd.group_norm_act(x, 2, bias=beta, act="relu")
    assert torch.equal(y, beta.clamp(min=0).view(1, 8, 1, 1).expand_as(x))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_norm_keeps_special_values_to_their_image_and_group(value):
    x, gamma, beta = norm_case(12, (3, 32, 9, 10), F32)
    clean = tdc_amd.group_norm_act(x, 4, gamma.cuda(), beta.cuda(), act="relu")
    x[1, 10, 4, 4] = value
    y = tdc_amd.group_norm_act(x, 4, gamma.cuda(), beta.cuda(), act="relu")
    assert y[1, 8:16].isnan().all()
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, 8:16] = True
    assert torch.equal(y[~hit], clean[~hit])


def grad_case(shape, groups, dtype, act, seed=31, dy_like=None):
    x, gamma, beta = norm_case(seed, shape, dtype)
    g = seeded(seed + 1)
    dy = torch.randn(shape, generator=g).to(dtype).cuda()
    if dy_like != "nchw" and len(shape) == 4:
        dy = dy.contiguous(memory_format=torch.channels_last)
    xg, w, b = x.detach().requires_grad_(), gamma.cuda().requires_grad_(), beta.cuda().requires_grad_()
    y = tdc_amd.group_norm_act(xg, groups, w, b, act=act)
    return x, gamma.double().numpy(), beta.double().numpy(), dy, y, torch.autograd.grad(y, (xg, w, b), dy)


def check_grads(x, gamma, beta, dy, grads, groups, act, what, eps=1e-5):
    xs, d = rows(x), rows(dy)
    dx, dgamma, dbeta = ref.norm_grads(xs, d, groups, gamma, beta, eps, act)
    xh, z, mean, rstd = ref.norm_parts(xs, groups, gamma, beta, eps)
    far = 1 + np.abs(mean) * rstd                      # what an error of the mean weighs
    size = np.abs(gamma * d) * far * (1 + np.abs(xh))
    B, S, C = xs.shape
    groups_of = lambda v: np.repeat(v.reshape(B, S, groups, -1).mean(axis=(1, 3)).reshape(B, 1, groups), C // groups, axis=2)  # noqa: E731
    mean_size = groups_of(size)
    bound = 64 * E * rstd * (size + mean_size * (1 + np.abs(xh))) + U[grads[0].dtype] * np.abs(dx) + (2.0 ** -25 if grads[0].dtype == F16 else 0)
    if act == "relu":      # at the kink a rounding error of z decides
        kink = np.abs(z) <= 16 * E * (np.abs(gamma) * (np.abs(xh) + np.abs(mean) * rstd) + np.abs(beta))
        bound = np.where(kink, np.inf, bound)
    close(torch.from_numpy(rows(grads[0])), dx, bound, what + " dx")
    total = (np.abs(d) * far * (1 + np.abs(xh)) ** 2).sum(axis=(0, 1))
    u = 0.0 if grads[1].dtype == F32 else U[grads[1].dtype]
    close(grads[1], dgamma, 64 * E * total + u * np.abs(dgamma), what + " dgamma")
    close(grads[2], dbeta, 64 * E * total + u * np.abs(dbeta), what + " dbeta")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", [n for n in NORMS if n[0][0] * math.prod(n[0][2:]) > 1])
def test_norm_gradients(shape, groups, dtype):
    for i, act in enumerate(("none", "relu", "silu")):
        x, gamma, beta, dy, y, grads = grad_case(shape, groups, dtype, act, seed=40 + i)
        check_forward(y, x, groups, gamma, beta, act)
        check_grads(x, gamma, beta, dy, grads, groups, act, f"{shape} {groups} {act}")


def test_norm_gradients_by_differences():
    """The slope of sum(y dy) along a direction, from two forwards.  Third derivatives are of order one, so a step of 2^-7
    is off by some 1e-5 of the sum of magnitudes, and rounding by 2^7 times 1e-6 of it over the root of the 10^4 terms."""
    for act in ("none", "silu"):
        x, gamma, beta, dy, y, grads = grad_case((2, 24, 15, 14), 4, F32, act)
        g = seeded(77)
        at = [x, torch.from_numpy(gamma).float().cuda(), torch.from_numpy(beta).float().cuda()]
        way = [torch.randn(t.shape, generator=g).cuda().contiguous(memory_format=torch.channels_last) if t.dim() == 4 else
               torch.randn(t.shape, generator=g).cuda() for t in at]
        for k in range(3):
            h, ends = 2.0 ** -7, []
            for sign in (1, -1):
                p = [t + sign * h * w if i == k else t for i, (t, w) in enumerate(zip(at, way))]
                ends.append((tdc_amd.group_norm_act(p[0], 4, p[1], p[2], act=act).double() * dy.double()).sum().item())
            slope = (ends[0] - ends[1]) / (2 * h)
            want = (grads[k].double() * way[k].double()).sum().item()
            size = (grads[k].double() * way[k].double()).abs().sum().item()
            assert abs(slope - want) <= 1e-3 * size, (act, k, slope, want, size)


def test_norm_gradients_of_other_orders_types_and_subsets():
    x, gamma, beta, dy, y, grads = grad_case((2, 30, 9, 7), 5, F16, "silu", dy_like="nchw")
    check_grads(x, gamma, beta, dy, grads, 5, "silu", "nchw dy")
    # a broadcast dy, parameters of x's type, and each gradient by itself
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        xs = x.detach().requires_grad_(bool(need[0]))
        w = torch.from_numpy(gamma).half().cuda().requires_grad_(bool(need[1]))
        b = torch.from_numpy(beta).half().cuda().requires_grad_(bool(need[2]))
        y = tdc_amd.group_norm_act(xs, 5, w, b, act="silu")
        wrt = [t for t in (xs, w, b) if t.requires_grad]
        got = torch.autograd.grad(y.sum(), wrt)
        every = [t.detach().requires_grad_() for t in (xs, w, b)]
        want = torch.autograd.grad(tdc_amd.group_norm_act(every[0], 5, every[1], every[2], act="silu").sum(), every)
        check_grads(x, w.detach().double().cpu().numpy(), b.detach().double().cpu().numpy(), torch.ones_like(x), want, 5, "silu", "sum")
        for t, gr in zip(wrt, got):
            k = [i for i, s in enumerate((xs, w, b)) if s is t][0]
            assert gr.dtype == t.dtype and torch.equal(gr, want[k])
    # a slice of a wider tensor
    x, gamma, beta = norm_case(9, (2, 40, 6, 6), BF16, wide=64)
    xs = x.detach().requires_grad_()
    dy = torch.randn(2, 40, 6, 6, generator=seeded(3)).bfloat16().cuda()
    grads = torch.autograd.grad(tdc_amd.group_norm_act(xs, 8, act="relu"), xs, dy)
    one = torch.ones(40, device="cuda")
    w, b = one.clone().requires_grad_(), torch.zeros(40, device="cuda", requires_grad=True)
    both = torch.autograd.grad(tdc_amd.group_norm_act(xs, 8, w, b, act="relu"), (xs, w, b), dy)
    check_grads(x, np.ones(40), np.zeros(40), dy, both, 8, "relu", "slice")
    assert torch.equal(grads[0], both[0])


# ---- 4-bit numbers ----

def special_numbers(dtype):
    """Ties of every kind, zeros, subnormal and largest numbers, infinities and NaN, a block each."""
    info = torch.finfo(dtype)
    tie = [0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -0.0, 7.9375, 4.0]
    blocks = [[v * 2.0 ** e for v in tie] for e in (0, 3, -9)]
    blocks += [[0.0] * 32, [-0.0] * 32, [info.max, info.max / 3, -info.max, 1.0], [info.tiny, info.tiny * 3, -info.tiny / 2, info.tiny / 4],
               [info.smallest_normal * 2.0 ** -5, 0.0], [math.inf, 1.0, -2.0], [1.0, math.nan], [-math.inf, math.nan], [2.0 ** -14] * 3 + [1.0]]
    x = torch.zeros(len(blocks), 32, dtype=torch.float64)
    for i, b in enumerate(blocks):
        x[i, :len(b)] = torch.tensor(b, dtype=torch.float64)
    return x.to(dtype)


def check_quantised(q, x, what=""):
    flat = x.detach().double().cpu().numpy().reshape(-1, x.shape[-1])
    codes, byte, values = ref.mx4(flat)
    got_codes, got_byte, pad = ref.mx4_unpack(q.codes.cpu().numpy(), q.scales.cpu().numpy(), x.shape[-1])
    assert np.array_equal(got_byte, byte), what
    plain = np.repeat(byte != 255, 32, axis=1)[:, :x.shape[-1]]
    assert np.array_equal(got_codes[plain], codes[plain]), what
    assert not pad.any(), what
    for dtype in (F32, BF16, x.dtype):
        back = q.dequantize(dtype)
        assert back.shape == x.shape and back.dtype == dtype
        assert np.array_equal(back.double().cpu().numpy().reshape(values.shape), values, equal_nan=True), (what, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantize(dtype):
    x = special_numbers(dtype)
    check_quantised(tdc_amd.mx4_quantize(x.cuda()), x, "specials")
    check_quantised(tdc_amd.mx4_quantize(x.reshape(1, -1).cuda()), x.reshape(1, -1), "specials in a row")
    for rows_, K in ((0, 8), (1, 1), (5, 31), (3, 32), (7, 33), (257, 100), (64, 128), (33, 300), (2, 4096), (1000, 64), (17, 2000)):
        g = seeded(rows_ + K)
        x = (torch.randn(rows_, K, generator=g) * torch.exp2(torch.randint(-12, 12, (rows_, 1), generator=g).float())).to(dtype)
        check_quantised(tdc_amd.mx4_quantize(x.cuda()), x, f"{rows_} x {K}")
    wide = torch.randn(40, 3, 75, generator=seeded(5)).to(dtype).cuda()
    check_quantised(tdc_amd.mx4_quantize(wide), wide, "three axes")
    check_quantised(tdc_amd.mx4_quantize(wide[:, 1, 3:70]), wide[:, 1, 3:70], "a slice")
    check_quantised(tdc_amd.mx4_quantize(wide[:, 1].t()), wide[:, 1].t(), "transposed")
    check_quantised(tdc_amd.mx4_quantize(wide[:1, 0].expand(9, 75)), wide[:1, 0].expand(9, 75), "broadcast rows")


# ---- product ----

def numbers(seed, *shape):
    g = seeded(seed)
    return torch.randn(shape, generator=g) * (1 + 15 * (torch.rand(shape[-1], generator=g) < 0.02))


def check_product(y, x, w, bias, residual, act, what=""):
    """x, w: what the operands stand for, in 64 bits."""
    K = x.shape[-1]
    x = x.reshape(-1, K)
    v, size = x @ w.T, np.abs(x) @ np.abs(w).T
    bound = (16 + K / 64) * E * size
    for t in (bias, residual):
        if t is not None:
            t = t.detach().double().cpu().numpy()
            t = t.reshape(-1, t.shape[-1])
            v, size = v + t, size + np.abs(t)
    want = ref.act(v, act)
    close(y.reshape(want.shape), want, 1.2 * (bound + 8 * E * size) + U[y.dtype] * np.abs(want) + (2.0 ** -25 if y.dtype == F16 else 0), what)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 32), (1, 1000, 2048), (2, 17, 33), (5, 100, 130), (15, 64, 128), (16, 33, 512), (17, 48, 96),
                                   (33, 1001, 2000), (64, 257, 300), (65, 128, 1024), (129, 130, 640), (200, 512, 128), (300, 70, 4100),
                                   (513, 384, 256), (1030, 260, 400), (3, 4096, 5000)])
def test_product(M, N, K, dtype):
    x, w = numbers(1, M, K).to(dtype), numbers(2, N, K) / math.sqrt(K)
    bias, residual = numbers(3, N) * 0.1, numbers(4, M, N).to(dtype)
    wq = tdc_amd.mx4_quantize(w.cuda())
    xv, wv = ref.mx4(x.double().numpy())[2], ref.mx4(w.double().numpy())[2]
    xd = x.cuda()
    check_product(tdc_amd.mx4_linear(xd, wq), xv, wv, None, None, "none", "plain")
    check_product(tdc_amd.mx4_linear(xd, wq, bias.cuda(), residual.cuda(), act="silu"), xv, wv, bias, residual, "silu", "all")
    xq = tdc_amd.mx4_quantize(xd)
    y = tdc_amd.mx4_linear(xq, wq, bias.to(dtype).cuda(), act="relu", out_dtype=dtype)
    check_product(y, xv, wv, bias.to(dtype), None, "relu", "quantised x")
    assert torch.equal(y, tdc_amd.mx4_linear(xq, wq, bias.to(dtype).cuda(), act="relu", out_dtype=dtype))
    assert torch.equal(y, tdc_amd.mx4_linear(xd, wq, bias.to(dtype).cuda(), act="relu"))
    other = BF16 if dtype == F32 else F32
    check_product(tdc_amd.mx4_linear(xd, wq, out_dtype=other), xv, wv, None, None, "none", "another type out")


@pytest.mark.parametrize("dtype,M,N,K", [(F32, 3333, 3850, 420), (F16, 4100, 3590, 128), (BF16, 3328, 4096, 1700), (BF16, 3333, 3850, 4100)])
def test_product_of_many_tiles(dtype, M, N, K):
    x, w = numbers(16, M, K).to(dtype), numbers(17, N, K) / math.sqrt(K)
    bias, residual = numbers(18, N), numbers(19, M, N).to(dtype)
    y = tdc_amd.mx4_linear(x.cuda(), tdc_amd.mx4_quantize(w.cuda()), bias.cuda(), residual.cuda(), act="relu")
    check_product(y, ref.mx4(x.double().numpy())[2], ref.mx4(w.double().numpy())[2], bias, residual, "relu")


def test_product_of_whole_numbers_is_exact():
    g = seeded(21)
    values = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -1, -1.5, -2, -3, -4, -6])
    for M, N, K in ((1, 40, 4096), (50, 70, 384), (260, 300, 1000)):
        x, w = values[torch.randint(0, 15, (M, K), generator=g)], values[torch.randint(0, 15, (N, K), generator=g)]
        x[:, ::32] = 6.0
        w[:, ::32] = 6.0
        y = tdc_amd.mx4_linear(x.cuda(), tdc_amd.mx4_quantize(w.cuda()))
        assert torch.equal(y.cpu().double(), x.double() @ w.double().t())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [(4400, 4500, 4200), (6200, 12400, 4096)])
def test_product_of_more_tiles_than_compute_units_is_exact(dtype, M, N, K):
    """Workgroups that take one tile after the other, the last ones not all of them: sums of quarters, exact in fp32 in any order."""
    g = torch.Generator(device="cuda").manual_seed(23)
    values = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    x, w = (values[torch.randint(0, 15, (n, K), generator=g, device="cuda")] for n in (M, N))
    x[:, ::32] = 6.0
    w[:, ::32] = 6.0
    bias, residual = (torch.randint(-9, 10, n, generator=g, device="cuda").float() for n in ((N,), (M, N)))
    want = torch.relu(x @ w.t() / 64 + bias + residual).to(dtype)
    y = tdc_amd.mx4_linear(x / 64, tdc_amd.mx4_quantize(w), bias, residual.to(dtype), act="relu", out_dtype=dtype)
    assert torch.equal(y, want)


def test_product_strides_axes_and_specials():
    base = numbers(6, 6, 9, 200).cuda()
    x = base[:, :, 20:170]
    w = numbers(7, 44, 150)
    wq = tdc_amd.mx4_quantize(w.cuda())
    residual = numbers(8, 6, 9, 90).cuda()[..., 5:49]
    y = tdc_amd.mx4_linear(x, wq, residual=residual)
    assert y.shape == (6, 9, 44)
    xv, wv = ref.mx4(x.reshape(-1, 150).double().cpu().numpy())[2], ref.mx4(w.double().numpy())[2]
    check_product(y, xv, wv, None, residual, "none", "slices")
    assert tdc_amd.mx4_linear(x[:0], wq).shape == (0, 9, 44)
    # one block without a value, in x and in the weights: its row and its column are lost, nothing else
    x, w = numbers(9, 70, 256), numbers(10, 90, 256)
    clean = tdc_amd.mx4_linear(x.cuda(), tdc_amd.mx4_quantize(w.cuda()))
    x[33, 40], w[57, 200] = math.inf, math.nan
    y = tdc_amd.mx4_linear(x.cuda(), tdc_amd.mx4_quantize(w.cuda()), act="relu")
    assert y[33].isnan().all() and y[:, 57].isnan().all()
    rest = torch.ones(70, 90, dtype=torch.bool, device="cuda")
    rest[33], rest[:, 57] = False, False
    assert torch.equal(y[rest], clean.clamp(min=0)[rest])


def test_conv1x1_is_the_product_over_pixels():
    x = numbers(12, 3, 5, 7, 96).half().cuda().permute(0, 3, 1, 2)
    w, bias = numbers(13, 40, 96) / 10, numbers(14, 40)
    residual = numbers(15, 3, 40, 5, 7).half().cuda()
    wq = tdc_amd.mx4_quantize(w.cuda())
    y = tdc_amd.mx4_conv1x1(x, wq, bias.cuda(), residual, act="silu")
    assert y.shape == (3, 40, 5, 7) and y.is_contiguous(memory_format=torch.channels_last)
    xv, wv = ref.mx4(x.permute(0, 2, 3, 1).reshape(-1, 96).double().cpu().numpy())[2], ref.mx4(w.double().numpy())[2]
    check_product(y.permute(0, 2, 3, 1), xv, wv, bias, residual.permute(0, 2, 3, 1), "silu")


# ---- the norm into 4 bits ----

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", [((1, 1024, 14, 14), 32), ((2, 512, 9, 9), 32), ((3, 114, 13, 7), 6), ((2, 33, 5, 9), 1), ((1, 8, 3, 3), 4),
                                          ((1, 4104, 4, 5), 1), ((1, 8008, 2, 3), 8), ((2, 2064, 3, 3), 16), ((2, 2600, 1, 9), 1300)])
def test_norm_into_4_bits(shape, groups, dtype):
    """A number may come out on either side of a halfway point, and a block's scale on either side of a power of two, that
    its 64-bit value is within the norm's own error of; everything else is what the 64-bit value rounds to."""
    for act in ("none", "relu", "silu"):
        x, gamma, beta = norm_case(51, shape, dtype)
        q = tdc_amd.group_norm_act_mx4(x, groups, gamma.cuda(), beta.cuda(), act=act)
        assert q.shape == (shape[0], *shape[2:], shape[1])
        gamma, beta = gamma.double().numpy(), beta.double().numpy()
        xh, z, mean, rstd = ref.norm_parts(rows(x), groups, gamma, beta, 1e-5)
        C = shape[1]
        err = (16 * E * (np.abs(gamma) * (np.abs(xh) + np.abs(mean) * rstd) + np.abs(beta))).reshape(-1, C)
        want = ref.act(z, act).reshape(-1, C)
        _, byte, values = ref.mx4(want)
        got = q.dequantize(F32).double().cpu().numpy().reshape(-1, C)
        _, got_byte, pad = ref.mx4_unpack(q.codes.cpu().numpy(), q.scales.cpu().numpy(), C)
        assert not pad.any()
        spread = [np.pad(t, ((0, 0), (0, -C % 32))).reshape(len(t), -1, 32).max(axis=2) for t in (np.abs(want), err)]
        moved = got_byte != byte
        edge = np.ldexp(1.0, np.maximum(got_byte, byte).astype(int) - 127 + 2)      # the power of two between the two scales
        assert (np.abs(spread[0] - edge)[moved] <= spread[1][moved]).all()
        scale = np.repeat(np.ldexp(1.0, got_byte.astype(int) - 127), 32, axis=1)[:, :C]
        size = np.minimum(np.abs(want) / scale, 6.0)
        nearest = np.abs(size[..., None] - ref.GRID).min(axis=-1) * scale
        off = np.abs(got - np.clip(want, -6 * scale, 6 * scale))
        assert (off <= nearest + 2 * err).all()


# ---- streams, graphs ----

def pipeline(x, gamma, beta, wq, bias, residual):
    h = tdc_amd.group_norm_act_mx4(x, 8, gamma, beta, act="silu")
    y = tdc_amd.mx4_conv1x1(h, wq, bias, residual, out_dtype=x.dtype)
    z = tdc_amd.mx4_linear(tdc_amd.group_norm_act(y, 4, act="relu").permute(0, 2, 3, 1), wq[1] if isinstance(wq, tuple) else wq)
    return y, z


def test_streams_and_graphs():
    """Same results on a side stream, and from every replay of a captured graph with eager work and new inputs between."""
    x, gamma, beta = norm_case(61, (2, 64, 12, 11), BF16)
    gamma, beta = gamma.cuda(), beta.cuda()
    wq, bias = tdc_amd.mx4_quantize(numbers(62, 64, 64).cuda()), numbers(63, 64).cuda()
    residual = numbers(64, 2, 12, 11, 64).bfloat16().cuda().permute(0, 3, 1, 2)
    want = pipeline(x, gamma, beta, wq, bias, residual)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = pipeline(x, gamma, beta, wq, bias, residual)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            held = pipeline(x, gamma, beta, wq, bias, residual)
    for rep in range(4):
        x.copy_(norm_case(70 + rep, (2, 64, 12, 11), BF16)[0])
        want = pipeline(x, gamma, beta, wq, bias, residual)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), rep


def test_backward_from_a_graph():
    x, gamma, beta = norm_case(81, (3, 48, 10, 10), F32)
    w, b = gamma.cuda().requires_grad_(), beta.cuda().requires_grad_()
    x.requires_grad_()
    dy = torch.randn(3, 48, 10, 10, generator=seeded(1)).cuda().contiguous(memory_format=torch.channels_last)

    def step():
        return torch.autograd.grad(tdc_amd.group_norm_act(x, 6, w, b, act="silu"), (x, w, b), dy)

    step()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            held = step()
    for rep in range(3):
        with torch.no_grad():
            x.copy_(norm_case(90 + rep, (3, 48, 10, 10), F32)[0])
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, held)), rep


def test_offsets_beyond_32_bits():
    """More than 2^31 elements between the first image and the last: a slice of a wide buffer, and rows of the product."""
    buf = torch.zeros(3, 4, 4, (1 << 26) + 8, dtype=F16, device="cuda")      # 2^30 elements an image
    x = buf[..., (1 << 26) - 32:(1 << 26)].permute(0, 3, 1, 2)
    x.copy_(norm_case(5, (3, 32, 4, 4), F16)[0])
    y = tdc_amd.group_norm_act(x, 4)
    check_forward(y, x, 4, np.ones(32), np.zeros(32), "none")
    flat = x.permute(0, 2, 3, 1).select(1, 3).select(1, 3)      # [3, 32], rows 2^30 apart
    wq = tdc_amd.mx4_quantize(torch.eye(32, device="cuda"))
    got = tdc_amd.mx4_linear(flat, wq)
    assert np.array_equal(got.double().cpu().numpy(), ref.mx4(flat.double().cpu().numpy())[2])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", [((2, 264, 50, 14), 8), ((1, 944, 22, 17), 16), ((3, 40, 70, 31), 5), ((5, 36, 9, 9), 3), ((70, 72, 6, 6), 9),
                                          ((1, 2056, 40, 3), 8), ((2, 24, 1, 1), 1), ((9, 296, 61, 61), 37)])
def test_norm_into_4_bits_where_the_last_block_is_not_full(shape, groups, dtype):
    test_norm_into_4_bits(shape, groups, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_norm_into_4_bits_takes_nothing_from_beside_its_channels(dtype):
    for B, C, S, groups in ((2, 40, 9, 5), (1, 72, 3000, 9), (1, 72, 800, 9)):
        x = numbers(61, B, S, C).to(dtype).cuda()
        wide = torch.full((B, S, C + 56), float("nan"), dtype=dtype, device="cuda")
        wide[..., 24:24 + C] = x
        want, got = (tdc_amd.group_norm_act_mx4(t.permute(0, 2, 1), groups, act="silu") for t in (x, wide[..., 24:24 + C]))
        assert torch.equal(want.dequantize(), got.dequantize()) and torch.equal(want.scales, got.scales)     # (codes past the last row are anything)
        assert got.dequantize().isfinite().all()


@pytest.mark.parametrize("shape,groups,dtype", [((1, 4, 1100, 1000), 2, F32), ((1, 24, 700, 500), 3, BF16)])
def test_norm_of_one_image_of_many_pixels(shape, groups, dtype):
    test_norm_forward(shape, groups, dtype)
    test_norm_gradients(shape, groups, dtype)


# ---- together ----

def test_tucker_block_in_4_bits():
    """The block is its operators one after the other, and near the same block in 32 bits: each of its two products is off by what
    rounding both operands to 4 bits costs (some 0.1 an operand), which the residual does not share."""
    torch.manual_seed(3)
    conv = tdc_amd.TKConv2dC(96, 96, 3, padding=1, hp_dict=tdc_amd.ranks_dict(conv=[40, 32]), name="conv")
    block = tdc_amd.TuckerBlockMx4(conv, groups=8, rank_groups=5).cuda()
    with torch.no_grad():
        block.norm_in.weight.add_(torch.randn(96, device="cuda") * 0.2)
        block.norm_core.bias.add_(torch.randn(40, device="cuda") * 0.2)
    x = torch.randn(3, 14, 13, 96, generator=seeded(5)).bfloat16().cuda().permute(0, 3, 1, 2)
    first0, core0, last0 = (p.detach().clone() for p in (conv.first_kernel, conv.core_kernel, conv.last_kernel))
    y = block(x)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous(memory_format=torch.channels_last)
    n, m = block.norm_in, block.norm_core
    h = tdc_amd.mx4_conv1x1(tdc_amd.group_norm_act_mx4(x, 8, n.weight, n.bias, act="silu"), tdc_amd.mx4_quantize(conv.first_kernel.detach().flatten(1)),
                            out_dtype=F32)
    plan = tdc_amd.Conv2dPlan(3, 32, 40, 14, 13, 3, 3, 1, 1).set_weights(conv.core_kernel)
    h = plan.forward(h.contiguous()).contiguous(memory_format=torch.channels_last)
    want = tdc_amd.mx4_conv1x1(tdc_amd.group_norm_act_mx4(h, 5, m.weight, m.bias, act="silu"), tdc_amd.mx4_quantize(conv.last_kernel.detach().flatten(1)),
                               conv.bias.detach(), x, out_dtype=BF16)
    plan.close()
    assert torch.equal(y, want) and torch.equal(y, block(x))
    with torch.no_grad():
        conv.last_kernel.zero_()
    assert torch.equal(block(x), (x.float() + conv.bias.view(1, -1, 1, 1)).to(BF16))     # 0 for the product, after the change
    conv.load_kernels(first0, core0, last0)
    assert torch.equal(y, block(x))
    plain = block.plain(x)
    assert torch.linalg.norm(y.float() - plain) < 0.4 * torch.linalg.norm(plain - x.float())
    with pytest.raises(ValueError, match="keep its input's size"):
        tdc_amd.TuckerBlockMx4(tdc_amd.TKConv2dC(8, 8, 3, hp_dict=tdc_amd.ranks_dict(conv=[4, 4]), name="conv"))


def test_norm_module_trains():
    """A few steps of gradient descent through the module: the loss falls as it does in 64 bits on the host, step by step."""
    g = seeded(9)
    x, target = torch.randn(4, 24, 6, 6, generator=g), torch.randn(4, 24, 6, 6, generator=g)
    norm = tdc_amd.GroupNormAct(6, 24, act="silu").cuda()
    w, b = torch.ones(24, dtype=torch.float64, requires_grad=True), torch.zeros(24, dtype=torch.float64, requires_grad=True)
    xd = x.cuda().contiguous(memory_format=torch.channels_last)
    for step in range(5):
        loss = ((norm(xd) - target.cuda()) ** 2).mean()
        plain = ((torch.nn.functional.silu(torch.nn.functional.group_norm(x.double(), 6, w, b)) - target.double()) ** 2).mean()
        assert abs(loss.item() - plain.item()) < 1e-5 * plain.item(), step
        grads, want = torch.autograd.grad(loss, (norm.weight, norm.bias)), torch.autograd.grad(plain, (w, b))
        with torch.no_grad():
            for p, d in ((norm.weight, grads[0]), (norm.bias, grads[1]), (w, want[0]), (b, want[1])):
                p -= 20 * d


# ---- sums that meet large and small numbers ----

def check_forward_on_device(y, x, groups, what):
    """check_forward without parameters, for tensors that are long work for the host, which only adds up the statistics (torch's
    reductions of many numbers to few, on the device, are not always right)."""
    B, C = x.shape[:2]
    for b in range(B):
        v, got = (t[b].permute(1, 2, 0).reshape(-1, groups, C // groups).double() for t in (x, y))
        host = v.cpu().numpy()
        mean = host.mean(axis=(0, 2), keepdims=True)
        rstd = 1 / np.sqrt(((host - mean) ** 2).mean(axis=(0, 2), keepdims=True) + 1e-5)
        mean, rstd = torch.from_numpy(mean).cuda(), torch.from_numpy(rstd).cuda()
        want = (v - mean) * rstd
        bound = E * want.abs() + 16 * E * (want.abs() + mean.abs() * rstd)
        far = ((got - want).abs() / bound.clamp(min=1e-300)).amax(dim=2).cpu().numpy().max()
        assert far <= 1, (what, b, far)


@pytest.mark.parametrize("shape,groups", [((1, 128, 112, 112), 32), ((1, 3, 1460, 1460), 1), ((1, 4, 2535, 2535), 2), ((1, 1, 5800, 5800), 1),
                                          ((8, 16, 1024, 1024), 4)])
def test_norm_of_images_that_begin_with_outliers(shape, groups):
    """The first number of a thread holds nearly all of its variance: fp32, two launches, 4 (the first shape) to 256 pixels a thread."""
    B, C, H, W = shape
    g = torch.Generator(device="cuda").manual_seed(71)
    for what in ("impulse", "a few among small ones", "another first row"):
        x = torch.zeros(B, H, W, C, device="cuda")
        if what == "impulse":
            x[:, 0, 0] = 1 + 3 * torch.rand(B, C, generator=g, device="cuda")
        elif what == "another first row":
            x += 0.3
            x[:, 0] = 40.0
        else:
            x.normal_(generator=g).mul_(0.05)
            x.view(B, -1, C)[:, :300] += 1 + 3 * torch.rand(B, 300, C, generator=g, device="cuda")
        x = x.permute(0, 3, 1, 2)
        check_forward_on_device(tdc_amd.group_norm_act(x, groups), x, groups, what)


@pytest.mark.parametrize("S", [896 * 896, 2048 * 2048])
def test_norm_into_4_bits_of_an_image_that_begins_with_an_outlier(S):
    """Numbers that lie 1e-5 of themselves from halfway between two codes, ten times their fp32 error, take the code of their side."""
    C, big = 32, float(np.float32(2.7))      # (its square is not exact in fp32)
    x = torch.zeros(1, S, C, device="cuda")
    x[:, 0] = big
    mean = big / S
    rstd = 1 / math.sqrt(big * mean - mean * mean + 1e-5)
    first = (big - mean) * rstd
    gamma = np.full(C, 2.5 / first)
    beta = np.where(np.arange(C) % 2 == 0, -2.5e-5, 2.5e-5)
    gamma[0], beta[0] = 6.0 / first, 0.0      # (the block's scale is 1)
    gamma, beta = torch.from_numpy(gamma).float(), torch.from_numpy(beta).float()
    z = first * gamma.double().numpy() + beta.double().numpy()
    assert np.abs(z[1:] - 2.5).min() > 2e-5
    q = tdc_amd.group_norm_act_mx4(x.permute(0, 2, 1), 1, gamma.cuda(), beta.cuda())
    got = q.dequantize()[0, 0].double().cpu().numpy()
    assert np.array_equal(got, ref.mx4(z[None])[2][0])


@pytest.mark.parametrize("shape,groups", [((1 << 20, 16), 2), ((300001, 3, 2, 1), 1), ((1, 1, 1500, 1500), 1)])
def test_norm_gradients_of_many_rows_with_one_slope(shape, groups):
    """dy as a mean's backward gives it, the same everywhere: every step of a long fp32 sum of it is rounded the same way."""
    g = torch.Generator(device="cuda").manual_seed(73)
    B, C, *space = shape
    x = torch.randn(B, *space, C, generator=g, device="cuda").movedim(-1, 1)
    gamma, beta = torch.rand(C, generator=g, device="cuda") + 0.5, torch.randn(C, generator=g, device="cuda")
    for act in ("none", "silu"):
        leaves = [t.detach().requires_grad_() for t in (x, gamma, beta)]
        dy = torch.full((), 0.3, device="cuda").expand(shape)
        grads = torch.autograd.grad(tdc_amd.group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act), leaves, dy)
        check_grads(x, gamma.double().cpu().numpy(), beta.double().cpu().numpy(), dy, grads, groups, act, f"{shape} {act}")


# ---- derivatives that the operators do not have ----

def test_4_bit_operators_refuse_what_wants_a_gradient():
    """None of them drops a gradient without a word: whatever would have to get one is refused, and taken under no_grad."""
    x = torch.randn(2, 64, 3, 4, device="cuda").contiguous(memory_format=torch.channels_last)
    wq = tdc_amd.mx4_quantize(torch.randn(64, 64, device="cuda"))
    bias, xq = torch.randn(64, device="cuda"), tdc_amd.group_norm_act_mx4(x, 4)
    norm = tdc_amd.GroupNormAct(4, 64).cuda()

    def wanting(t):
        return t.detach().clone(memory_format=torch.preserve_format).requires_grad_()

    calls = {
        "x": lambda: tdc_amd.mx4_conv1x1(wanting(x), wq),
        "bias": lambda: tdc_amd.mx4_conv1x1(x, wq, wanting(bias)),
        "residual": lambda: tdc_amd.mx4_conv1x1(xq, wq, bias, wanting(x), out_dtype=F32),
        "residual with a history": lambda: tdc_amd.mx4_conv1x1(xq, wq, None, wanting(x) * 2, out_dtype=F32),
        "residual of rows": lambda: tdc_amd.mx4_linear(torch.randn(3, 64, device="cuda"), wq, residual=wanting(torch.randn(3, 64, device="cuda"))),
        "quantised": lambda: tdc_amd.mx4_quantize(wanting(x)),
        "norm into 4 bits": lambda: tdc_amd.group_norm_act_mx4(wanting(x), 4),
        "the module's parameters": lambda: norm.mx4(x),
    }
    for what, call in calls.items():
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
            pytest.fail(what)
        with torch.no_grad():
            call()
    # as an argument of the function they are taken as numbers, with a warning
    with pytest.warns(UserWarning, match="no gradient"):
        q = tdc_amd.group_norm_act_mx4(x, 4, norm.weight, norm.bias)
    with torch.no_grad():
        assert torch.equal(q.dequantize(), norm.mx4(x).dequantize())


def test_tangents_are_refused():
    """Forward mode: a dual tensor need not require a gradient, and its tangent would be lost."""
    from torch.autograd import forward_ad
    x = torch.randn(2, 64, 3, 4, device="cuda").contiguous(memory_format=torch.channels_last)
    w = torch.ones(64, device="cuda")
    wq = tdc_amd.mx4_quantize(torch.randn(64, 64, device="cuda"))
    residual = torch.randn(2, 64, 3, 4, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: tdc_amd.group_norm_act(dual, 4), lambda: tdc_amd.group_norm_act(x, 4, forward_ad.make_dual(w, w)),
                     lambda: tdc_amd.group_norm_act(x, 4, None, forward_ad.make_dual(w, w)), lambda: tdc_amd.group_norm_act_mx4(dual, 4),
                     lambda: tdc_amd.mx4_quantize(dual), lambda: tdc_amd.mx4_conv1x1(dual, wq),
                     lambda: tdc_amd.mx4_conv1x1(x, wq, None, forward_ad.make_dual(residual, residual))):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
        want = tdc_amd.group_norm_act(x, 4, w)
    assert torch.equal(want, tdc_amd.group_norm_act(x, 4, w))
    leaf = x.detach().requires_grad_()
    y = tdc_amd.group_norm_act(leaf, 4)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_copies_of_a_4_bit_tensor():
    import copy
    import io
    x = numbers(91, 5, 70, 300).cuda()
    q = tdc_amd.mx4_quantize(x)
    file = io.BytesIO()
    torch.save(q, file)
    file.seek(0)
    copies = [copy.deepcopy(q), torch.load(file, weights_only=False), copy.copy(q)]
    want = q.dequantize()
    del q
    torch.full((1 << 20,), 7.0, device="cuda")      # (what the original held may be another's by now)
    for other in copies:
        assert torch.equal(other.dequantize(), want)
    file.seek(0)
    away = torch.load(file, map_location="cpu", weights_only=False)
    with pytest.raises(ValueError):
        away.dequantize()
    with pytest.raises(ValueError):
        tdc_amd.mx4_linear(away, tdc_amd.mx4_quantize(torch.ones(4, 300, device="cuda")))


def test_tucker_block_on_streams_and_in_a_graph():
    """Same results on two streams in turn, nothing between, after the weights have changed, and from a graph captured on a stream that the block has not seen."""
    torch.manual_seed(4)
    conv = tdc_amd.TKConv2dC(96, 96, 3, padding=1, hp_dict=tdc_amd.ranks_dict(conv=[40, 32]), name="conv")
    block = tdc_amd.TuckerBlockMx4(conv, groups=8, rank_groups=5).cuda()
    xs = [torch.randn(4, 28, 28, 96, device="cuda").bfloat16().permute(0, 3, 1, 2) for _ in range(6)]
    sides = torch.cuda.Stream(), torch.cuda.Stream()
    for change in range(2):
        with torch.no_grad():
            conv.first_kernel.mul_(1.5)
        torch.cuda.synchronize()
        got = []
        for i, x in enumerate(xs):
            with torch.cuda.stream(sides[i % 2]):
                got.append(block(x))
        torch.cuda.synchronize()
        assert all(torch.equal(y, block(x)) for x, y in zip(xs, got)), change
    graph, x = torch.cuda.CUDAGraph(), xs[0].clone(memory_format=torch.channels_last)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = block(x)
    for rep in range(4):
        x.copy_(xs[rep + 1])
        want = block(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want), rep


# ---- arguments ----

def test_norm_parameters_of_other_types_are_refused_by_name():
    x = torch.randn(2, 8, 3, 3, device="cuda").contiguous(memory_format=torch.channels_last)
    w = torch.ones(8, device="cuda")
    for call in (tdc_amd.group_norm_act, tdc_amd.group_norm_act_mx4):
        for bad in (w.double(), w.int()):
            with pytest.raises(TypeError, match="weight has to be float32"):
                call(x, 2, bad)
            with pytest.raises(TypeError, match="bias has to be float32"):
                call(x, 2, None, bad)
        with pytest.raises(ValueError, match="weight must be a tensor"):
            call(x, 2, [1.0] * 8)
        with pytest.raises(ValueError, match="bias must be a tensor"):
            call(x, 2, w, 1.0)
        with pytest.raises(ValueError, match="weight must be a tensor"):
            call(x, 2, w.cpu())


def test_product_with_no_outputs_or_no_rows():
    none, some = tdc_amd.mx4_quantize(torch.empty(0, 64, device="cuda")), tdc_amd.mx4_quantize(torch.ones(5, 64, device="cuda"))
    for lead in ((2, 3), (0, 3), (4,), ()):
        x = torch.ones(*lead, 64, device="cuda")
        for w, N in ((none, 0), (some, 5)):
            for residual in (None, torch.ones(*lead, N, device="cuda")):
                y = tdc_amd.mx4_linear(x, w, torch.ones(N, device="cuda"), residual)
                assert y.shape == (*lead, N)
                assert bool((y == 65 + (residual is not None)).all())
    x = torch.ones(2, 64, 3, 3, device="cuda").contiguous(memory_format=torch.channels_last)
    assert tdc_amd.mx4_conv1x1(x, none, residual=torch.ones(2, 0, 3, 3, device="cuda")).shape == (2, 0, 3, 3)


# ---- what only the C entries have ----

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", [((2, 64, 9, 9), 8), ((3, 48, 70, 90), 4), ((2, 33, 5, 9), 1), ((1, 4104, 40, 5), 1), ((1, 2600, 1, 9), 1300)])
def test_norm_into_a_slice_and_its_statistics(shape, groups, dtype):
    """y with strides of its own (nothing beside it is touched), mean and rstd as the entry returns them: off by some ten roundings of what
    they come from."""
    from tdc_amd import _lib
    x, gamma, beta = norm_case(93, shape, dtype)
    B, C, pixels = shape[0], shape[1], math.prod(shape[2:])
    wide = torch.full((B, pixels + 2, C + 5), -7.0, dtype=dtype, device="cuda")
    y = wide[:, 1:1 + pixels, 3:3 + C]
    kind = {F32: 0, F16: 1, BF16: 2}[dtype]
    desc = _lib.GroupNormDesc(B, C, groups, 2, kind, 0, 1e-5, 0, pixels, 0, 0, y.stride(1), y.stride(0))
    need = ctypes.c_size_t()
    assert tdc_amd.lib().tdc_group_norm_workspace(ctypes.byref(desc), ctypes.byref(need), None) == 0
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    stats = torch.full((2, B, groups), float("nan"), device="cuda")
    gd, bd = gamma.cuda(), beta.cuda()
    assert tdc_amd.lib().tdc_group_norm_forward(ctypes.byref(desc), x.data_ptr(), gd.data_ptr(), bd.data_ptr(), y.data_ptr(), stats[0].data_ptr(),
                                                stats[1].data_ptr(), ws.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream) == 0
    check_forward(y.permute(0, 2, 1), x.reshape(B, C, pixels), groups, gamma.double().numpy(), beta.double().numpy(), "silu")
    beside = torch.ones_like(wide, dtype=torch.bool)
    beside[:, 1:1 + pixels, 3:3 + C] = False
    assert bool((wide[beside] == -7.0).all())
    v = rows(x).reshape(B, pixels, groups, C // groups)
    mean, var = v.mean(axis=(1, 3)), v.var(axis=(1, 3))
    got = stats.double().cpu().numpy()
    rstd = 1 / np.sqrt(var + 1e-5)
    assert (np.abs(got[0] - mean) <= E * np.abs(mean) + 1e-12 * np.abs(v).max()).all()
    assert (np.abs(got[1] / rstd - 1) <= 10 * E).all()


def test_relu_gradient_of_infinities():
    """An infinite gradient where the result is 0 is as any other there."""
    x = torch.randn(2, 24, 5, 7, generator=seeded(900)).cuda().contiguous(memory_format=torch.channels_last)
    dy = torch.randn(2, 24, 5, 7, generator=seeded(901)).cuda().contiguous(memory_format=torch.channels_last)
    w, b = torch.rand(24, generator=seeded(902)).cuda() + 0.5, torch.randn(24, generator=seeded(903)).cuda()
    wrt = [t.requires_grad_() for t in (x, w, b)]
    y = tdc_amd.group_norm_act(x, 4, w, b, act="relu")
    off = (y == 0) & (torch.arange(7, device="cuda") % 2 == 0)
    assert off.any()
    got = [torch.autograd.grad(tdc_amd.group_norm_act(x, 4, w, b, act="relu"), wrt, dy.masked_fill(off, v)) for v in (float("inf"), 1.0)]
    assert all(torch.isfinite(g).all() and torch.equal(g, v) for g, v in zip(*got))
