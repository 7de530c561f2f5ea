"""The 16- and 8-bit products, RMS norm, their gradients and checkpoints, against plain 64-bit forms.

Tolerances, from the arithmetic.  u is the unit roundoff of the output's type (2^-24, 2^-11, 2^-8), e = 2^-24, S the sum of the
magnitudes of a sum's terms.
16-bit product: an instruction adds 16 exact products to a sum and rounds within 2 e of the magnitudes met, bias, residual and
activation are a few operations more: (16 + K / 8) e S, then u |y|.
8-bit product: an instruction keeps of each of its 64 products what lies above 2^-14 of the largest: 64 2^-14 times that for each 64
numbers, besides the above.
Its gradient: dz = dy act'(z) is rounded (u |dz|), z for "silu" too, and |act''| is at most 1/2: u |dz| + |dy| (u |z| + the product's error) / 2;
"relu" has either slope where z is within its error of 0.  That error goes through dx = dz w and dw = dz^T x term by term, which add their own.
dbias adds in chains of at most 256: 512 e S.
RMS norm: a row's squares add in chains of at most 32 and trees, 1 / sqrt is good to 2 e: 64 e |y|, then u |y|; its gradient the same of the
magnitudes of its terms; the weight's gradient adds in chains of at most 256: 512 e S.
Half precision has 2^-25 more wherever it rounds."""
import ctypes

import numpy as np
import pytest
import torch

import tdc_amd
from oracle import pointwise_ref as ref
from oracle.channels_last_ref import act as ref_act
from util import seeded

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
LEAST = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def host(t):
    return t.detach().double().cpu().numpy()


def close(got, want, bound, what=""):
    got = host(got) if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((np.abs(got - want) <= bound) | (np.isnan(got) & np.isnan(want)) | (got == want))
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.nan_to_num(np.abs(got - want), nan=1e300), 0)), got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside; at {i} got {got[i]!r} want {want[i]!r} bound {np.broadcast_to(bound, got.shape)[i]:.3g}")


def rounded(want, dtype):
    return U[dtype] * np.abs(want) + LEAST[dtype]


def numbers(seed, shape, dtype, by=1.0):
    return (torch.randn(shape, generator=seeded(seed)) * by).to(dtype).cuda()


def case(seed, M, N, K, dtype, bias=True, residual=True, bias_dtype=None):
    x, w = numbers(seed, (M, K), dtype), numbers(seed + 1, (N, K), dtype, K ** -0.5)
    b = numbers(seed + 2, (N,), bias_dtype or dtype) if bias else None
    return x, w, b, numbers(seed + 3, (M, N), dtype) if residual else None


def opt(t):
    return None if t is None else host(t)


def check_linear(y, x, w, b, r, act, dtype, what=""):
    """(z, bound of its error)"""
    z, want = ref.linear(host(x), host(w), opt(b), opt(r), act)
    S = np.abs(host(x)) @ np.abs(host(w)).T + (0 if b is None else np.abs(host(b))) + (0 if r is None else np.abs(host(r)))
    off = (16 + x.shape[1] / 8) * E * S
    close(y, want, 1.1 * off + rounded(want, dtype) * (1 + 1e-3), what)      # (the slope of "silu" is at most 1.1)
    return z, off


PRODUCTS = [(1, 1, 1), (1, 16, 32), (1, 1000, 2048), (2, 17, 33), (5, 100, 130), (15, 64, 128), (16, 33, 512), (31, 129, 72), (33, 256, 96),
            (64, 40, 1000), (100, 300, 31), (129, 127, 257), (130, 258, 640), (257, 128, 4100), (300, 1001, 203), (1000, 24, 64)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear(M, N, K, dtype):
    for i, act in enumerate(("none", "relu", "silu")):
        x, w, b, r = case(10 * i, M, N, K, dtype, bias=i != 1, residual=i != 2, bias_dtype=F32 if i == 2 else dtype)
        y = tdc_amd.linear_act(x, w, b, r, act=act)
        assert y.dtype == dtype and y.shape == (M, N)
        check_linear(y, x, w, b, r, act, dtype, f"{M} {N} {K} {act}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", [(3400, 3500, 2200), (4096, 3336, 2048), (3333, 3850, 128), (40, 40, 40000), (20000, 64, 256)])
def test_linear_of_whole_numbers_is_exact(M, N, K, dtype):
    """Of many tiles, and of sums in parts: sums below 2^8 in magnitude are exact in either type."""
    g = seeded(5)
    x = torch.zeros(M, K)
    x.scatter_(1, torch.randint(0, K, (M, 20), generator=g), torch.randint(-3, 4, (M, 20), generator=g).float())
    w = torch.randint(-4, 5, (N, K), generator=g).float()
    r = torch.randint(-8, 9, (M, N), generator=g).float()
    y = tdc_amd.linear_act(x.to(dtype).cuda(), w.to(dtype).cuda(), None, r.to(dtype).cuda())
    want = x.cuda() @ w.t().contiguous().cuda() + r.cuda()      # (whole numbers: exact in fp32)
    assert torch.equal(y.float(), want)


def grads(out, wrt, dout):
    return torch.autograd.grad(out, wrt, dout)


def check_grads(M, N, K, dtype, act, checkpoint=None, bias_dtype=None, seed=50, residual=True):
    x, w, b, r = case(seed, M, N, K, dtype, residual=residual, bias_dtype=bias_dtype)
    dy = numbers(seed + 9, (M, N), dtype)
    wrt = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    y = tdc_amd.linear_act(x, w, b, r, act=act, checkpoint=checkpoint)
    got = grads(y, wrt, dy)
    what = f"{M} {N} {K} {act} {checkpoint}"
    z, off = check_linear(y, x, w, b, r, act, dtype, what)
    kept = ref.quantize8(host(x))[0] if checkpoint else host(x)
    dz, dx, dw, db = ref.linear_grads(host(x), host(w), z, host(dy), act, kept)
    a = np.abs(host(dy))
    slope = 0 if act == "none" else np.where(np.abs(z) <= off, a, 0) if act == "relu" else a * (rounded(z, dtype) + off) / 2 * 1.01 + 32 * E * a
    if act == "relu" and dtype == F16:
        slope = np.where(np.abs(z) <= off + LEAST[F16], a, 0)      # (what is kept is the rounded result)
    # (dz's rounding is of what the kernel has before it; its own gradient may come as dy itself)
    ez = np.broadcast_to(slope + (0 if act == "none" else rounded(np.abs(dz) + slope, dtype)), dz.shape)
    own = lambda L, S: (16 + L / 8) * E * S  # noqa: E731
    adz = np.abs(dz) + ez
    close(got[0], dx, ez @ np.abs(host(w)) + own(N, adz @ np.abs(host(w))) + rounded(np.abs(dx) + ez @ np.abs(host(w)), dtype), what + " dx")
    S = ez.T @ np.abs(kept)
    close(got[1], dw, S + own(M, adz.T @ np.abs(kept)) + rounded(np.abs(dw) + S, dtype), what + " dw")
    S = np.broadcast_to(slope, dz.shape).sum(0)
    close(got[2], db, S + 512 * E * adz.sum(0) + rounded(np.abs(db) + S, b.dtype), what + " dbias")
    if residual:
        close(got[3], dz, ez, what + " dresidual")
    for t, g in zip(wrt, got):
        assert g.shape == t.shape and g.dtype == t.dtype


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear_gradients(M, N, K, dtype):
    check_grads(M, N, K, dtype, "silu")
    check_grads(M, N, K, dtype, "none", checkpoint="mx8", bias_dtype=F32)
    check_grads(M, N, K, dtype, "relu", residual=False)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", [(5000, 96, 160), (2100, 1030, 1100), (9000, 33, 40)])
def test_linear_gradients_of_many_rows(M, N, K, dtype):
    check_grads(M, N, K, dtype, "silu", checkpoint="mx8")
    check_grads(M, N, K, dtype, "none")


def test_linear_gradients_by_differences():
    """The gradient against differences of the forward pass along a direction (in 64 bits of the sums that the outputs make)."""
    M, N, K = 40, 24, 56
    x, w, b, r = case(70, M, N, K, BF16)
    dy = numbers(71, (M, N), BF16)
    wrt = [t.requires_grad_() for t in (x, w, b, r)]
    got = grads(tdc_amd.linear_act(x, w, b, r, act="silu"), wrt, dy)
    f = lambda *v: float((ref.linear(*v, "silu")[1] * host(dy)).sum())  # noqa: E731
    at = [host(t) for t in wrt]
    for i, g in enumerate(got):
        d = np.random.default_rng(i).standard_normal(at[i].shape)
        step = [a + (1e-5 * d if j == i else 0) for j, a in enumerate(at)]
        back = [a - (1e-5 * d if j == i else 0) for j, a in enumerate(at)]
        slope = (f(*step) - f(*back)) / 2e-5
        # every number of a gradient carries some 2 u of its terms' magnitudes, in random directions
        assert abs((host(g) * d).sum() - slope) <= 8 * U[BF16] * np.sqrt(((np.abs(host(g)) + 1) ** 2 * d ** 2).sum()) + 1e-6 * abs(slope)


def test_linear_strides_axes_and_specials():
    wide = numbers(80, (6, 9, 200), BF16)
    w = numbers(81, (50, 96), BF16)
    for x in (wide[..., 8:104], wide[..., 3:99], wide[:, ::2, 40:136], wide[:, :, 10:106].transpose(0, 1), wide[:1, :1, 1:97].expand(4, 3, 96)):
        y = tdc_amd.linear_act(x, w)
        assert torch.equal(y, tdc_amd.linear_act(x.clone(memory_format=torch.contiguous_format), w)) and y.shape == (*x.shape[:-1], 50)
    big = numbers(82, (50, 300), BF16)
    for v in (big[:, 5:101], big[:, 16:112], big[::2, 8:104]):
        assert torch.equal(tdc_amd.linear_act(wide[0, :, 8:104], v), tdc_amd.linear_act(wide[0, :, 8:104], v.contiguous()))
    r = numbers(83, (6, 9, 51), BF16)
    assert torch.equal(tdc_amd.linear_act(wide[..., :96], w, None, r[..., 1:]), tdc_amd.linear_act(wide[..., :96], w, None, r[..., 1:].contiguous()))
    # what is beside an operand does not come in, what is in it stays in its row and column
    hot = torch.full((20, 300), float("nan"), dtype=BF16, device="cuda")
    hot[:, 100:140] = 1
    assert torch.equal(tdc_amd.linear_act(hot[:, 100:140], torch.ones(9, 40, dtype=BF16, device="cuda")), torch.full((20, 9), 40.0, dtype=BF16, device="cuda"))
    x = numbers(84, (70, 40), BF16)
    want = tdc_amd.linear_act(x, w[:, :40].contiguous())
    for v in (float("nan"), float("inf")):
        y = x.clone()
        y[33, 7] = v
        y = tdc_amd.linear_act(y, w[:, :40].contiguous())
        assert torch.equal(y[:33], want[:33]) and torch.equal(y[34:], want[34:]) and not torch.isfinite(y[33]).any()


def test_conv1x1_is_the_product_over_pixels():
    x = numbers(90, (3, 48, 5, 7), BF16).contiguous(memory_format=torch.channels_last)
    w, r = numbers(91, (20, 48, 1, 1), BF16), numbers(92, (3, 20, 5, 7), BF16).contiguous(memory_format=torch.channels_last)
    y = tdc_amd.conv1x1_act(x, w, None, r, act="relu")
    flat = tdc_amd.linear_act(x.permute(0, 2, 3, 1), w.flatten(1), None, r.permute(0, 2, 3, 1), act="relu")
    assert y.is_contiguous(memory_format=torch.channels_last) and torch.equal(y.permute(0, 2, 3, 1), flat)
    wrt = [t.requires_grad_() for t in (x, w, r)]
    dy = numbers(93, (3, 20, 5, 7), BF16).contiguous(memory_format=torch.channels_last)
    got = grads(tdc_amd.conv1x1_act(x, w, None, r, act="silu"), wrt, dy)
    want = grads(tdc_amd.linear_act(x.permute(0, 2, 3, 1), w.flatten(1), None, r.permute(0, 2, 3, 1), act="silu"), wrt, dy.permute(0, 2, 3, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[1].shape == w.shape
    h = tdc_amd.mx8_conv1x1(x.detach(), tdc_amd.mx8_quantize(w.detach().flatten(1)))
    assert torch.equal(h.permute(0, 2, 3, 1), tdc_amd.mx8_linear(x.detach().permute(0, 2, 3, 1), tdc_amd.mx8_quantize(w.detach().flatten(1))))


def test_linear_of_nothing():
    x, w, b, r = case(95, 0, 10, 24, BF16)
    wrt = [t.requires_grad_() for t in (x, w, b, r)]
    for checkpoint in (None, "mx8"):
        y = tdc_amd.linear_act(x, w, b, r, act="silu", checkpoint=checkpoint)
        dx, dw, db, dr = grads(y, wrt, torch.empty_like(y))
        assert y.shape == (0, 10) and dx.shape == x.shape and not dw.any() and not db.any() and dr.shape == r.shape
    x, w, _, _ = case(96, 7, 1, 24, BF16)
    x, w = x.requires_grad_(), w[:0].detach().requires_grad_()
    y = tdc_amd.linear_act(x, w)
    dx, dw = grads(y, (x, w), torch.empty_like(y))
    assert y.shape == (7, 0) and not dx.any() and dw.shape == (0, 24)
    q = tdc_amd.mx8_quantize(torch.empty(0, 40, device="cuda"))
    assert tdc_amd.mx8_linear(q, tdc_amd.mx8_quantize(torch.ones(3, 40, device="cuda"))).shape == (0, 3) and q.dequantize().shape == (0, 40)
    assert tdc_amd.rms_norm(torch.empty(0, 40, device="cuda")).shape == (0, 40)


def test_gradients_of_nothing_are_zeros_at_any_size():
    """2^28 of them and some: more than a launch of sixteen threads a number could take."""
    w = torch.ones(32769, 8192, device="cuda", dtype=BF16, requires_grad=True)
    x = torch.ones(0, 8192, device="cuda", dtype=BF16)
    dw, = grads(tdc_amd.linear_act(x, w), (w,), torch.ones(0, 32769, device="cuda", dtype=BF16))
    assert dw.shape == w.shape and not dw.view(torch.int16).any()
    x = torch.ones(1 << 20, 264, device="cuda", dtype=F16, requires_grad=True)
    w = torch.ones(0, 264, device="cuda", dtype=F16)
    dx, = grads(tdc_amd.linear_act(x, w), (x,), torch.ones(1 << 20, 0, device="cuda", dtype=F16))
    assert dx.shape == x.shape and not dx.view(torch.int16).any()
    for dtype in (F32, BF16):
        w = torch.ones(1001, device="cuda", dtype=dtype, requires_grad=True)
        dw, = grads(tdc_amd.rms_norm(torch.ones(0, 1001, device="cuda", dtype=BF16), w), (w,), torch.ones(0, 1001, device="cuda", dtype=BF16))
        assert dw.dtype == dtype and dw.shape == (1001,) and not dw.any()


def test_rms_norm_of_squares_past_32_bits_is_zeros():
    x = torch.full((3, 100), 3.0, device="cuda")
    x[1] = 3e19
    y = tdc_amd.rms_norm(x)
    assert not y[1].any() and (y[[0, 2]] - 1).abs().max() < 1e-5


# ---- 8 bits ----

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 31), (5, 32), (17, 100), (33, 512), (40, 1001), (2, 4097)])
def test_mx8_quantize(rows, K, dtype):
    x = numbers(100, (rows, K), dtype) * torch.exp2(torch.randint(-9, 9, (rows, K), generator=seeded(101))).cuda().to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, K // 2] = float("inf")
        x[rows - 1, 0] = float("nan")
    q = tdc_amd.mx8_quantize(x)
    want, byte = ref.quantize8(host(x))
    got = host(q.dequantize())
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(host(q.dequantize(BF16)), want, equal_nan=True)
    codes, scales = q.codes.cpu().numpy(), q.scales.cpu().numpy()
    assert not codes[:, K:].any()
    blocks = (K + 31) // 32
    flat = np.stack([scales[b // 16, :, 4 * (b % 4) + b % 16 // 4] for b in range((K + 511) // 512 * 16)], 1)
    assert np.array_equal(flat[:, :blocks], byte) and not flat[:, blocks:].any()


def test_mx8_rounding_at_every_border():
    """Every halfway point of the grid, its neighbours, saturation, the smallest and the largest scales."""
    half = (ref.GRID8[1:] + ref.GRID8[:-1]) / 2
    v = np.concatenate([half, np.nextafter(half.astype(np.float32), 0).astype(np.float64), np.nextafter(half.astype(np.float32), 1e9).astype(np.float64),
                        ref.GRID8, [449, 463.9, 464, 465, 480, 496, 511.9]])
    v = v[: len(v) // 31 * 31].reshape(-1, 31)
    for power in (0, -60, 100):
        x = np.concatenate([np.full((len(v), 1), 300.0), v * np.where(np.arange(31) % 2, -1, 1)], 1).astype(np.float32).astype(np.float64) * 2.0 ** power
        got = host(tdc_amd.mx8_quantize(torch.from_numpy(x).float().cuda()).dequantize())
        assert np.array_equal(got, ref.quantize8(x)[0])
    x = torch.full((1, 32), 65504.0, device="cuda")
    # 65504 = 511.75 2^7 saturates at 448 2^7: half precision's numbers stay finite in 8 bits and back
    assert tdc_amd.mx8_quantize(x).dequantize()[0, 0] == 57344 and tdc_amd.mx8_quantize(x.half()).dequantize(F16)[0, 0] == 57344
    tiny = torch.full((1, 32), 2.0 ** -140, device="cuda")
    assert torch.equal(tdc_amd.mx8_quantize(tiny).dequantize(), torch.zeros_like(tiny))


def check_mx8(y, x, w, b, r, act, dtype, what=""):
    """x, w: the values that the 8 bits stand for."""
    _, want = ref.linear(x, w, opt(b), opt(r), act)
    S = np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(host(b))) + (0 if r is None else np.abs(host(r)))
    K = x.shape[1]
    top = lambda v: np.abs(np.pad(v, ((0, 0), (0, -K % 64)))).reshape(len(v), -1, 64).max(2)  # noqa: E731
    off = (16 + K / 8) * E * S + 64 * 2.0 ** -14 * (top(x) @ top(w).T)
    close(y, want, 1.1 * off + rounded(want, dtype) * (1 + 1e-2), what)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", PRODUCTS + [(40, 200, 5000), (600, 520, 8200)])
def test_mx8_linear(M, N, K, dtype):
    for i, act in enumerate(("none", "relu", "silu")):
        x, w, b, r = case(110 + 10 * i, M, N, K, dtype, bias=i != 1, residual=i != 2, bias_dtype=F32 if i == 2 else dtype)
        q, qw = tdc_amd.mx8_quantize(x), tdc_amd.mx8_quantize(w)
        y = tdc_amd.mx8_linear(x, qw, b, r, act=act)
        assert y.dtype == dtype and torch.equal(y, tdc_amd.mx8_linear(q, qw, b, r, act=act, out_dtype=dtype))
        check_mx8(y, host(q.dequantize()), host(qw.dequantize()), b, r, act, dtype, f"{M} {N} {K} {act}")


@pytest.mark.parametrize("M,N,K", [(3400, 3500, 4200), (3333, 3850, 128), (30, 40, 40000)])
def test_mx8_linear_of_whole_numbers_is_exact(M, N, K):
    """Whole numbers of up to 8 in magnitude are E4M3 values at the scales of blocks that hold an 8 (2^-5), and so are their products above what
    an instruction keeps."""
    g = seeded(6)
    x = torch.zeros(M, K)
    x.scatter_(1, torch.randint(0, K, (M, 20), generator=g), torch.randint(-3, 4, (M, 20), generator=g).float())
    w = torch.randint(-4, 5, (N, K), generator=g).float()
    y = tdc_amd.mx8_linear(x.cuda(), tdc_amd.mx8_quantize(w.cuda()), out_dtype=BF16)
    assert torch.equal(y.float(), x.cuda() @ w.t().contiguous().cuda())


def test_mx8_linear_keeps_nans_to_their_rows():
    x, w = numbers(130, (70, 700), BF16), numbers(131, (90, 700), BF16)
    qw = tdc_amd.mx8_quantize(w)
    want = tdc_amd.mx8_linear(x, qw)
    x[40, 699] = float("inf")
    got = tdc_amd.mx8_linear(x, qw)
    assert torch.equal(got[:40], want[:40]) and torch.equal(got[41:], want[41:]) and got[40].isnan().all()
    w[7, 300] = float("nan")
    got = tdc_amd.mx8_linear(x[:40], tdc_amd.mx8_quantize(w))
    assert got[:, 7].isnan().all() and torch.equal(got[:, :7], want[:40, :7]) and torch.equal(got[:, 8:], want[:40, 8:])


# ---- RMS norm ----

ROWS = [(1, 1), (1, 4096), (2, 7), (3, 128), (5, 129), (17, 256), (100, 300), (33, 512), (300, 513), (7, 1001), (40, 2048), (9, 2050), (6, 8192), (3, 5000)]


def rms_case(seed, M, C, dtype, residual, weight_dtype=None):
    x = numbers(seed, (M, C), dtype, 2.0) + 0.5
    return x, (numbers(seed + 1, (C,), F32) * 0.3 + 1).to(weight_dtype or F32), numbers(seed + 2, (M, C), dtype) if residual else None


def summed(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,C", ROWS)
def test_rms_norm(M, C, dtype):
    for residual in (False, True):
        x, w, r = rms_case(140, M, C, dtype, residual, dtype if residual else F32)
        out = tdc_amd.rms_norm(x, w, r, eps=1e-3)
        y, h = out if residual else (out, x)
        assert torch.equal(h, summed(x, r))
        _, want, _ = ref.rms(host(h), host(w), float(np.float32(1e-3)))
        close(y, want, 64 * E * np.abs(want) + rounded(want, dtype) * (1 + 1e-3), f"{M} {C}")
        close(tdc_amd.rms_norm(x, None, r, eps=1e-3)[0] if residual else tdc_amd.rms_norm(x, eps=1e-3), ref.rms(host(h), 1.0, float(np.float32(1e-3)))[1],
              (64 * E + U[dtype]) * 1.001 * np.abs(ref.rms(host(h), 1.0, float(np.float32(1e-3)))[1]) + LEAST[dtype])
        out = tdc_amd.rms_norm_mx8(x, w, r, eps=1e-3)
        q, h8 = out if residual else (out, x)
        assert torch.equal(h8, h)
        # the nearest values, but for numbers within the norm's own error of a border between two
        low, _ = ref.quantize8(want)
        got = host(q.dequantize())
        step = np.maximum(np.abs(want), 0)
        near = np.abs(got - low) <= 2.0 ** -3 * np.maximum(step, np.abs(want).max() * 2.0 ** -14)
        assert near.all() and (got != low).mean() <= 0.001 + 2.0 / got.size


def check_rms_grads(M, C, dtype, residual, checkpoint, with_dh=True, weight_dtype=None):
    x, w, r = rms_case(150, M, C, dtype, residual, weight_dtype)
    dy, dh = numbers(153, (M, C), dtype), numbers(154, (M, C), dtype)
    wrt = [t.requires_grad_() for t in (x, w, r) if t is not None]
    out = tdc_amd.rms_norm(x, w, r, eps=1e-3, checkpoint=checkpoint)
    if residual:
        got = grads(out, wrt, (dy, dh)) if with_dh else grads(out[0], wrt, dy)
    else:
        got = grads(out, wrt, dy)
    h = host(summed(x.detach(), None if r is None else r.detach()))
    u, _, rstd = ref.rms(h, host(w), float(np.float32(1e-3)))
    u = ref.quantize8(h)[0] * rstd if checkpoint else u
    extra = host(dh) if residual and with_dh else 0.0
    dx, dw = ref.rms_grads(u, rstd, host(w), host(dy), extra)
    g = np.abs(host(dy) * host(w))
    size = rstd * (g + np.abs(u) * (g * np.abs(u)).mean(-1, keepdims=True)) + np.abs(extra)
    what = f"{M} {C} {residual} {checkpoint}"
    close(got[0], dx, 64 * E * size + rounded(np.abs(dx) + 64 * E * size, dtype), what + " dx")
    S = (np.abs(host(dy) * u)).sum(0)
    close(got[1], dw, 512 * E * S + rounded(np.abs(dw) + 512 * E * S, w.dtype), what + " dweight")
    if residual:
        assert torch.equal(got[2], got[0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,C", ROWS + [(20000, 24), (3000, 700)])
def test_rms_norm_gradients(M, C, dtype):
    check_rms_grads(M, C, dtype, False, None)
    check_rms_grads(M, C, dtype, True, "mx8", weight_dtype=dtype)
    check_rms_grads(M, C, dtype, True, None, with_dh=False)


def test_rms_norm_where_only_the_sum_is_used():
    x, w, r = rms_case(160, 5, 40, BF16, True)
    wrt = [t.requires_grad_() for t in (x, w, r)]
    y, h = tdc_amd.rms_norm(x, w, r)
    dh = numbers(161, (5, 40), BF16)
    got = grads(h, wrt, dh)
    assert torch.equal(got[0], dh) and torch.equal(got[2], dh) and not got[1].any()


def test_rms_norm_strides_specials_and_zeros():
    wide = numbers(170, (4, 6, 100), BF16)
    for x in (wide[..., 3:67], wide[:, ::2, 8:72], wide[..., 0:64].transpose(0, 1), wide[:1, :1, :64].expand(3, 2, 64)):
        assert torch.equal(tdc_amd.rms_norm(x), tdc_amd.rms_norm(x.contiguous()))
        r = wide[:x.shape[0], :x.shape[1], 33:97].expand(x.shape) if x.shape[1] <= 6 and x.shape[0] <= 4 else None
        if r is not None:
            a, b = tdc_amd.rms_norm(x, None, r), tdc_amd.rms_norm(x.contiguous(), None, r.contiguous())
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = numbers(171, (9, 333), F32)
    want = tdc_amd.rms_norm(x)
    for v in (float("nan"), float("inf")):
        y = x.clone()
        y[4, 10] = v
        y = tdc_amd.rms_norm(y)
        assert torch.equal(y[:4], want[:4]) and torch.equal(y[5:], want[5:]) and y[4, 10].isnan()
    assert not tdc_amd.rms_norm(torch.zeros(3, 50, device="cuda")).any()


# ---- together ----

def test_block_in_training_and_in_8_bits():
    """residual -> norm -> factor with an activation -> factor with the residual, as a network's block runs: gradients through all of it against
    64 bits, and the same block served in 8 bits near the 16-bit one."""
    M, C, R = 300, 192, 96
    x, r = numbers(180, (M, C), BF16), numbers(181, (M, C), BF16)
    gamma = (numbers(182, (C,), F32) * 0.2 + 1)
    w1, w2, b1 = numbers(183, (R, C), BF16, C ** -0.5), numbers(184, (C, R), BF16, R ** -0.5), numbers(185, (R,), BF16, 0.1)
    dy = numbers(186, (M, C), BF16)
    wrt = [t.requires_grad_() for t in (x, r, gamma, w1, w2, b1)]

    def block(checkpoint):
        n, h = tdc_amd.rms_norm(x, gamma, r, checkpoint=checkpoint)
        return tdc_amd.linear_act(tdc_amd.linear_act(n, w1, b1, act="silu", checkpoint=checkpoint), w2, None, h, checkpoint=checkpoint)
    y = block(None)
    got = grads(y, wrt, dy)
    d = [t.detach().double().cpu().requires_grad_() for t in wrt]
    h = d[0] + d[1]
    n = h / torch.sqrt((h ** 2).mean(-1, keepdim=True) + 1e-6) * d[2]
    t = n @ d[3].t() + d[5]
    want_y = t * torch.sigmoid(t) @ d[4].t() + h
    want = torch.autograd.grad(want_y, d, dy.double().cpu())
    # some eight roundings to 16 bits one after the other, each u / sqrt(3) of its tensor in the mean
    for a, b in zip((y, *got), (want_y, *want)):
        assert (a.detach().double().cpu() - b).norm() <= 8 * U[BF16] * b.norm()
    # 8 bits: two products of numbers rounded to 4 bits of significand, each 2^-4 / sqrt(3) at most
    for a, b in zip(grads(block("mx8"), wrt, dy), want):
        assert (a.double().cpu() - b).norm() <= 2 * 2.0 ** -4 * b.norm()
    with torch.no_grad():
        q, h = tdc_amd.rms_norm_mx8(x, gamma, r)
        z = tdc_amd.mx8_linear(tdc_amd.mx8_linear(q, tdc_amd.mx8_quantize(w1), b1, act="silu"), tdc_amd.mx8_quantize(w2), None, h)
    assert (z.double().cpu() - want_y).norm() <= 4 * 2.0 ** -4 * want_y.norm()


def test_streams_graphs_and_repeats():
    """Replays with new inputs and the program's own work between them, on a stream that is not the default one, against eager results."""
    M, N, K = 70, 120, 520
    x, w, b, r = case(190, M, N, K, BF16)
    dy = numbers(191, (M, N), BF16)
    gamma = numbers(192, (K,), F32)
    qw = tdc_amd.mx8_quantize(w)
    wrt = [t.requires_grad_() for t in (x, w, b)]

    def step():
        n, h = tdc_amd.rms_norm(x, gamma, x.detach(), checkpoint="mx8")
        y = tdc_amd.linear_act(n, w, b, r, act="silu", checkpoint="mx8")
        g = grads((y, h), wrt, (dy, n.detach()))
        with torch.no_grad():
            return (y.detach(), *g, tdc_amd.mx8_linear(x, qw), tdc_amd.mx8_linear(tdc_amd.rms_norm_mx8(x, gamma), qw))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(numbers(200 + k, (M, K), BF16))
            dy.copy_(numbers(210 + k, (M, N), BF16))
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in out]
        want = step()
        assert all(torch.equal(a, c) for a, c in zip(held, want)), k
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, c) for a, c in zip(again, want)), k


def test_refusals():
    x, w, b, r = case(220, 4, 8, 32, BF16)
    f = tdc_amd.linear_act
    for bad in (lambda: f(x.float(), w.float()), lambda: f(x, w.half()), lambda: f(x[:, :31], w), lambda: f(x, w, b[:7]), lambda: f(x, w, b.half()),
                lambda: f(x, w, None, r[:, :7]), lambda: f(x, w, None, r.float()), lambda: f(x, w, act="gelu"), lambda: f(x, w, checkpoint="mx4"),
                lambda: f(x.cpu(), w), lambda: f(x, w.cpu()), lambda: f(x, w[0]), lambda: tdc_amd.conv1x1_act(x, w),
                lambda: tdc_amd.mx8_linear(x, w), lambda: tdc_amd.mx8_linear(x.float(), tdc_amd.mx8_quantize(w)),
                lambda: tdc_amd.mx8_linear(x, tdc_amd.mx4_quantize(w)), lambda: tdc_amd.mx8_linear(x, tdc_amd.mx8_quantize(w), out_dtype=F32),
                lambda: tdc_amd.rms_norm(x, b), lambda: tdc_amd.rms_norm(x, None, x.float()), lambda: tdc_amd.rms_norm(torch.zeros(2, 8193, device="cuda")),
                lambda: tdc_amd.rms_norm(x, eps=-1.0), lambda: tdc_amd.rms_norm(x, checkpoint="mx4"), lambda: tdc_amd.rms_norm(x.int())):
        with pytest.raises((TypeError, ValueError, tdc_amd.TdcError)):
            bad()
    q = tdc_amd.mx8_quantize(w)
    g = x.clone().requires_grad_()
    for bad in (lambda: tdc_amd.mx8_quantize(g), lambda: tdc_amd.mx8_linear(g, q), lambda: tdc_amd.mx8_linear(x, q, b.clone().requires_grad_()),
                lambda: tdc_amd.rms_norm_mx8(g), lambda: tdc_amd.rms_norm_mx8(x, None, g)):
        with pytest.raises(RuntimeError, match="gradient"):
            bad()
    with torch.no_grad():
        assert tdc_amd.mx8_linear(g, q).shape == (4, 8)
    y = f(g, w)
    (d,) = torch.autograd.grad(y, g, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_copies_of_an_8_bit_tensor():
    import copy
    import pickle
    q = tdc_amd.mx8_quantize(numbers(230, (5, 70), BF16))
    for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), tdc_amd.Mx8Tensor(q.codes.clone(), q.scales.clone(), q.shape)):
        assert c._codes_at != q._codes_at and torch.equal(c.dequantize(), q.dequantize())


def test_rows_of_other_forms():
    """One row without a leading axis, a transposed weight, a gradient that is one number everywhere, a graph that is walked twice."""
    x, w, b, r = case(240, 6, 40, 64, BF16)
    one = tdc_amd.linear_act(x[0], w, b, r[0], act="silu")
    assert one.shape == (40,) and torch.equal(one, tdc_amd.linear_act(x[:1], w, b, r[:1], act="silu")[0])
    t = numbers(241, (64, 40), BF16).t()
    assert torch.equal(tdc_amd.linear_act(x, t), tdc_amd.linear_act(x, t.contiguous()))
    wrt = [v.requires_grad_() for v in (x, w, b, r)]
    for act in ("none", "silu"):
        y = tdc_amd.linear_act(x, w, b, r, act=act)
        first = torch.autograd.grad(y.sum(), wrt, retain_graph=True)
        again = torch.autograd.grad(y.sum(), wrt)
        want = torch.autograd.grad(tdc_amd.linear_act(x, w, b, r, act=act), wrt, torch.ones_like(y))
        assert all(torch.equal(p, q) and torch.equal(p, s) for p, q, s in zip(first, again, want))
        with torch.autograd.set_multithreading_enabled(False):
            here = torch.autograd.grad(tdc_amd.linear_act(x, w, b, r, act=act), wrt, torch.ones_like(y))
        assert all(torch.equal(p, q) for p, q in zip(here, want))
    x1 = x.detach()[0].clone().requires_grad_()
    (d,) = torch.autograd.grad(tdc_amd.linear_act(x1, w.detach(), act="silu"), x1, torch.ones(40, dtype=BF16, device="cuda"))
    assert d.shape == (64,)
    y, h = tdc_amd.rms_norm(x.detach()[0], None, x.detach()[1])
    assert y.shape == h.shape == (64,)
    # a residual for all rows at once, whose gradient is summed over them
    shared = numbers(242, (40,), BF16).requires_grad_()
    (g,) = torch.autograd.grad(tdc_amd.linear_act(x.detach(), w.detach(), None, shared.expand(6, 40)), shared, torch.ones(6, 40, dtype=BF16, device="cuda"))
    assert torch.equal(g, torch.full_like(g, 6))


@pytest.mark.parametrize("needs", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 1, 0), (0, 1, 0, 1)])
@pytest.mark.parametrize("N,K", [(40, 64), (41, 67)])
def test_gradients_that_are_wanted_alone(needs, N, K):
    x, w, b, r = case(250, 9, N, K, F16)
    dy = numbers(251, (9, N), F16)
    for act in ("none", "relu", "silu"):
        for checkpoint in (None, "mx8"):
            full = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]
            want = grads(tdc_amd.linear_act(*full, act=act, checkpoint=checkpoint), full, dy)
            some = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, w, b, r), needs)]
            got = grads(tdc_amd.linear_act(*some, act=act, checkpoint=checkpoint), [t for t in some if t.requires_grad], dy)
            assert all(torch.equal(p, q) for p, q in zip(got, [v for v, n in zip(want, needs) if n]))


def test_recomputed_layers_and_accumulated_gradients():
    """torch's recomputing checkpoints around the operators, and .grad of leaves that two terms share."""
    from torch.utils.checkpoint import checkpoint
    x, w, _, r = case(260, 30, 64, 64, BF16)
    gamma = numbers(261, (64,), F32)
    leaves = [t.requires_grad_() for t in (x, w, gamma, r)]

    def layer(x, w, gamma, r):
        n, h = tdc_amd.rms_norm(x, gamma, r)
        return tdc_amd.linear_act(n, w, None, h, act="silu", checkpoint="mx8")
    plain = grads(layer(*leaves), leaves, torch.ones(30, 64, dtype=BF16, device="cuda"))
    again = grads(checkpoint(layer, *leaves, use_reentrant=False), leaves, torch.ones(30, 64, dtype=BF16, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(plain, again))
    layer(*leaves).backward(torch.ones(30, 64, dtype=BF16, device="cuda"))
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, plain))
    assert x.grad.data_ptr() != r.grad.data_ptr()
    x.grad.zero_()
    assert torch.equal(r.grad, plain[3])


def test_calls_on_two_streams_at_once():
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x, w, _, _ = case(270, 500, 300, 2000, BF16)
    y, v, _, _ = case(280, 40, 700, 3300, BF16)
    q, qv = tdc_amd.mx8_quantize(w), tdc_amd.mx8_quantize(v)
    want = [(tdc_amd.linear_act(x, w), tdc_amd.mx8_linear(x, q)), (tdc_amd.linear_act(y, v), tdc_amd.mx8_linear(y, qv))]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, (s, args) in enumerate(((a, (x, w, q)), (b, (y, v, qv)))):
            with torch.cuda.stream(s):
                got[k].append((tdc_amd.linear_act(args[0], args[1]), tdc_amd.mx8_linear(args[0], args[2])))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(p, want[k][0]) and torch.equal(r, want[k][1]) for p, r in got[k])


def test_offsets_beyond_32_bits():
    """Operands of more than 4 GiB: the last rows of each, against the same rows by themselves."""
    M, K, N = 300000, 8200, 24
    x = torch.empty((M, K), dtype=BF16, device="cuda")
    x[:1000] = 0
    x[1000:] = numbers(290, (1, K), BF16)
    x[-100:] = numbers(291, (100, K), BF16)
    w = numbers(292, (N, K), BF16, K ** -0.5)
    small = x[-100:].clone()
    y = tdc_amd.linear_act(x, w)
    assert torch.equal(y[:1000], torch.zeros_like(y[:1000]))
    want = tdc_amd.linear_act(small, w)
    assert (y[-100:].double() - want.double()).abs().max() <= 2 * U[BF16] * want.double().abs().max()      # (summed in other parts)
    n = tdc_amd.rms_norm(x[:, :8192])
    assert torch.equal(n[-100:], tdc_amd.rms_norm(small[:, :8192]))
    del n
    q = tdc_amd.mx8_quantize(x)
    assert torch.equal(q.codes[-100:], tdc_amd.mx8_quantize(small).codes)
    del q
    # the weight's gradient: rows of zeros but for the last hundred
    dy = torch.zeros((M, N), dtype=BF16, device="cuda")
    dy[-100:] = numbers(293, (100, N), BF16)
    w.requires_grad_()
    (dw,) = grads(tdc_amd.linear_act(x, w), (w,), dy)
    want = dy[-100:].double().cpu().t() @ small.double().cpu()
    assert (dw.double().cpu() - want).abs().max() <= 2 * U[BF16] * want.abs().max()


def test_long_rows():
    K = 1 << 21
    x, w = torch.zeros(2, K, dtype=BF16, device="cuda"), torch.zeros(3, K, dtype=BF16, device="cuda")
    x[:, ::4096] = 1
    w[:, ::2048] = torch.tensor([[1.0], [2.0], [-1.0]], dtype=BF16, device="cuda")
    want = torch.tensor([512.0, 1024.0, -512.0], device="cuda").expand(2, 3)
    assert torch.equal(tdc_amd.linear_act(x, w).float(), want)
    assert torch.equal(tdc_amd.mx8_linear(x, tdc_amd.mx8_quantize(w)).float(), want)
    with pytest.raises(tdc_amd.TdcError):
        tdc_amd.linear_act(torch.zeros(1, K + 1, dtype=BF16, device="cuda"), torch.zeros(1, K + 1, dtype=BF16, device="cuda"))
    # rows further apart than a request's offset reaches are copied first
    far = torch.zeros(3 * (1 << 22) + 64, dtype=BF16, device="cuda").as_strided((3, 64), (1 << 22, 1))
    far.copy_(numbers(295, (3, 64), BF16))
    v = numbers(296, (10, 64), BF16)
    assert torch.equal(tdc_amd.linear_act(far, v), tdc_amd.linear_act(far.contiguous(), v))


@pytest.mark.parametrize("needs", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)])
@pytest.mark.parametrize("C", [64, 301, 4100])
def test_norm_gradients_that_are_wanted_alone(needs, C):
    x, w, r = rms_case(300, 40, C, BF16, True)
    dy, dh = numbers(303, (40, C), BF16), numbers(304, (40, C), BF16)
    for checkpoint in (None, "mx8"):
        full = [t.detach().clone().requires_grad_() for t in (x, w, r)]
        want = grads(tdc_amd.rms_norm(*full, checkpoint=checkpoint), full, (dy, dh))
        some = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, w, r), needs)]
        got = grads(tdc_amd.rms_norm(*some, checkpoint=checkpoint), [t for t in some if t.requires_grad], (dy, dh))
        assert all(torch.equal(p, q) for p, q in zip(got, [v for v, n in zip(want, needs) if n]))


def test_what_is_kept_may_wait_on_the_host():
    """What a gradient needs goes to the host and comes back elsewhere; how much it is."""
    x, w, b, _ = case(310, 50, 70, 96, BF16)
    gamma = numbers(311, (96,), F32)
    leaves = [t.requires_grad_() for t in (x, w, b, gamma)]
    dy = numbers(312, (50, 70), BF16)
    for checkpoint in (None, "mx8"):
        layer = lambda: tdc_amd.linear_act(tdc_amd.rms_norm(x, gamma, checkpoint=checkpoint), w, b, act="silu", checkpoint=checkpoint)  # noqa: E731, B023
        want = grads(layer(), leaves, dy)
        with torch.autograd.graph.save_on_cpu():
            y = layer()
        assert all(torch.equal(p, q) for p, q in zip(grads(y, leaves, dy), want))
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
            layer()
        rows = 50 * 128 + 50 * 16 if checkpoint else 50 * 96 * 2
        # x twice (of the norm, of the product), z, and the parameters and 1 / root mean square
        assert sum(kept) <= 2 * rows + 50 * 70 * 2 + 70 * 96 * 2 + 96 * 4 + 50 * 4


@pytest.mark.parametrize("M,N,K", [(5, 24, 40), (70, 120, 520), (33, 1001, 2001), (300, 96, 64)])
@pytest.mark.parametrize("dtype,far", [(F16, 1e5), (BF16, 3.4e38)])
def test_silu_gradient_where_what_it_is_taken_of_leaves_the_type(M, N, K, dtype, far):
    """Sums that are finite in 32 bits and infinite in 16: the slope there is 0 or 1, as it is in 32 bits 50 from the origin."""
    x, w, _, r = case(320, M, N, K, dtype)
    dy = numbers(321, (M, N), dtype)

    def at(distance):
        b = torch.zeros(N, device="cuda")
        b[3], b[5] = -distance, distance
        wrt = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]
        y = tdc_amd.linear_act(*wrt, act="silu")
        return y.detach(), grads(y, wrt, dy)
    y, got = at(far)
    _, want = at(50.0)
    assert not y[:, 3].any() and (y[:, 5] > 6e4).all()
    for g, v in zip(got, want):
        # (50 from the origin it is 2^-66 off, and so is what is summed of it)
        assert torch.isfinite(g).all() and (g.double() - v.double()).abs().max() <= M * 16 * 2.0 ** -60
    assert not got[3][:, 3].any() and torch.equal(got[3][:, 5], dy[:, 5])


def test_relu_gradient_at_nans_and_of_infinities():
    """What is not a number passes its gradient on; where the result is 0 an infinite gradient is as none."""
    M, N, K = 40, 24, 64
    x, w, b, _ = case(330, M, N, K, BF16, residual=False)
    dy = numbers(331, (M, N), BF16)
    bad = x.clone()
    bad[7, 3] = float("nan")
    for rows in (slice(0, M), slice(0, 9)):
        wrt = [t.detach().clone().requires_grad_() for t in (bad[rows], w, b)]
        y = tdc_amd.linear_act(*wrt, act="relu")
        assert y[7].isnan().all()
        dx, _, db = grads(y, wrt, dy[rows])
        passed = torch.where(y.isnan() | (y > 0), dy[rows], torch.zeros_like(y)).double().cpu()
        close(dx, (passed @ w.double().cpu()).numpy(), host(rounded_products(passed, w)), "dx")
        S = passed.abs().sum(0).numpy()
        close(db, passed.sum(0).numpy(), 512 * E * S + rounded(S, BF16), "dbias")
        wrt = [t.detach().clone().requires_grad_() for t in (x[rows], w, b)]
        y = tdc_amd.linear_act(*wrt, act="relu")
        off = (y == 0) & (torch.arange(N, device="cuda") % 5 == 0)
        assert off.any()
        far = dy[rows].clone()
        far[off] = float("inf")
        got = grads(y, wrt, far)
        far[off] = 1
        assert all(torch.equal(g, v) for g, v in zip(got, grads(tdc_amd.linear_act(*wrt, act="relu"), wrt, far)))


def rounded_products(a, w):
    """The bound on a row of products a w: their sums in fp32, rounded to 16 bits once."""
    S = a.abs() @ w.double().cpu().abs()
    return ((16 + a.shape[1] / 8) * E + U[BF16] * 1.001) * S + LEAST[BF16]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [1, 40, 100, 300, 1001, 2100, 5000])
def test_rms_norm_mx8_leaves_zeros_behind_a_row_of_nans(C, dtype):
    """Codes and scales past the last number are zeros, also in rows whose root mean square is a NaN or, of zeros without eps, 0."""
    x = numbers(340, (5, C), dtype)
    x[1, C // 2] = float("nan")
    x[2, 0] = float("inf")
    x[3] = 0
    for eps in (1e-6, 0.0):
        for r in (None, torch.zeros_like(x)):
            out = tdc_amd.rms_norm_mx8(x, None, r, eps=eps)
            q = out if r is None else out[0]
            got = q.dequantize()
            assert got[1].isnan().all() and got[2, 0].isnan() and torch.isfinite(got[[0, 4]]).all()
            assert got[3].isnan().all() if eps == 0 else not got[3].any()
            assert not q.codes[:, C:].any()
            scales = torch.stack([q.scales[b // 16, :, 4 * (b % 4) + b % 16 // 4] for b in range((C + 511) // 512 * 16)], 1)
            assert not scales[:, (C + 31) // 32:].any()


def test_the_residuals_gradient_is_made_once():
    """Where the gradient that the activation hands on is a result, the workspace holds no second one."""
    M, N, K = 4096, 2048, 64
    x, w, _, r = case(360, M, N, K, BF16)
    dy = numbers(361, (M, N), BF16)
    wrt = [t.requires_grad_() for t in (x, w, r)]
    y = tdc_amd.linear_act(x, w, None, r, act="silu")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    got = grads(y, wrt, dy)
    torch.cuda.synchronize()
    made = torch.cuda.max_memory_allocated() - held
    # dresidual, dx and dw, and what else the workspace is for: a tenth of a second one is more than enough
    assert sum(t.numel() * 2 for t in got) <= made <= sum(t.numel() * 2 for t in got) + M * N * 2 * 0.6, made


# Sizes at which the product, w's gradient and x's take each of the six tiles, whole and in parts of the sum: 20 to 145 rows take tiles of 32 and 64
# rows and the deep one of 128, 2022 x 6488 x 1031 and 14328 x 456 x 2072 those of 256 x 256 and 256 x 128 in every layout.
TILES = [(20, 9, 42), (8506, 11, 40), (21, 1483, 1280), (2801, 33, 1428), (19193, 195, 50), (250, 8720, 176), (69, 2544, 4744), (2022, 6488, 1031),
         (14328, 456, 2072), (430, 924, 15735), (8559, 8896, 152), (2796, 10, 11494), (145, 8299, 8858)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", TILES)
def test_every_tile_and_layout_on_whole_numbers(M, N, K, dtype):
    """Sums of small whole numbers are exact in fp32 in any order, and rounded once: results are those, to the bit.  With "silu" what the
    activation is taken of is a whole number too, so that its gradient in each place is known to its own rounding."""
    g = torch.Generator(device="cuda").manual_seed(7)
    whole = lambda *shape: torch.randint(-4, 5, shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, w, r, dy = whole(M, K), whole(N, K), whole(M, N), whole(M, N)
    f = lambda t: t.detach().float()  # noqa: E731
    z = f(x) @ f(w).t().contiguous() + f(r)
    assert z.abs().max() < 2 ** 24
    x, w, r = (t.requires_grad_() for t in (x, w, r))
    y = tdc_amd.linear_act(x, w, None, r)
    assert torch.equal(y, z.to(dtype))
    dx, dw, dr = grads(y, (x, w, r), dy)
    assert torch.equal(dx, (f(dy) @ f(w)).to(dtype)) and torch.equal(dw, (f(dy).t().contiguous() @ f(x)).to(dtype)) and torch.equal(dr, dy)
    del dx, dw, dr, y
    # an eighth of the product: numbers at which "silu" bends
    x8 = (x.detach() / 8).requires_grad_()
    y = tdc_amd.linear_act(x8, w, None, r, act="silu")
    z = ((z - f(r)) / 8 + f(r)).double()
    s = torch.sigmoid(z)
    u, least = U[dtype], LEAST[dtype]
    # (the hardware's sigmoid is good to 2^-22 and |z| 2^-24 of itself, and to 2^-126 where e^-z passes 32 bits)
    assert ((y.double() - z * s).abs() <= (u + 2.0 ** -20 + z.abs() * 2.0 ** -22) * (z * s).abs() + z.abs() * 2.0 ** -125 + 2 * least).all()
    _, _, dr = grads(y, (x8, w, r), dy)
    z = z.to(dtype).double()      # (what is kept)
    s = torch.sigmoid(z)
    slope, d = s * (1 + z * (1 - s)), dy.double()
    # (1 + z (1 - s) may cancel)
    off = d.abs() * (1 + z.abs()) * (s * (2.0 ** -20 + z.abs() * 2.0 ** -22) + 2.0 ** -125)
    assert ((dr.double() - d * slope).abs() <= off + u * 1.001 * (d * slope).abs() + 2 * least).all()


TILES8 = [(17, 10, 42), (17, 9, 2994), (9828, 9, 47), (266, 9, 17403), (19659, 9, 352), (1593, 9, 6595), (16794, 136, 46), (8356, 9, 6438),
          (1926, 4040, 960), (8069, 1995, 533), (9161, 156, 14045), (25088, 128, 512)]


@pytest.mark.parametrize("M,N,K", TILES8)
def test_every_tile_of_the_8_bit_product_on_whole_numbers(M, N, K):
    """The six tiles in 8 bits, whole and in parts of the sum, on numbers that 8 bits hold and sums that an instruction keeps whole."""
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.zeros(M, K, device="cuda")
    x.scatter_(1, torch.randint(0, K, (M, 20), generator=g, device="cuda"), torch.randint(-3, 4, (M, 20), generator=g, device="cuda").float())
    w = torch.randint(-4, 5, (N, K), generator=g, device="cuda").float()
    r = torch.randint(-8, 9, (M, N), generator=g, device="cuda").to(BF16)
    y = tdc_amd.mx8_linear(x, tdc_amd.mx8_quantize(w), None, r, act="relu", out_dtype=BF16)
    assert torch.equal(y.float(), (x @ w.t().contiguous() + r.float()).clamp(min=0).to(BF16).float())


@pytest.mark.parametrize("M,C", [(40000, 256), (20000, 512), (36000, 100), (9000, 1001), (2600, 2100), (2100, 5000)])
def test_rms_norm_of_more_rows_than_run_at_once(M, C):
    """Every team of lanes goes on to further rows, whose numbers are on their way meanwhile: all rows, in every form of the result."""
    test_rms_norm(M, C, BF16)
    for residual in (False, True):
        check_rms_grads(M, C, BF16, residual, "mx8")


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("M,C", [(1300, 2100), (700, 8192), (2300, 900), (9000, 200)])
def test_rms_norm_gradients_of_more_rows_than_run_at_once(M, C, dtype):
    for checkpoint in (None, "mx8"):
        check_rms_grads(M, C, dtype, True, checkpoint)
        check_rms_grads(M, C, dtype, False, checkpoint, weight_dtype=dtype)


def test_mx8_at_the_smallest_and_largest_scales():
    """Blocks whose largest magnitudes lie on either side of where the scale byte stops at 0, and those of the largest numbers there are."""
    top = np.array([2.0 ** -119, 1.9 * 2.0 ** -119, 2.0 ** -120, 1.3 * 2.0 ** -122, 2.0 ** -125, 1.7 * 2.0 ** -126, 2.0 ** -127, 2.0 ** -130, 2.0 ** -135, 2.0 ** -136,
                    2.0 ** 126, 2.0 ** 127, 1.5 * 2.0 ** 127, 1.75 * 2.0 ** 127, float(np.finfo(np.float32).max)])
    share = np.random.default_rng(9).uniform(-1, 1, (len(top), 32))
    share[:, 5] = 1
    x = (share * top[:, None]).astype(np.float32)
    want, byte = ref.quantize8(x.astype(np.float64))
    assert byte[:, 0].tolist() == [0] * 10 + [245] + [246] * 4 and (want[:10] != 0).any(1).all()
    q = tdc_amd.mx8_quantize(torch.from_numpy(x).cuda())
    assert np.array_equal(q.scales[0, :, 0].cpu().numpy(), byte[:, 0]) and np.array_equal(host(q.dequantize()), want)
    # and in the products, small ones with large ones
    for M, N, K in ((5, 24, 96), (70, 40, 200), (300, 200, 700)):
        a, b = torch.randint(-4, 5, (M, K), generator=seeded(350)).float(), torch.randint(-4, 5, (N, K), generator=seeded(351)).float()
        a[:, 20:] *= (torch.arange(K - 20) % 16 == 0).float()      # (sums below 2^8: whole in 16 bits)
        for small in (2.0 ** -122, 2.0 ** -124, 2.0 ** -126):
            y = tdc_amd.mx8_linear(a.cuda() * small, tdc_amd.mx8_quantize(b.cuda() * 2.0 ** 120), out_dtype=BF16)
            assert torch.equal(y.float(), (a.cuda() @ b.t().contiguous().cuda() * (small * 2.0 ** 120)).to(BF16).float())


@pytest.mark.parametrize("dtype,small,large", [(F16, 2.0 ** -22, 2.0 ** 12), (BF16, 2.0 ** -131, 2.0 ** 121)])
@pytest.mark.parametrize("M,N,K", [(3, 40, 96), (70, 40, 96), (300, 130, 203)])
def test_numbers_below_the_normal_ones_take_part(M, N, K, dtype, small, large):
    """Subnormal numbers of either type, as operands (each of x, w and dy in turn) and as results."""
    g = seeded(370)
    x, w, dy = (torch.randint(-3, 4, s, generator=g).float().cuda() for s in ((M, K), (N, K), (M, N)))
    # (a sum whose terms' magnitudes stay below 2^127 passes nothing on the way, and 64 bits hold it: the others are left out)
    def same(got, p, q, by):
        whole = (p.abs() @ q.abs()).double() * by < 2.0 ** 127
        assert torch.equal(got[whole], ((p @ q).double() * by).to(dtype)[whole]) and (whole.all() or by == large)
    for a, b, c in ((small, large, 1.0), (large, small, 1.0), (1.0, large, small), (large, 1.0, small)):
        p, q = ((t * s).to(dtype).requires_grad_() for t, s in ((x, a), (w, b)))
        y = tdc_amd.linear_act(p, q)
        dx, dw = grads(y, (p, q), (dy * c).to(dtype))
        same(y, x, w.t().contiguous(), a * b)
        same(dx, dy, w, c * b)
        same(dw, dy.t().contiguous(), x, c * a)
    tiny = (x * small).to(dtype)
    gamma = torch.ones(K, device="cuda")
    assert torch.equal(tdc_amd.rms_norm(tiny, gamma, torch.zeros_like(tiny))[1], tiny)


# ---- the C entries, with strides that Python does not pass ----

class Guarded:
    """A tensor with numbers of its own before and behind it, which have to stay."""

    def __init__(self, shape, dtype):
        n, self.pad = int(np.prod(shape)), 64 // torch.empty((), dtype=dtype).element_size()
        self.held = torch.full((n + 2 * self.pad,), 77, dtype=dtype, device="cuda")
        self.t = self.held[self.pad:self.pad + n].view(shape)

    def kept(self):
        return bool((self.held[:self.pad] == 77).all() and (self.held[len(self.held) - self.pad:] == 77).all())


def entry(name, *args):
    at = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    assert getattr(tdc_amd.lib(), name)(*at, torch.cuda.current_stream().cuda_stream) == 0, tdc_amd.lib().tdc_last_error_string()


def workspace(name, *args):
    need = ctypes.c_size_t()
    assert getattr(tdc_amd.lib(), name)(*args, ctypes.byref(need)) == 0
    return Guarded((need.value,), torch.uint8)


ENTRY_CASES = [(1, 1, 1), (5, 24, 40), (16, 100, 1000), (33, 1001, 2001), (70, 2544, 744), (129, 127, 257), (300, 96, 64), (1000, 24, 64), (2100, 1030, 1100), (9000, 33, 40)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", ENTRY_CASES)
def test_entries_of_the_product_write_what_is_theirs(M, N, K, dtype):
    """Results in slices of wider tensors and workspaces of just the size that is asked for: nothing beside them is touched."""
    from tdc_amd import _lib
    x, w, b, r = case(380, M, N, K, dtype)
    dy = numbers(381, (M, N), dtype)
    wrt = [t.requires_grad_() for t in (x, w, b, r)]
    want_y = tdc_amd.linear_act(*wrt, act="silu")
    want = grads(want_y, wrt, dy)
    kind = 1 if dtype == F16 else 2
    wide, wide_r = Guarded((M, N + 9), dtype), torch.full((M, N + 5), float("nan"), dtype=dtype, device="cuda")
    y = wide.t[:, 3:3 + N]
    wide_r[:, 1:1 + N] = r.detach()
    z, residual = Guarded((M, N), dtype), wide_r[:, 1:1 + N]
    desc = _lib.LinearDesc(M, N, K, kind, kind, 2, kind, 0, 0, N + 9, N + 5)
    need = ctypes.c_size_t()
    assert tdc_amd.lib().tdc_linear_workspace(ctypes.byref(desc), ctypes.byref(need), None) == 0
    ws = Guarded((need.value,), torch.uint8)
    entry("tdc_linear_forward", ctypes.byref(desc), x, w, b, residual, y, z.t, ws.t, need.value)
    assert torch.equal(y, want_y) and wide.kept() and z.kept() and ws.kept()
    assert (wide.t[:, :3] == 77).all() and (wide.t[:, 3 + N:] == 77).all()
    # z is what the activation is taken of: the result without one
    assert torch.equal(z.t, tdc_amd.linear_act(x.detach(), w.detach(), b.detach(), r.detach()))
    for step in ((N + 7) // 8 * 8 + 24, N + 13):
        wide_dy = torch.full((M, step), float("nan"), dtype=dtype, device="cuda")
        wide_dy[:, 8:8 + N] = dy
        desc = _lib.LinearDesc(M, N, K, kind, kind, 2, kind, 0, 0, step, 0)
        dx, dw, db, dz = (Guarded(s, dtype) for s in ((M, K), (N, K), (N,), (M, (N + 7) // 8 * 8)))
        for given in (1, 0):
            ws = workspace("tdc_linear_backward_workspace", ctypes.byref(desc), given)
            entry("tdc_linear_backward", ctypes.byref(desc), x, None, w, z.t, wide_dy[:, 8:], dx.t, dw.t, db.t, dz.t if given else None, ws.t, ws.t.numel())
            assert all(g.kept() for g in (dx, dw, db, dz, ws))
            assert torch.equal(dx.t, want[0]) and torch.equal(dw.t, want[1]) and torch.equal(db.t, want[2]) and torch.equal(dz.t[:, :N], want[3])
            assert not dz.t[:, N:].any()
            for g in (dx, dw, db):
                g.t.fill_(77)


@pytest.mark.parametrize("M,N,K", ENTRY_CASES + [(40, 33, 513)])
def test_entries_in_8_bits_write_what_is_theirs(M, N, K):
    from tdc_amd import _lib
    x, w, b, r = case(390, M, N, K, BF16)
    want_q, qw = tdc_amd.mx8_quantize(x), tdc_amd.mx8_quantize(w)
    codes, scales = Guarded(tuple(want_q.codes.shape), torch.uint8), Guarded(tuple(want_q.scales.shape), torch.uint8)
    wide_x = torch.full((M, K + 3), float("nan"), dtype=BF16, device="cuda")
    wide_x[:, 1:1 + K] = x
    entry("tdc_mx8_quantize", wide_x[:, 1:], 2, M, K, K + 3, codes.t, scales.t)
    assert codes.kept() and scales.kept() and torch.equal(codes.t, want_q.codes) and torch.equal(scales.t, want_q.scales)
    back = Guarded((M, K + 7), BF16)
    entry("tdc_mx8_dequantize", codes.t, scales.t, M, K, back.t[:, 2:], 2, K + 7)
    assert back.kept() and torch.equal(back.t[:, 2:2 + K], want_q.dequantize(BF16)) and (back.t[:, :2] == 77).all() and (back.t[:, 2 + K:] == 77).all()
    want = tdc_amd.mx8_linear(x, qw, b, r, act="relu")
    for kind in (2, 4):
        wide = Guarded((M, N + 9), BF16)
        desc = _lib.Mx4LinearDesc(M, N, K, kind, 2, 2, 1, K + 3 if kind == 2 else 0, N + 9, 0)
        ws = workspace("tdc_mx8_linear_workspace", ctypes.byref(desc))
        entry("tdc_mx8_linear", ctypes.byref(desc), wide_x[:, 1:] if kind == 2 else codes.t, None if kind == 2 else scales.t, qw.codes, qw.scales, b, r, wide.t[:, 3:],
              ws.t, ws.t.numel())
        assert wide.kept() and ws.kept() and torch.equal(wide.t[:, 3:3 + N], want) and (wide.t[:, :3] == 77).all() and (wide.t[:, 3 + N:] == 77).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,C", [(1, 1), (3, 129), (40, 513), (9, 2050), (3000, 700), (20000, 24), (5, 8191)])
def test_entries_of_rms_norm_write_what_is_theirs(M, C, dtype):
    from tdc_amd import _lib
    x, w, r = rms_case(400, M, C, dtype, True, dtype)
    dy, dh = numbers(403, (M, C), dtype), numbers(404, (M, C), dtype)
    wrt = [t.requires_grad_() for t in (x, w, r)]
    out = tdc_amd.rms_norm(x, w, r, checkpoint="mx8")
    want = grads(out, wrt, (dy, dh))
    kind = {F32: 0, BF16: 2}[dtype]
    p = ctypes.byref(_lib.RmsNormDesc(M, C, kind, kind, 1e-6, 0, 0, 0, 0))
    y, h, rstd = Guarded((M, C), dtype), Guarded((M, C), dtype), Guarded((M,), F32)
    codes, scales = Guarded((M, (C + 127) // 128 * 128), torch.uint8), Guarded(((C + 511) // 512, M, 16), torch.uint8)
    entry("tdc_rms_norm_forward", p, x, r, w, y.t, h.t, rstd.t, codes.t, scales.t)
    assert all(g.kept() for g in (y, h, rstd, codes, scales)) and torch.equal(y.t, out[0]) and torch.equal(h.t, out[1])
    q = tdc_amd.mx8_quantize(h.t)
    assert torch.equal(codes.t, q.codes) and torch.equal(scales.t, q.scales)
    dx, dw = Guarded((M, C), dtype), Guarded((C,), dtype)
    ws = workspace("tdc_rms_norm_workspace", p)
    entry("tdc_rms_norm_backward", p, codes.t, scales.t, w, dy, dh, rstd.t, dx.t, dw.t, ws.t, ws.t.numel())
    assert all(g.kept() for g in (dx, dw, ws)) and torch.equal(dx.t, want[0]) and torch.equal(dw.t, want[1])
    want = tdc_amd.rms_norm_mx8(x.detach(), w.detach(), r.detach())
    entry("tdc_rms_norm_forward_mx8", p, x, r, w, codes.t, scales.t, h.t)
    assert all(g.kept() for g in (codes, scales, h)) and torch.equal(codes.t, want[0].codes) and torch.equal(scales.t, want[0].scales) and torch.equal(h.t, want[1])
