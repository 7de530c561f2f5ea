"""What the 16- and 8-bit operators over rows refuse (no GPU needed), and their 64-bit oracle against hand-worked numbers."""
import ctypes

import numpy as np
import pytest
import torch

import tdc_amd
from oracle import pointwise_ref as ref
from tdc_amd import _lib

INVALID = _lib.TDC_ERR_INVALID


def desc(kind, base, kw):
    d = dict(base)
    d.update(kw)
    return kind(*[d[n] for n, _ in kind._fields_])


def linear(**kw):
    return desc(_lib.LinearDesc, dict(M=4, N=5, K=40, dtype=2, bias_dtype=0, act=0, kept_dtype=2, x_stride=0, w_stride=0, y_stride=0, residual_stride=0), kw)


def linear8(**kw):
    return desc(_lib.Mx4LinearDesc, dict(M=4, N=5, K=40, x_dtype=4, y_dtype=2, bias_dtype=0, act=0, x_stride=0, y_stride=0, residual_stride=0), kw)


def rms(**kw):
    return desc(_lib.RmsNormDesc, dict(rows=4, C=40, dtype=2, weight_dtype=0, eps=1e-6, x_stride=0, residual_stride=0, dy_stride=0, dh_stride=0), kw)


def error():
    return tdc_amd.lib().tdc_last_error_string().decode()


def sizes(d):
    L, a, b = tdc_amd.lib(), ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tdc_linear_workspace(ctypes.byref(d), ctypes.byref(a), ctypes.byref(b)) == 0, error()
    return a.value, b.value


def test_struct_layouts():
    assert ctypes.sizeof(_lib.LinearDesc) == 3 * 8 + 4 * 4 + 4 * 8
    assert ctypes.sizeof(_lib.RmsNormDesc) == 8 + 4 * 4 + 4 * 8


@pytest.mark.parametrize("bad", [dict(M=-1), dict(N=-1), dict(K=0), dict(K=(1 << 21) + 1), dict(N=(1 << 21) + 1), dict(M=1 << 31), dict(dtype=0), dict(dtype=3),
                                 dict(bias_dtype=1), dict(act=3), dict(act=-1), dict(kept_dtype=1), dict(x_stride=39), dict(w_stride=-40),
                                 dict(y_stride=4), dict(residual_stride=1)])
def test_linear_descriptors_are_refused(bad):
    L, d, a, b = tdc_amd.lib(), linear(**bad), ctypes.c_size_t(), ctypes.c_size_t()
    p = ctypes.byref(d)
    assert L.tdc_linear_workspace(p, ctypes.byref(a), ctypes.byref(b)) == INVALID and len(error()) > 15
    assert L.tdc_linear_forward(p, 16, 16, None, None, 16, None, 16, 1 << 40, None) == INVALID
    assert L.tdc_linear_backward(p, 16, None, 16, 16, 16, 16, 16, None, None, 16, 1 << 40, None) == INVALID


def test_linear_arguments_are_refused():
    L, d = tdc_amd.lib(), linear(K=41, M=300, N=300)
    p, (a, b) = ctypes.byref(d), sizes(linear(K=41, M=300, N=300))
    assert 0 < a < b
    f = L.tdc_linear_forward
    assert f(None, 16, 16, None, None, 16, None, 16, a, None) == INVALID
    assert f(p, None, 16, None, None, 16, None, 16, a, None) == INVALID and f(p, 16, None, None, None, 16, None, 16, a, None) == INVALID
    assert f(p, 16, 16, None, None, None, None, 16, a, None) == INVALID
    assert f(p, 24, 16, None, None, 16, None, 16, a, None) == INVALID and "aligned" in error()
    assert f(p, 16, 18, None, None, 16, None, 16, a, None) == INVALID and "aligned" in error()
    assert f(p, 16, 16, None, None, 16, None, 16, a - 1, None) == INVALID and "workspace" in error()
    assert f(p, 16, 16, None, None, 16, None, None, a, None) == INVALID and f(p, 16, 16, None, None, 16, None, 8, a, None) == INVALID
    g, silu, mx8 = L.tdc_linear_backward, ctypes.byref(linear(act=2)), ctypes.byref(linear(kept_dtype=4))
    big = 1 << 30
    assert g(p, 16, None, 16, None, None, 16, None, None, None, 16, big, None) == INVALID       # no dy
    assert g(p, None, None, 16, None, 16, 16, 16, None, None, 16, big, None) == INVALID         # dw without x
    assert g(p, 16, None, None, None, 16, 16, 16, None, None, 16, big, None) == INVALID         # dx without w
    assert g(silu, 16, None, 16, None, 16, 16, None, None, None, 16, big, None) == INVALID and "activation" in error()
    assert g(p, 16, 16, 16, None, 16, None, 16, None, None, 16, big, None) == INVALID and "scales" in error()
    assert g(mx8, 16, None, 16, None, 16, None, 16, None, None, 16, big, None) == INVALID and "scales" in error()
    assert g(p, 16, None, 16, None, 18, 16, None, None, None, 16, big, None) == INVALID and "aligned" in error()
    assert g(p, 16, None, 16, None, 16, 16, None, None, 8, 16, big, None) == INVALID and "aligned" in error()
    assert g(p, 16, None, 16, None, 16, 16, None, None, None, 16, b - 1, None) == INVALID and "workspace" in error()
    # nothing to do is no error, whatever the pointers
    assert f(ctypes.byref(linear(M=0)), None, None, None, None, None, None, None, 0, None) == 0
    assert f(ctypes.byref(linear(N=0)), None, None, None, None, None, None, None, 0, None) == 0
    assert g(p, None, None, None, None, None, None, None, None, None, None, 0, None) == 0


def test_workspaces():
    assert sizes(linear(M=4096, N=4096, K=4096))[0] == 0
    for M in (0, 1, 7, 5000):
        for N in (0, 1, 7, 3001):
            for K in (1, 40, 2999, 40000):
                forward, backward = sizes(linear(M=M, N=N, K=K))
                assert (forward, backward) == (0, 0) if not M or not N else backward > 0
    assert sizes(linear(K=48))[0] == 0 and sizes(linear(K=48, x_stride=50))[0] > 0 and sizes(linear(K=48, x_stride=1 << 22))[0] > 0
    # a row by itself has no stride
    assert sizes(linear(M=1, K=48, x_stride=51))[0] == 0


@pytest.mark.parametrize("d", [dict(M=(1 << 31) - 1, N=1 << 21), dict(M=(1 << 31) - 1, N=4096), dict(M=1 << 30, N=64, K=1 << 20, x_stride=(1 << 20) + 1)])
def test_products_of_more_tiles_than_a_launch_has(d):
    L, n = tdc_amd.lib(), ctypes.c_size_t()
    assert L.tdc_linear_workspace(ctypes.byref(linear(**d)), ctypes.byref(n), None) == INVALID and "work items" in error()


def test_gradients_of_more_rows_than_a_launch_has():
    L, n = tdc_amd.lib(), ctypes.c_size_t()
    d = linear(M=(1 << 31) - 1, N=8, K=512, kept_dtype=4)
    assert L.tdc_linear_workspace(ctypes.byref(d), None, ctypes.byref(n)) == INVALID and "work items" in error()
    d = linear(M=(1 << 24), N=8, K=512, kept_dtype=4)
    assert L.tdc_linear_workspace(ctypes.byref(d), None, ctypes.byref(n)) == 0 and n.value >= (1 << 24) * 512 * 2


@pytest.mark.parametrize("bad", [dict(M=-1), dict(N=-1), dict(K=0), dict(K=1 << 22), dict(x_dtype=3), dict(x_dtype=5), dict(y_dtype=0), dict(y_dtype=4), dict(bias_dtype=1),
                                 dict(act=3), dict(x_dtype=0, x_stride=39), dict(y_stride=4), dict(residual_stride=-5)])
def test_8_bit_product_descriptors_are_refused(bad):
    L, n, d = tdc_amd.lib(), ctypes.c_size_t(), linear8(**bad)
    assert L.tdc_mx8_linear_workspace(ctypes.byref(d), ctypes.byref(n)) == INVALID and len(error()) > 15
    assert L.tdc_mx8_linear(ctypes.byref(d), 16, 16, 16, 16, None, None, 16, 16, 1 << 30, None) == INVALID


def test_8_bit_arguments_are_refused():
    L, c, s = tdc_amd.lib(), ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tdc_mx8_sizes(3, 130, ctypes.byref(c), ctypes.byref(s)) == 0 and (c.value, s.value) == (3 * 256, 3 * 16)
    for rows, K in ((-1, 4), (2, 0), (1 << 36, 64), (2, 1 << 31)):
        assert L.tdc_mx8_sizes(rows, K, ctypes.byref(c), ctypes.byref(s)) == INVALID
    assert L.tdc_mx8_quantize(16, 3, 2, 32, 0, 16, 16, None) == INVALID and "dtype" in error()
    assert L.tdc_mx8_quantize(16, 0, 2, 32, 31, 16, 16, None) == INVALID and "stride" in error()
    assert L.tdc_mx8_quantize(None, 0, 2, 32, 0, 16, 16, None) == INVALID
    assert L.tdc_mx8_quantize(16, 0, 2, 32, 0, 24, 16, None) == INVALID and "aligned" in error()
    assert L.tdc_mx8_dequantize(16, 16, 2, 32, None, 0, 0, None) == INVALID and L.tdc_mx8_dequantize(16, None, 2, 32, 16, 0, 0, None) == INVALID
    assert L.tdc_mx8_quantize(None, 0, 0, 32, 0, None, None, None) == 0
    f, n = L.tdc_mx8_linear, ctypes.c_size_t()
    d = ctypes.byref(linear8(x_dtype=0, M=300))
    assert L.tdc_mx8_linear_workspace(d, ctypes.byref(n)) == 0 and n.value >= 300 * (128 + 16)
    assert f(d, 16, None, 16, 16, None, None, 16, 16, n.value - 1, None) == INVALID and "workspace" in error()
    d = ctypes.byref(linear8())
    assert f(d, None, 16, 16, 16, None, None, 16, 16, 0, None) == INVALID and f(d, 16, None, 16, 16, None, None, 16, 16, 0, None) == INVALID
    assert f(d, 16, 16, 16, 8, None, None, 16, 16, 0, None) == INVALID and f(d, 16, 16, 16, 16, None, None, None, 16, 0, None) == INVALID
    assert f(ctypes.byref(linear8(M=0)), None, None, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(C=0), dict(C=8193), dict(rows=1 << 36, C=64), dict(dtype=3), dict(weight_dtype=1), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(x_stride=39), dict(residual_stride=-1), dict(dy_stride=1), dict(dh_stride=39)])
def test_rms_descriptors_are_refused(bad):
    L, d, n = tdc_amd.lib(), rms(**bad), ctypes.c_size_t()
    p = ctypes.byref(d)
    assert L.tdc_rms_norm_workspace(p, ctypes.byref(n)) == INVALID and len(error()) > 15
    assert L.tdc_rms_norm_forward(p, 16, None, None, 16, None, None, None, None, None) == INVALID
    assert L.tdc_rms_norm_forward_mx8(p, 16, None, None, 16, 16, None, None) == INVALID
    assert L.tdc_rms_norm_backward(p, 16, None, None, 16, None, 16, 16, 16, 16, 1 << 30, None) == INVALID


def test_rms_arguments_are_refused():
    L, p, n = tdc_amd.lib(), ctypes.byref(rms()), ctypes.c_size_t()
    assert L.tdc_rms_norm_workspace(p, ctypes.byref(n)) == 0 and n.value >= 40 * 4
    f, e, g = L.tdc_rms_norm_forward, L.tdc_rms_norm_forward_mx8, L.tdc_rms_norm_backward
    assert f(p, None, None, None, 16, None, None, None, None, None) == INVALID and f(p, 16, None, None, None, None, None, None, None, None) == INVALID
    assert f(p, 16, 16, None, 16, None, None, None, None, None) == INVALID and "together" in error()
    assert f(p, 16, None, None, 16, None, None, 16, None, None) == INVALID and "together" in error()
    assert f(p, 16, None, None, 16, None, None, 8, 16, None) == INVALID and "aligned" in error()
    assert e(p, 16, None, None, None, 16, None, None) == INVALID and e(p, 16, None, None, 16, 16, 16, None) == INVALID
    assert g(p, None, None, None, 16, None, 16, 16, None, None, 0, None) == INVALID and g(p, 16, None, None, 16, None, None, 16, None, None, 0, None) == INVALID
    assert g(p, 16, None, None, 16, None, 16, 16, 16, 16, n.value - 1, None) == INVALID and "workspace" in error()
    assert g(p, 16, 8, None, 16, None, 16, 16, None, None, 0, None) == INVALID and "aligned" in error()
    assert f(ctypes.byref(rms(rows=0)), None, None, None, None, None, None, None, None, None) == 0
    assert g(p, None, None, None, None, None, None, None, None, None, 0, None) == 0


def test_python_refusals_without_a_device():
    x, w = torch.zeros(3, 32, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.bfloat16)
    for bad in (lambda: tdc_amd.linear_act(x, w), lambda: tdc_amd.conv1x1_act(x, w), lambda: tdc_amd.mx8_quantize(x), lambda: tdc_amd.rms_norm(x),
                lambda: tdc_amd.rms_norm_mx8(x), lambda: tdc_amd.linear_act([1.0], w)):
        with pytest.raises((TypeError, ValueError)):
            bad()
    with pytest.raises(TypeError, match="Mx8Tensor"):
        tdc_amd.mx8_linear(x, w)
    with pytest.raises(ValueError):
        tdc_amd.Mx8Tensor(torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(1, 3, 16, dtype=torch.uint8), (3, 40))


def test_oracle_of_8_bit_numbers():
    x = np.zeros((2, 40))
    x[0, :6] = [448, 300, 17, 19, 0.001, -464]
    x[0, 32:] = [1.0, 1.0625, 1.1875, -0.3, 0, 0, 0, 0]
    x[1, 5] = np.inf
    v, byte = ref.quantize8(x)
    # scales 1 and 2^-8: 300 lies between 288 and 320, 17 and 19 halfway between even and odd places, 0.001 above half of 2^-9
    assert byte.tolist() == [[127, 119], [255, 0]]
    assert v[0, :6].tolist() == [448, 288, 16, 20, 2.0 ** -9, -448]
    assert v[0, 32:36].tolist() == [1.0, 1.0, 1.25, -0.3125] and np.isnan(v[1, :32]).all() and not v[1, 32:].any()


def test_oracle_gradients_by_differences():
    g = np.random.default_rng(0)
    x, w, b, r, dy = (g.standard_normal(s) for s in ((5, 7), (4, 7), (4,), (5, 4), (5, 4)))
    z, y = ref.linear(x, w, b, r, "silu")
    dz, dx, dw, db = ref.linear_grads(x, w, z, dy, "silu")
    h, wt, dh = g.standard_normal((5, 7)), g.standard_normal(7), g.standard_normal((5, 7))
    u, _, rstd = ref.rms(h, wt, 0.1)
    dn, dwt = ref.rms_grads(u, rstd, wt, dh)

    def slope(f, at, d):
        return (f(at + 1e-6 * d) - f(at - 1e-6 * d)) / 2e-6
    f = lambda *v: (ref.linear(*v, "silu")[1] * dy).sum()  # noqa: E731
    n = lambda *v: (ref.rms(*v, 0.1)[1] * dh).sum()  # noqa: E731
    for got, fn, at in ((dx, lambda v: f(v, w, b, r), x), (dw, lambda v: f(x, v, b, r), w), (db, lambda v: f(x, w, v, r), b),
                        (dz, lambda v: f(x, w, b, v), r), (dn, lambda v: n(v, wt), h), (dwt, lambda v: n(h, v), wt)):
        d = g.standard_normal(at.shape)
        assert abs((got * d).sum() - slope(fn, at, d)) < 1e-7


@pytest.mark.parametrize("act,N,second", [(2, 300, 300 * 304 * 2), (1, 304, 300 * 304 * 2), (0, 300, 300 * 304 * 2), (0, 304, 0)])
def test_the_workspace_of_a_gradient_that_is_given_dz_holds_no_other(act, N, second):
    L, need, given = tdc_amd.lib(), ctypes.c_size_t(), ctypes.c_size_t()
    d = ctypes.byref(linear(M=300, N=N, K=41, act=act))
    assert L.tdc_linear_backward_workspace(d, 0, ctypes.byref(need)) == 0 and need.value == sizes(linear(M=300, N=N, K=41, act=act))[1]
    assert L.tdc_linear_backward_workspace(d, 1, ctypes.byref(given)) == 0
    assert given.value == need.value - (second + 255) // 256 * 256 and given.value > 0
    g = L.tdc_linear_backward
    assert g(d, 16, None, 16, 16, 16, 16, 16, None, 16, 16, given.value - 1, None) == INVALID and "workspace" in error()
    assert g(d, 16, None, 16, 16, 16, 16, 16, None, None, 16, need.value - 1, None) == INVALID and "workspace" in error()
    assert L.tdc_linear_backward_workspace(None, 0, ctypes.byref(need)) == INVALID and L.tdc_linear_backward_workspace(d, 0, None) == INVALID
    assert L.tdc_linear_backward_workspace(ctypes.byref(linear(M=0)), 1, ctypes.byref(need)) == 0 and need.value == 0
