"""The 16- and 8-bit operators over rows in 64 bits, from their definitions (numpy; test infrastructure)."""
import numpy as np

from .channels_last_ref import act, act_slope

# The magnitudes of E4M3 in the order of their codes: eight multiples of 2^-9, then eight numbers to each power of two.
GRID8 = np.array([n / 512 for n in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])


def quantize8(x):
    """x [..., K]: (codes as the values they stand for, scale bytes [..., blocks]); a block with an infinity or a NaN is NaNs."""
    K = x.shape[-1]
    pad = np.zeros((*x.shape[:-1], -K % 32))
    v = np.concatenate((x, pad), -1).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(v).max(-1)
    bad = ~np.isfinite(top)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.where(bad, 1.0, top))) - 8
    byte = np.where(top == 0, 0, np.maximum(e + 127, 0))
    byte = np.where(bad, 255, byte).astype(np.int64)
    scale = np.exp2(np.where(bad, 0, byte - 127.0))[..., None]
    size = np.abs(np.where(bad[..., None], 0.0, v)) / scale
    halfway = (GRID8[1:] + GRID8[:-1]) / 2
    low, high = np.searchsorted(halfway, size, "left"), np.searchsorted(halfway, size, "right")
    place = np.where(low % 2 == 0, low, high)
    out = np.where(bad[..., None], np.nan, GRID8[place] * scale * np.sign(v))
    return out.reshape(*x.shape[:-1], -1)[..., :K], byte


def linear(x, w, bias, residual, name):
    """(z, act(z)) of rows."""
    z = x @ w.T
    z = z if bias is None else z + bias
    z = z if residual is None else z + residual
    return z, act(z, name)


def linear_grads(x, w, z, dy, name, kept=None):
    """(dz, dx, dw, dbias); `kept`: what stands for x in the weight's gradient."""
    dz = dy * act_slope(z, name)
    return dz, dz @ w, dz.T @ (x if kept is None else kept), dz.sum(0)


def rms(h, weight, eps):
    """(u = h rstd, y, rstd)."""
    rstd = 1 / np.sqrt((h ** 2).mean(-1, keepdims=True) + eps)
    return h * rstd, h * rstd * weight, rstd


def rms_grads(u, rstd, weight, dy, dh=0.0):
    """(dx, dweight)."""
    g = dy * weight
    return rstd * (g - u * (g * u).mean(-1, keepdims=True)) + dh, (dy * u).sum(0)
