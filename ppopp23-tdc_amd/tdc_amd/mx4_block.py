"""A Tucker block with its factors in 4 bits: the channels-last operators together with the library's core convolution.

    norm -> activation -> first factor -> KxK core -> norm -> activation -> last factor (+ bias, + x)

The two 1x1 factors of a ``TKConv2dC`` (inference/TKConv.py:90-95) are matrix products over pixels and hold most of its
weights; here they run in microscaled 4-bit floating point on tensors whose norm has written them in 4 bits already.  The
core keeps the library's 32-bit kernels.  As a command it times the block next to the same block in 32 bits and says how
far apart they are:

    python -m tdc_amd.mx4_block --batch 32 --size 28 --channels 512 --ranks 128 128
"""
from __future__ import annotations

import threading

import torch
from torch import nn
from torch.nn import functional as F

from .channels_last import _on, group_norm_act, group_norm_act_mx4, mx4_conv1x1, mx4_quantize
from .conv import Conv2dPlan, _raw_stream


class GroupNormAct(nn.Module):
    """``group_norm_act`` with parameters: group norm, scale and shift per channel, activation; trainable."""

    def __init__(self, groups, channels, eps=1e-5, act="none", affine=True):
        super().__init__()
        if channels % groups:
            raise ValueError(f"{groups} groups do not divide {channels} channels")
        self.groups, self.channels, self.eps, self.act = groups, channels, eps, act
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels)) if affine else None

    def forward(self, x):
        return group_norm_act(x, self.groups, self.weight, self.bias, self.eps, self.act)

    def mx4(self, x):
        """The result in 4 bits, for ``mx4_conv1x1``; without a gradient, so that parameters that train need ``torch.no_grad()``."""
        if torch.is_grad_enabled() and any(p.requires_grad for p in self.parameters()):
            raise RuntimeError("the norm into 4 bits has no gradient, and its parameters require one: call it under torch.no_grad()")
        return group_norm_act_mx4(x, self.groups, self.weight, self.bias, self.eps, self.act)

    def extra_repr(self):
        return f"{self.groups}, {self.channels}, eps={self.eps}, act={self.act}"


class TuckerBlockMx4(nn.Module):
    """The block above, for inference, from a ``TKConv2dC`` (stride 1, output as large as the input) and its two norms.

    ``forward`` takes and returns channels-last tensors [batch, channels, height, width]; ``x`` is added to the result where
    the channels agree.  The factors are put into 4 bits, and the core packed, when first used and again when the parameters'
    version counters have moved; writes those do not see (``.data``) need ``invalidate()``.  Threads may share a block: their
    calls queue their work one at a time, and a call on another stream than the last one's waits for that stream on the device (the
    core's scratch belongs to the block).  A captured call waits for nothing outside its graph: its replays must not overlap other
    calls, and neither packing nor ``invalidate()`` may happen in a capture."""

    MAX_CACHED_SHAPES = 8   # plans of the core kept, least recently used first out

    def __init__(self, conv, groups=32, rank_groups=8, act="silu"):
        super().__init__()
        k = conv.kernel_size[0]
        if conv.stride[0] != 1 or 2 * conv.padding[0] != conv.dilation[0] * (k - 1):
            raise ValueError("the convolution has to keep its input's size: stride 1, padding dilation * (kernel - 1) / 2")
        self.conv = conv
        self.norm_in = GroupNormAct(groups, conv.in_channels, act=act)
        self.norm_core = GroupNormAct(rank_groups, conv.out_rank, act=act)
        self._forget()

    def _forget(self):
        self._turn = threading.RLock()      # of the thread whose call compares, packs, queues or closes
        self._factors, self._plans, self._packed, self._stamp = None, {}, None, None
        self._last = None, None      # the last call's stream, as its handle and itself

    def __getstate__(self):      # (a copy packs its own)
        return {k: v for k, v in self.__dict__.items() if k not in ("_turn", "_factors", "_plans", "_packed", "_stamp", "_last")}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._forget()

    def invalidate(self):
        with self._turn:
            if self._factors is not None and self._factors[0].device.type == "cuda":
                torch.cuda.synchronize(self._factors[0].device)      # (streams other than the one they were made on may be reading)
            for plan in self._plans.values():
                plan.close()
            self._factors, self._plans, self._packed, self._stamp = None, {}, None, None

    def _apply(self, fn, *args, **kwargs):
        out = super()._apply(fn, *args, **kwargs)
        self.invalidate()
        return out

    def _core(self, shape):
        plan = self._plans.pop(shape, None)
        if plan is None:
            c, (B, _, H, W) = self.conv, shape
            plan = Conv2dPlan(B, c.in_rank, c.out_rank, H, W, c.kernel_size[0], c.kernel_size[0], 1, c.padding[0],
                              c.dilation[0]).set_weights(c.core_kernel)
            while len(self._plans) >= self.MAX_CACHED_SHAPES:
                self._plans.pop(next(iter(self._plans))).close()
        self._plans[shape] = plan      # most recently used last
        return plan

    @torch.no_grad()
    def forward(self, x):
        with self._turn:
            return _on(x, self._queue, x)      # (the core works on the current device)

    def _queue(self, x):
        c = self.conv
        if x.is_cuda:
            stream = _raw_stream(x.get_device())
            if stream != self._last[0] and not torch.cuda.is_current_stream_capturing():
                now = torch.cuda.current_stream()
                if self._last[1] is not None:
                    now.wait_stream(self._last[1])
                self._last = stream, now
        packed = c.first_kernel, c.core_kernel, c.last_kernel
        stamp = tuple((id(p), p.data_ptr(), p._version) for p in packed)
        if stamp != self._stamp:
            self.invalidate()
            self._factors = mx4_quantize(c.first_kernel.flatten(1)), mx4_quantize(c.last_kernel.flatten(1))
            if x.is_cuda:
                torch.cuda.current_stream().synchronize()      # (whatever stream uses them next)
            self._packed, self._stamp = packed, stamp      # (parameters that are held keep their ids to themselves)
        first, last = self._factors
        h = mx4_conv1x1(self.norm_in.mx4(x), first, out_dtype=torch.float32)
        h = self._core(tuple(h.shape)).forward(h.contiguous())
        h = self.norm_core.mx4(h.contiguous(memory_format=torch.channels_last))
        return mx4_conv1x1(h, last, c.bias, x if c.out_channels == c.in_channels else None, out_dtype=x.dtype)

    @torch.no_grad()
    def plain(self, x):
        """The same block in 32 bits, in torch operations."""
        c, x32 = self.conv, x.float()

        def norm(n, t):
            t = F.group_norm(t, n.groups, n.weight.float(), n.bias.float(), n.eps)
            return F.silu(t) if n.act == "silu" else F.relu(t) if n.act == "relu" else t

        h = F.conv2d(norm(self.norm_in, x32), c.first_kernel)
        h = F.conv2d(h, c.core_kernel, None, 1, c.padding, c.dilation)
        h = F.conv2d(norm(self.norm_core, h), c.last_kernel, c.bias)
        return h + x32 if c.out_channels == c.in_channels else h


def main():
    import argparse
    from .TKConv import TKConv2dC, ranks_dict
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--size", type=int, default=28)
    ap.add_argument("--channels", type=int, default=512)
    ap.add_argument("--ranks", type=int, nargs=2, default=(128, 128), metavar=("OUT", "IN"))
    a = ap.parse_args()
    torch.manual_seed(0)
    conv = TKConv2dC(a.channels, a.channels, 3, padding=1, hp_dict=ranks_dict(conv=list(a.ranks)), name="conv")
    block = TuckerBlockMx4(conv).cuda()
    x = torch.randn(a.batch, a.size, a.size, a.channels, device="cuda").bfloat16().permute(0, 3, 1, 2)
    y, want = block(x), block.plain(x)
    change = torch.linalg.norm(want - x.float())
    print(f"deviation from 32 bits: {float(torch.linalg.norm(y.float() - want) / change):.3f} of what the block adds to x")
    for name, call in (("4-bit factors", block), ("32 bits, torch", block.plain)):
        for _ in range(5):
            call(x)
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(20):
            call(x)
        end.record()
        end.synchronize()
        print(f"{name}: {begin.elapsed_time(end) / 20 * 1000:.1f} us")


if __name__ == "__main__":
    main()
