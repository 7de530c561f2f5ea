"""What the channels-last operators refuse (no GPU needed), and their 64-bit oracle against hand-worked numbers."""
import copy
import ctypes
import pickle
import threading

import numpy as np
import pytest
import torch

import tdc_amd
from oracle import channels_last_ref as ref
from tdc_amd import _lib
from tdc_amd.channels_last import _dense_strides, _pixel_strides

INVALID = _lib.TDC_ERR_INVALID


def norm(**kw):
    d = dict(batch=2, C=8, groups=2, act=0, dtype=0, param_dtype=0, eps=1e-5, reserved=0, pixels=9, x_pixel_stride=0, x_image_stride=0,
             y_pixel_stride=0, y_image_stride=0)
    d.update(kw)
    return _lib.GroupNormDesc(*[d[n] for n, _ in _lib.GroupNormDesc._fields_])


def linear(**kw):
    d = dict(M=4, N=5, K=40, x_dtype=0, y_dtype=0, bias_dtype=0, act=0, x_stride=0, y_stride=0, residual_stride=0)
    d.update(kw)
    return _lib.Mx4LinearDesc(*[d[n] for n, _ in _lib.Mx4LinearDesc._fields_])


def error():
    return tdc_amd.lib().tdc_last_error_string().decode()


def test_struct_layouts():
    assert ctypes.sizeof(_lib.GroupNormDesc) == 8 * 4 + 5 * 8
    assert ctypes.sizeof(_lib.Mx4LinearDesc) == 3 * 8 + 4 * 4 + 3 * 8


@pytest.mark.parametrize("bad,word", [
    (dict(C=0), "C"), (dict(groups=3), "divide"), (dict(groups=0), "divide"), (dict(batch=-1), "batch"), (dict(pixels=-1), "pixels"),
    (dict(pixels=1 << 31), "2^31"), (dict(dtype=3), "dtype"), (dict(dtype=1, param_dtype=2), "param_dtype"), (dict(act=3), "activation"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x_pixel_stride=7), "pixel stride"), (dict(x_image_stride=71), "image stride"),
    (dict(y_pixel_stride=-8), "pixel stride"), (dict(y_image_stride=8), "image stride"), (dict(reserved=1), "reserved")])
def test_norm_descriptors_are_refused(bad, word):
    L, d, a, b = tdc_amd.lib(), norm(**bad), ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tdc_group_norm_workspace(ctypes.byref(d), ctypes.byref(a), ctypes.byref(b)) == INVALID and word in error()
    assert L.tdc_group_norm_forward(ctypes.byref(d), 16, None, None, 16, None, None, 16, 1 << 20, None) == INVALID
    assert L.tdc_group_norm_backward(ctypes.byref(d), 16, 16, None, None, 16, 16, 16, None, None, 16, 1 << 30, None) == INVALID
    assert L.tdc_group_norm_forward_mx4(ctypes.byref(d), 16, None, None, 16, 16, 16, 1 << 30, None) == INVALID


def test_norm_arguments_are_refused():
    L, d, a, b = tdc_amd.lib(), norm(pixels=1 << 20), ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tdc_group_norm_workspace(None, ctypes.byref(a), ctypes.byref(b)) == INVALID
    assert L.tdc_group_norm_workspace(ctypes.byref(d), ctypes.byref(a), ctypes.byref(b)) == 0 and 0 < a.value < b.value
    p = ctypes.byref(d)
    assert L.tdc_group_norm_forward(p, None, None, None, 16, None, None, 16, a, None) == INVALID
    assert L.tdc_group_norm_forward(p, 16, None, None, None, None, None, 16, a, None) == INVALID
    assert L.tdc_group_norm_forward(p, 16, None, None, 16, None, None, None, a, None) == INVALID
    assert L.tdc_group_norm_forward(p, 16, None, None, 16, None, None, 16, a.value - 1, None) == INVALID and "workspace" in error()
    assert L.tdc_group_norm_forward(p, 16, None, None, 16, None, None, 8, a, None) == INVALID and "aligned" in error()
    assert L.tdc_group_norm_backward(p, 16, 16, None, None, None, 16, 16, None, None, 16, b, None) == INVALID
    assert L.tdc_group_norm_forward_mx4(p, 16, None, None, 8, 16, 16, b, None) == INVALID and "aligned" in error()
    # nothing to do is no error, whatever the pointers
    assert L.tdc_group_norm_forward(ctypes.byref(norm(batch=0)), None, None, None, None, None, None, None, 0, None) == 0
    assert L.tdc_group_norm_backward(p, None, None, None, None, None, None, None, None, None, None, 0, None) == 0


def test_4_bit_arguments_are_refused():
    L, c, s = tdc_amd.lib(), ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tdc_mx4_sizes(3, 130, ctypes.byref(c), ctypes.byref(s)) == 0 and (c.value, s.value) == (32 * 128, 3 * 16)
    for rows, K in ((-1, 4), (2, 0), (1 << 36, 64), (2, 1 << 31)):
        assert L.tdc_mx4_sizes(rows, K, ctypes.byref(c), ctypes.byref(s)) == INVALID
    assert L.tdc_mx4_quantize(16, 3, 2, 32, 0, 16, 16, None) == INVALID and "dtype" in error()
    assert L.tdc_mx4_quantize(16, 0, 2, 32, 31, 16, 16, None) == INVALID and "stride" in error()
    assert L.tdc_mx4_quantize(None, 0, 2, 32, 0, 16, 16, None) == INVALID
    assert L.tdc_mx4_quantize(16, 0, 2, 32, 0, 24, 16, None) == INVALID and "aligned" in error()
    assert L.tdc_mx4_quantize(16, 0, 2, 32, 0, 16, 18, None) == INVALID
    assert L.tdc_mx4_dequantize(16, 16, 2, 32, None, 0, 0, None) == INVALID
    assert L.tdc_mx4_dequantize(16, None, 2, 32, 16, 0, 0, None) == INVALID
    assert L.tdc_mx4_quantize(None, 0, 0, 32, 0, None, None, None) == 0


@pytest.mark.parametrize("bad", [dict(M=-1), dict(N=-1), dict(K=0), dict(x_dtype=4), dict(y_dtype=3), dict(y_dtype=1, bias_dtype=2), dict(act=-1),
                                 dict(x_stride=39), dict(y_stride=4), dict(residual_stride=-5), dict(M=1 << 30, N=1 << 30)])
def test_product_descriptors_are_refused(bad):
    L, n, d = tdc_amd.lib(), ctypes.c_size_t(), linear(**bad)
    assert L.tdc_mx4_linear_workspace(ctypes.byref(d), ctypes.byref(n)) == INVALID and len(error()) > 15
    assert L.tdc_mx4_linear(ctypes.byref(d), 16, None, 16, 16, None, None, 16, 16, 1 << 20, None) == INVALID


def test_product_arguments_are_refused():
    L, n, d = tdc_amd.lib(), ctypes.c_size_t(), linear()
    assert L.tdc_mx4_linear_workspace(ctypes.byref(d), ctypes.byref(n)) == 0
    assert L.tdc_mx4_linear(ctypes.byref(d), None, None, 16, 16, None, None, 16, 16, n, None) == INVALID
    assert L.tdc_mx4_linear(ctypes.byref(d), 16, None, 16, 16, None, None, None, 16, n, None) == INVALID
    assert L.tdc_mx4_linear(ctypes.byref(d), 16, None, 16, None, None, None, 16, 16, n, None) == INVALID
    if n.value:
        assert L.tdc_mx4_linear(ctypes.byref(d), 16, None, 16, 16, None, None, 16, None, 0, None) == INVALID
    q = linear(x_dtype=3)
    assert L.tdc_mx4_linear(ctypes.byref(q), 16, None, 16, 16, None, None, 16, None, 0, None) == INVALID
    assert L.tdc_mx4_linear(ctypes.byref(linear(M=0)), None, None, None, None, None, None, None, None, 0, None) == 0


def test_python_refusals_without_a_device():
    x = torch.zeros(2, 8, 3, 3).contiguous(memory_format=torch.channels_last)
    with pytest.raises(ValueError, match="device tensor"):
        tdc_amd.group_norm_act(x, 2)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        tdc_amd.group_norm_act(x.double(), 2)
    with pytest.raises(ValueError, match="device tensor"):
        tdc_amd.mx4_quantize(x)
    with pytest.raises(TypeError, match="has to be a tensor"):
        tdc_amd.mx4_quantize([1.0])
    with pytest.raises(TypeError, match="Mx4Tensor"):
        tdc_amd.mx4_linear(x, torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="no gradient"):
        tdc_amd.group_norm_act_mx4(x.requires_grad_(), 2)
    with pytest.raises(ValueError, match="uint8 device tensor"):
        tdc_amd.Mx4Tensor(torch.zeros(1, 1, 4, 32, 16, dtype=torch.uint8), torch.zeros(1, 2, 16, dtype=torch.uint8), (2, 128))


def test_channels_last_is_recognised():
    def of(t):
        return _pixel_strides(tuple(t.shape), t.stride())
    t = torch.zeros(2, 5, 6, 8)
    assert of(t.permute(0, 3, 1, 2)) == (30, 8, 240)
    assert of(t) is None
    assert of(t.permute(0, 3, 1, 2)[:, 2:6]) == (30, 8, 240)
    assert of(t.permute(0, 3, 1, 2)[:, :, ::2]) is None                       # rows skipped
    assert of(t.permute(0, 3, 1, 2)[:, :, :, ::2]) == (15, 16, 240)           # columns skipped: still evenly spaced
    assert of(torch.zeros(4, 7, 1, 1)) == (1, 7, 7)
    assert of(torch.zeros(4, 1, 3, 5)) == (15, 1, 15)
    assert of(torch.zeros(1, 8, 1, 1).expand(4, 8, 3, 3)) is None
    assert of(torch.zeros(1, 3, 3, 8).permute(0, 3, 1, 2).expand(4, 8, 3, 3)) is None
    assert _dense_strides((2, 8, 5, 6)) == (240, 1, 48, 8)
    assert _dense_strides((3, 4)) == (4, 1)


def test_oracle_of_4_bit_numbers():
    x = np.zeros((1, 40))
    x[0, :10] = [6, 5, 3.5, 2.5, 1.75, 0.75, 0.25, -0.25, -5.1, 7.9]
    x[0, 32:35] = [0.1, -0.05, 0.0]
    codes, byte, values = ref.mx4(x)
    assert byte.tolist() == [[127, 127 - 6]]
    assert values[0, :10].tolist() == [6, 4, 4, 2, 2, 1, 0, 0, -6, 6]
    assert codes[0, :10].tolist() == [7, 6, 6, 4, 4, 2, 0, 8, 15, 7]
    assert values[0, 32:35].tolist() == [6 / 64, -3 / 64, 0]      # 0.1 * 64 = 6.4, 0.05 * 64 = 3.2


def test_copies_of_a_4_bit_tensor_have_their_own_addresses():
    """What kernels are handed is where a copy's own bytes lie, not where the original's lay."""
    q = tdc_amd.Mx4Tensor._new(6, 200, (2, 3, 200), torch.device("cpu"), -1)
    q._held.random_(0, 255, generator=torch.Generator().manual_seed(1))
    for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q)), copy.deepcopy(pickle.loads(pickle.dumps(q)))):
        assert (other.shape, other.rows, other.K, other.device) == (q.shape, 6, 200, q.device)
        assert torch.equal(other.codes, q.codes) and torch.equal(other.scales, q.scales)
        assert other._codes_at == other.codes.data_ptr() and other._scales_at == other.scales.data_ptr()
    assert copy.deepcopy(q)._codes_at != q._codes_at


# ---- the block's host side, with stand-ins for everything that needs a device ----

class StandIn:
    """The block's operators and plans on the host; `calls` names them in order, `at[name]` runs inside the call of that name."""

    def __init__(self, monkeypatch):
        from tdc_amd import mx4_block
        self.calls, self.at, self.plans = [], {}, []
        outer = self

        def said(name):
            outer.calls.append(name)
            outer.at.get(name, lambda: None)()

        class Plan:
            def __init__(self, B, C, N, H, W, *rest):
                self.open, self.shape, self._h = True, (B, N, H, W), ctypes.c_void_p(1)
                outer.plans.append(self)

            def set_weights(self, w):
                said("set_weights")
                return self

            def forward(self, x):
                said("core")
                assert self.open, "the plan was closed while it was in use"
                return torch.zeros(self.shape)

            def close(self):
                said("close")
                self.open = False

        def product(x, w, bias=None, residual=None, out_dtype=None):
            said("product")
            return torch.zeros(x.shape[0], w.shape[0], *x.shape[2:])

        def quantize(w):
            said("quantize")
            return w.clone()

        for name, value in (("Conv2dPlan", Plan), ("mx4_conv1x1", product), ("mx4_quantize", quantize)):
            monkeypatch.setattr(mx4_block, name, value)
        monkeypatch.setattr(mx4_block.GroupNormAct, "mx4", lambda norm, x: x)
        conv = tdc_amd.TKConv2dC(8, 8, 3, padding=1, hp_dict=tdc_amd.ranks_dict(conv=[4, 4]), name="conv")
        self.block = tdc_amd.TuckerBlockMx4(conv, groups=2, rank_groups=2)
        self.x = torch.zeros(2, 8, 5, 5).contiguous(memory_format=torch.channels_last)


def in_threads(*bodies):
    """Runs them, each in a thread; their errors."""
    errors = []

    def guarded(body):
        try:
            body()
        except BaseException as e:  # noqa: B036
            errors.append(e)

    threads = [threading.Thread(target=guarded, args=(b,)) for b in bodies]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
        assert not t.is_alive()
    return errors


def test_block_is_built_once_for_two_threads(monkeypatch):
    s, inside, second = StandIn(monkeypatch), threading.Event(), threading.Event()

    def first_factor():
        inside.set()
        second.wait(0.5)      # (the other thread comes meanwhile, and is held or goes wrong)

    s.at["quantize"] = first_factor

    def other():
        assert inside.wait(10)
        s.block(s.x)
        second.set()

    assert in_threads(lambda: s.block(s.x), other) == []
    assert s.calls.count("quantize") == 2 and s.calls.count("core") == 2 and len(s.plans) == 1


def test_block_is_not_invalidated_under_a_call(monkeypatch):
    s, inside, done = StandIn(monkeypatch), threading.Event(), threading.Event()
    s.block(s.x)

    def core():
        inside.set()
        done.wait(0.5)

    s.at["core"] = core

    def other():
        assert inside.wait(10)
        s.block.invalidate()
        done.set()

    assert in_threads(lambda: s.block(s.x), other) == []
    assert not s.plans[0].open
    s.block(s.x)
    assert len(s.plans) == 2 and s.plans[1].open


def test_block_that_could_not_be_built_is_built_by_the_next_call(monkeypatch):
    s = StandIn(monkeypatch)

    def fails():
        del s.at["quantize"]
        raise MemoryError

    s.at["quantize"] = fails
    with pytest.raises(MemoryError):
        s.block(s.x)
    assert s.block(s.x).shape == (2, 8, 5, 5)


def test_block_is_copied_without_what_it_keeps(monkeypatch):
    s = StandIn(monkeypatch)
    s.block(s.x)
    other = copy.deepcopy(s.block)
    assert other(s.x).shape == (2, 8, 5, 5) and len(s.plans) == 2 and s.plans[0].open
    s.block(s.x)
    assert len(s.plans) == 2


def test_block_sees_another_parameter_in_the_same_place(monkeypatch):
    """A new parameter may lie where the old one lay, with the same version."""
    s, held = StandIn(monkeypatch), np.zeros((4, 8, 1, 1), np.float32)
    s.block.conv.first_kernel = torch.nn.Parameter(torch.from_numpy(held))
    s.block(s.x)
    held += 1
    s.block.conv.first_kernel = torch.nn.Parameter(torch.from_numpy(held))
    s.block(s.x)
    assert s.calls.count("quantize") == 4
    s.block(s.x)
    assert s.calls.count("quantize") == 4


class OnDevice(torch.Tensor):
    """A host tensor that says it lies on the second device."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", 1))

    def get_device(self):
        return 1


class Streams:
    """Streams of a device by their numbers: what waits for what is noted among the stand-in's calls."""

    def __init__(self, monkeypatch, s):
        from tdc_amd import mx4_block
        self.now, self.capturing = 1, False
        outer = self

        class Stream:
            def __init__(self, number):
                self.number = number

            def synchronize(self):
                s.calls.append(f"host waits for {self.number}")

            def wait_stream(self, other):
                s.calls.append(f"{self.number} waits for {other.number}")

        monkeypatch.setattr(mx4_block, "_raw_stream", lambda device: outer.now, raising=False)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(outer.now))
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: outer.capturing)
        monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: s.calls.append("host waits for all"))
        product, quantize = mx4_block.mx4_conv1x1, mx4_block.mx4_quantize
        monkeypatch.setattr(mx4_block, "mx4_quantize", lambda w: quantize(w).detach().as_subclass(OnDevice))
        monkeypatch.setattr(mx4_block, "mx4_conv1x1", lambda *a, **k: product(*a, **k).as_subclass(OnDevice))


def test_block_works_on_the_device_of_its_input(monkeypatch):
    from tdc_amd import channels_last
    s, current = StandIn(monkeypatch), [0]
    Streams(monkeypatch, s)

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *error):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(channels_last, "_device", lambda: current[0])
    seen = []
    for name in ("set_weights", "core"):
        s.at[name] = lambda: seen.append(current[0])
    s.block(s.x.as_subclass(OnDevice))
    assert seen == [1, 1] and current == [0]


def test_block_is_ordered_across_streams(monkeypatch):
    """Factors are there for every stream before the first one uses them; a call on another stream than the last one's waits for it, for
    the core's scratch is theirs in turn; nothing is freed that a stream may still read.  A capture cannot wait for what lies outside."""
    from tdc_amd import mx4_block
    s = StandIn(monkeypatch)
    streams = Streams(monkeypatch, s)
    monkeypatch.setattr(mx4_block, "_on", lambda t, call, *args: call(*args))
    x = s.x.as_subclass(OnDevice)

    def calls(now, capturing=False):
        s.calls.clear()
        streams.now, streams.capturing = now, capturing
        s.block(x)
        return s.calls

    c = calls(1)
    assert max(i for i, n in enumerate(c) if n == "quantize") < c.index("host waits for 1") < c.index("product")
    assert calls(1) == ["product", "core", "product"]
    assert calls(2) == ["2 waits for 1", "product", "core", "product"]
    assert calls(2) == ["product", "core", "product"]
    assert calls(7, capturing=True) == ["product", "core", "product"]
    assert calls(1) == ["1 waits for 2", "product", "core", "product"]
    s.calls.clear()
    s.block.invalidate()
    assert s.calls[0] == "host waits for all" and "close" in s.calls


# ---- sizes that no launch can have ----

def test_4_bit_numbers_of_more_rows_than_a_launch_has():
    """A launch has fewer than 2^32 work items: 16 rows (and 512 numbers of each) take 256."""
    L, c, s = tdc_amd.lib(), ctypes.c_size_t(), ctypes.c_size_t()
    for rows, K in (((1 << 28) - 15, 32), ((1 << 27) - 15, 513), (1 << 28, 512), (1 << 33, 128), ((1 << 26) - 15, 2000)):
        for call in (lambda: L.tdc_mx4_sizes(rows, K, ctypes.byref(c), ctypes.byref(s)), lambda: L.tdc_mx4_quantize(16, 1, rows, K, 0, 16, 16, None),
                     lambda: L.tdc_mx4_dequantize(16, 16, rows, K, 16, 1, 0, None)):
            assert call() == INVALID and "2^32" in error(), (rows, K)
    for rows, K in (((1 << 28) - 16, 512), ((1 << 27) - 16, 513), ((1 << 26) - 16, 2000)):
        assert L.tdc_mx4_sizes(rows, K, ctypes.byref(c), ctypes.byref(s)) == 0
        assert c.value >= rows * K // 2


@pytest.mark.parametrize("desc", [dict(batch=1 << 26, C=2048, groups=32, dtype=2, pixels=1), dict(batch=1 << 24, C=16, groups=2, pixels=1 << 16),
                                  dict(batch=(1 << 31) - 1, C=8, groups=1, pixels=1),
                                  dict(batch=(1 << 31) - 1, C=1 << 23, groups=1, pixels=(1 << 31) - 1),
                                  dict(batch=1 << 16, C=1 << 23, groups=1 << 23, pixels=(1 << 31) - 1)])
def test_norms_of_more_workgroups_than_a_launch_has(desc):
    L, d, a, b = tdc_amd.lib(), norm(**desc), ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tdc_group_norm_workspace(ctypes.byref(d), ctypes.byref(a), ctypes.byref(b)) == INVALID and "too large" in error()
    assert L.tdc_group_norm_mx4_workspace(ctypes.byref(d), ctypes.byref(a)) == INVALID and "too large" in error()
    assert L.tdc_group_norm_forward(ctypes.byref(d), 16, None, None, 16, None, None, 16, 1 << 60, None) == INVALID
    assert L.tdc_group_norm_forward_mx4(ctypes.byref(d), 16, None, None, 16, 16, 16, 1 << 60, None) == INVALID
    assert L.tdc_group_norm_backward(ctypes.byref(d), 16, 16, None, None, 16, 16, 16, None, None, 16, 1 << 60, None) == INVALID


@pytest.mark.parametrize("desc", [dict(M=8, N=1 << 31, K=32, x_dtype=1), dict(M=1 << 31, N=64, K=512, x_dtype=3),
                                  dict(M=1 << 29, N=64, K=64, x_dtype=2), dict(M=1 << 33, N=64, K=8192, x_dtype=3)])
def test_products_of_more_tiles_than_a_launch_has(desc):
    L, n, d = tdc_amd.lib(), ctypes.c_size_t(), linear(**desc)
    assert L.tdc_mx4_linear_workspace(ctypes.byref(d), ctypes.byref(n)) == INVALID and "2^32" in error()
    assert L.tdc_mx4_linear(ctypes.byref(d), 16, 16, 16, 16, None, None, 16, 16, 1 << 60, None) == INVALID


def test_products_of_more_outputs_than_64_bits_count():
    L, n = tdc_amd.lib(), ctypes.c_size_t()
    for size in (1 << 32, 1 << 34):
        d = linear(M=size, N=size)
        assert L.tdc_mx4_linear_workspace(ctypes.byref(d), ctypes.byref(n)) == INVALID and "2^40" in error()


@pytest.mark.parametrize("desc", [dict(batch=1 << 25, C=64, groups=8, dtype=2, pixels=1), dict(batch=(1 << 26) - 1, C=16, groups=2, pixels=1),
                                  dict(batch=1, C=(1 << 24) - 1, groups=1, pixels=1)])
def test_norms_of_nearly_as_many_work_items_as_a_launch_has(desc):
    L, d, a, b = tdc_amd.lib(), norm(**desc), ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tdc_group_norm_workspace(ctypes.byref(d), ctypes.byref(a), ctypes.byref(b)) == 0
    assert L.tdc_group_norm_mx4_workspace(ctypes.byref(d), ctypes.byref(a)) == 0
