"""The host side of act.py and rope.py without a GPU: a recorded library and
stand-ins for device tensors; and the library's own refusals before any device
call."""
import contextlib
import types

import pytest
import torch

from ark_amd import _abi, _lib, act


class Fake:
    """A contiguous device tensor as far as act.py and rope.py look at one."""

    def __init__(self, shape, dtype=torch.float16, device=1, requires_grad=False):
        self.shape, self.dtype = torch.Size(shape), dtype
        self.device = torch.device("cuda", device)
        self.is_cuda, self.requires_grad = True, requires_grad

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, i=None):
        st = [1] * len(self.shape)
        for j in range(len(st) - 2, -1, -1):
            st[j] = st[j + 1] * self.shape[j + 1]
        return tuple(st) if i is None else st[i]

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device.index

    def data_ptr(self):
        return 4096

    def new_empty(self, shape, dtype=None):
        return Fake((shape,) if isinstance(shape, int) else shape, dtype or self.dtype,
                    self.device.index)


@pytest.fixture
def gpus(monkeypatch):
    """Two devices, the first of them current, and a library that notes, call by
    call, its name, the current device and the stream."""
    calls, current = [], [0]

    @contextlib.contextmanager
    def device(dev):
        before, current[0] = current[0], torch.device("cuda", dev).index
        yield
        current[0] = before

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                calls.append((name, current[0], args[-1]))
                return 0
            return call

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(act, "_device", lambda: current[0])
    monkeypatch.setattr(act, "_raw_stream", lambda dev: 700 + dev)
    monkeypatch.setattr(act, "lib", Lib)
    monkeypatch.setattr(act, "_workspace", lambda *a: 0)
    return types.SimpleNamespace(calls=calls, current=current)


@pytest.mark.parametrize("dev", [0, 1])
def test_act_runs_on_its_tensors_device(gpus, dev):
    x, dy = Fake((64, 8), device=dev), Fake((64, 16), device=dev)
    kept = act.pack(x)
    act.unpack(kept)
    act.weight_grad(kept, dy)
    assert gpus.calls == [(name, dev, 700 + dev) for name in
                          ("ark_act_pack", "ark_act_unpack", "ark_act_weight_grad_noalloc")]
    assert gpus.current == [0]


def test_act8_on_a_device_by_number(monkeypatch):
    where = []
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: where.append(device))
    for given in (None, 0, 1, "cuda:1"):
        act.Act8(32, 4, torch.float16, device=given)
    assert where == ["cuda", 0, 1, "cuda:1"]


@pytest.fixture
def rope(gpus, monkeypatch):
    """A Rope of heads of 8 made on device 0."""
    from ark_amd import rope
    monkeypatch.setattr(rope, "lib", act.lib)
    monkeypatch.setattr(rope, "_raw_stream", act._raw_stream)
    monkeypatch.setattr(rope, "_like", lambda t: t.new_empty(t.shape))
    r = rope.Rope(8)
    gpus.calls.clear()
    return r


def test_rope_refuses_another_device_than_its_own(gpus, rope):
    q = [Fake((5, 2, 8), device=d) for d in (0, 1)]
    k = [Fake((5, 1, 8), device=d) for d in (0, 1)]
    g = [Fake((8,), torch.float32, d) for d in (0, 1)]
    for call in (lambda i: rope.apply(q[i], k[i]), lambda i: rope.apply(q[i]),
                 lambda i: rope.norm(q[i], k[i], g[i], g[i]),
                 lambda i: rope.norm_backward(q[i], k[i], q[i], k[i], g[i], g[i])):
        call(0)
        assert gpus.calls.pop()[1:] == (0, 700) and not gpus.calls
        for current in (0, 1):
            gpus.current[0] = current
            with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
                call(1)
        gpus.current[0] = 0
        assert not gpus.calls


def test_rope_refuses_what_would_lose_a_graph(gpus, rope):
    """Results carry no graph: an input that requires grad is refused while one
    is recorded, and taken under no_grad (as inside an autograd.Function)."""
    q, k, g = Fake((5, 2, 8)), Fake((5, 1, 8)), Fake((8,), torch.float32)
    for t in (q, k, g):
        t.device = torch.device("cuda", 0)
    calls = (lambda: rope.apply(q), lambda: rope.apply(q, k), lambda: rope.norm(q, k, g, g))
    for which, needs in ((q, (1, 1, 1)), (k, (0, 1, 1)), (g, (0, 0, 1))):
        which.requires_grad = True
        for call, need in zip(calls, needs):
            if need:
                with pytest.raises(ValueError, match="requires grad"):
                    call()
            else:
                call()
            with torch.no_grad():
                call()
        which.requires_grad = False
    assert len(gpus.calls) == 9 + 3


@pytest.mark.parametrize("columns,outputs,flags", [(1 << 30, 1, 0), (1, 1 << 30, 2),
                                                   ((1 << 30) + 7, 3, 0), (1 << 20, 1 << 24, 0)])
def test_weight_grad_refuses_more_blocks_than_a_launch_holds(columns, outputs, flags):
    """A launch holds fewer than 2^32 lanes: 64 x 64 outputs' blocks have 512."""
    L = _lib.lib()
    gb = 1 << 40
    rc = L.ark_act_weight_grad(gb, _abi.ACT_F16, 32, columns, 100 * gb, outputs, _abi.ACT_F16,
                               outputs, 200 * gb, columns if flags else outputs, flags, None)
    assert rc == _abi.EINVAL and "too large" in L.ark_opt_last_error().decode()


@pytest.mark.parametrize("columns", [2, 700])
def test_packing_refuses_more_groups_than_a_launch_holds(columns):
    """65535 x 32768 groups of 32 tokens."""
    L = _lib.lib()
    gb, t = 1 << 50, (65535 * 32768 + 1) * 32
    for rc in (L.ark_act_pack(gb, 0, _abi.ACT_F16, t, columns, 3 * gb, None),
               L.ark_act_unpack(3 * gb, t, columns, _abi.ACT_F16, gb, columns, None)):
        assert rc == _abi.EINVAL and "too large" in L.ark_opt_last_error().decode()
