"""The host side of head.py and embed.py without a GPU: a recorded library and
stand-ins for device tensors."""
import contextlib
import types

import pytest
import torch

from ark_amd import act, embed, head


class Fake:
    """A contiguous device tensor as far as the modules look at one."""

    def __init__(self, shape, dtype=torch.float16, device=1):
        self.shape, self.dtype = torch.Size(shape), dtype
        self.device = torch.device("cuda", device)
        self.is_cuda, self.requires_grad = True, False

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self):
        st = [1] * len(self.shape)
        for j in range(len(st) - 2, -1, -1):
            st[j] = st[j + 1] * self.shape[j + 1]
        return tuple(st)

    def is_contiguous(self):
        return True

    def view(self, *shape):
        n = self.numel() // -(torch.Size(shape).numel()) if -1 in shape else 0
        return Fake([n if s == -1 else s for s in shape], self.dtype, self.device.index)

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

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(act, "_device", lambda: current[0])
    monkeypatch.setattr(act, "_raw_stream", lambda dev: 700 + dev)
    for m in (act, head, embed):
        monkeypatch.setattr(m, "lib", Lib)
    monkeypatch.setattr(head, "_workspace", lambda *a: 64)
    monkeypatch.setattr(embed, "_workspace", lambda *a: 64)
    return types.SimpleNamespace(calls=calls, current=current)


def _calls(dev):
    x, w = Fake((5, 8), device=dev), Fake((7, 8), device=dev)
    y = Fake((5,), torch.int64, dev)
    index, logits = Fake((5, 3), torch.int32, dev), Fake((5, 3), torch.float32, dev)
    return [("ark_head_cross_entropy", lambda: head.cross_entropy(x, w, y)),
            ("ark_head_cross_entropy_grad", lambda: head.cross_entropy_grad(x, w, y)),
            ("ark_head_distill", lambda: head.distill(x, w, index, logits)),
            ("ark_head_distill_grad", lambda: head.distill_grad(x, w, index, logits)),
            ("ark_embed_lookup", lambda: embed.lookup(w, y)),
            ("ark_embed_grad", lambda: embed.lookup_grad(x, y, 7))]


@pytest.mark.parametrize("dev", [0, 1])
def test_calls_run_on_their_tensors_device(gpus, dev):
    for name, call in _calls(dev):
        call()
        assert gpus.calls.pop() == (name, dev, 700 + dev) and not gpus.calls
        assert gpus.current == [0]


def test_tensors_of_another_device_are_refused(gpus):
    here, there = Fake((5, 8), device=0), Fake((5, 8), device=1)
    w, y, far = Fake((7, 8), device=0), Fake((5,), torch.int64, 0), Fake((5,), torch.int64, 1)
    i, l = Fake((5, 3), torch.int32, 0), Fake((5, 3), torch.float32, 0)
    i1, l1 = Fake((5, 3), torch.int32, 1), Fake((5, 3), torch.float32, 1)
    f32 = Fake((7, 8), torch.float32, 1)
    for call in (lambda: head.cross_entropy(there, w, far), lambda: head.cross_entropy(here, w, far),
                 lambda: head.distill(here, w, i1, l), lambda: head.distill(here, w, i, l1),
                 lambda: head.cross_entropy_grad(here, w, y, grad=torch.ones(5)),
                 lambda: head.cross_entropy_grad(here, w, y, dx=there),
                 lambda: head.cross_entropy_grad(here, w, y, dw=f32),
                 lambda: embed.lookup(w, far), lambda: embed.lookup(w, y, out=there),
                 lambda: embed.lookup_grad(here, far, 7),
                 lambda: embed.lookup_grad(here, y, 7, dw=f32)):
        with pytest.raises((ValueError, TypeError)):
            call()
    assert not gpus.calls


def test_what_would_lose_a_graph_is_refused(gpus):
    x, w, y = Fake((5, 8)), Fake((7, 8)), Fake((5,), torch.int64)
    i, l = Fake((5, 3), torch.int32), Fake((5, 3), torch.float32)
    for t, calls in ((x, (lambda: head.cross_entropy(x, w, y), lambda: head.distill(x, w, i, l))),
                     (w, (lambda: head.cross_entropy(x, w, y), lambda: embed.lookup(w, y))),
                     (l, (lambda: head.distill(x, w, i, l),))):
        t.requires_grad = True
        for call in calls:
            with pytest.raises(ValueError, match="requires grad"):
                call()
            with torch.no_grad():
                call()
        head.cross_entropy_grad(x, w, y)  # gives gradients, not a graph
        t.requires_grad = False


@pytest.mark.parametrize("ignore", [2 ** 31, -2 ** 31 - 1])
def test_an_ignored_target_is_an_int32(gpus, ignore):
    with pytest.raises(ValueError, match="int32"):
        head.cross_entropy(Fake((5, 8)), Fake((7, 8)), Fake((5,), torch.int64), ignore=ignore)


def test_rows_and_tokens_of_no_one_stride_are_refused_by_name():
    """Slices that users take (a sequence without its last token) are no matrix of
    rows, and no list: a refusal of the module's own says so."""
    text, rows = torch.zeros((3, 9), dtype=torch.int64), torch.zeros((3, 9, 8))
    table = torch.zeros((7, 8))
    with pytest.raises(ValueError, match="tokens.*contiguous.*strides"):
        embed.lookup(Table(table), text[:, :-1])
    with pytest.raises(ValueError, match="dy.*contiguous"):
        embed.lookup_grad(rows[:, :-1], text[:, :-1].contiguous(), 7)
    with pytest.raises(ValueError, match="out.*contiguous"):
        embed.lookup(Table(table), text[:, :-1].contiguous(), out=rows[:, :-1])
    for call in (lambda: embed.lookup_grad(torch.zeros(()), text[0, 0], 7),
                 lambda: embed.lookup(Table(table), text[0, 0], out=torch.zeros(()))):
        with pytest.raises(ValueError, match="dy is|out is"):
            call()
    with pytest.raises(ValueError, match="targets.*contiguous"):
        head.cross_entropy(Fake((24, 8)), Fake((7, 8)), text[:, :-1])


class Table(Fake):
    """A table beside host tensors, for what is refused before a call."""

    def __init__(self, like):
        super().__init__(like.shape, like.dtype)
        self.device = like.device
