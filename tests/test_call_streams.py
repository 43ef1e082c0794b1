"""Which stream a call's own tensors are made for, without a GPU: the wrappers run on stand-ins for torch's tensors, streams and
the library, which note the stream that was current at each allocation."""
import contextlib

import pytest
import torch

from inferno_hip import _lib, mixers, quantized_kernels as qk

HERE, THERE = 11, 22  # handles: torch's current stream, the one that is given


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


class World:
    """What is current, what was allocated and recorded, what was launched."""

    def __init__(self):
        self.current, self.made, self.launched, self.next = HERE, [], [], 1 << 20

    @contextlib.contextmanager
    def stream(self, s):
        was, self.current = self.current, s.cuda_stream
        yield
        self.current = was


class Tensor:
    """A contiguous tensor on device 0."""
    is_cuda, device = True, "cuda:0"

    def __init__(self, world, shape, dtype, made=None):
        self.world, self.shape, self.dtype, self.made, self.recorded = world, torch.Size(shape), dtype, made, []
        self.at, world.next = world.next, world.next + (1 << 20)
        if made is not None:
            world.made.append(self)

    def get_device(self): return 0
    def data_ptr(self): return self.at
    def dim(self): return len(self.shape)
    def is_contiguous(self): return True
    def numel(self): return self.shape.numel()
    def stride(self, i=None):
        st = torch.empty(self.shape, device="meta").stride()
        return st if i is None else st[i]
    def new_empty(self, shape, dtype=None):
        return Tensor(self.world, (shape,) if isinstance(shape, int) else shape, dtype or self.dtype, self.world.current)
    def record_stream(self, s): self.recorded.append(s.cuda_stream)


@pytest.fixture
def world(monkeypatch):
    w = World()
    monkeypatch.setattr(torch.cuda, "stream", w.stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(w.current))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(qk, "_raw", lambda device: w.current)
    mixers._torch()
    for name, value in (("_Tensor", Tensor), ("_current_device", lambda: 0), ("_stream_of", lambda device: w.current)):
        monkeypatch.setattr(mixers, name, value)
    monkeypatch.setattr(mixers, "_call", lambda name: lambda *a: w.launched.append((name, a)) or 0)
    return w


def cache(n_seq, cap, heads, d):
    c = mixers.KVCache.__new__(mixers.KVCache)
    c.n_seq, c.capacity, c.n_kv, c.head_dim = n_seq, cap, heads, d
    c._c = _lib.Kv(mixers.F16, n_seq, heads, d, cap, 1 << 30, 1 << 31, cap * heads * d, heads * d, d)
    c._ref, c._dev = mixers.C.byref(c._c), 0
    return c


def calls(w):
    f = lambda *s: Tensor(w, s, torch.float32)  # noqa: E731
    i = lambda *s: Tensor(w, s, torch.int32)  # noqa: E731
    rp = mixers.RopeParams(64)
    return {
        "rope": lambda **kw: mixers.rope(f(6, 128), i(6), 2, rp, **kw),
        "rope_append": lambda **kw: mixers.rope_append(f(6, 8 * 64), 4, cache(2, 9, 2, 64), i(2), rp, **kw),
        "attn_prefix": lambda **kw: mixers.attn_prefix(f(6, 4 * 64), 4, cache(2, 9, 2, 64), i(2), **kw),
        "gated_delta_rule": lambda **kw: mixers.gated_delta_rule(f(2, 70, 1, 64), f(2, 70, 1, 64), f(2, 70, 2, 32),
                                                                 f(2, 70, 2), f(2, 70, 2), None, **kw),
    }


NAMES = ["rope", "rope_append", "attn_prefix", "gated_delta_rule"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("as_handle", [False, True])
def test_on_another_stream(world, name, as_handle):
    """out and ws are made on the stream that the kernels run on; out is known to the current one too."""
    out = calls(world)[name](stream=THERE if as_handle else Stream(THERE))
    assert len(world.launched) == 1 and world.launched[0][1][-1] == THERE
    assert len(world.made) == (2 if name in NAMES[2:] else 1) and [t.made for t in world.made] == [THERE] * len(world.made)
    assert out in world.made and out.recorded == [HERE] and world.current == HERE
    assert all(not t.recorded for t in world.made if t is not out)  # (ws is dropped here: its memory stays the stream's)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("stream", [None, HERE])
def test_on_the_current_stream(world, name, stream):
    out = calls(world)[name](**({} if stream is None else {"stream": Stream(stream)}))
    assert world.launched[0][1][-1] == HERE and [t.made for t in world.made] == [HERE] * len(world.made)
    assert out in world.made and out.recorded == []
