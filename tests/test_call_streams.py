"""Which stream a call's own tensors are made for, without a GPU: the wrappers run on stand-ins for torch's tensors, streams and
the library, which note the stream that was current at each allocation."""
import contextlib

import pytest
import torch

from inferno_hip import _lib, gguf, mixers, quantized_kernels as qk, sampler, speculative as sp

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


# ---- the other wrappers: made with torch.empty and torch.zeros, launched through the loaded library ----

class Lib:
    """The library, whose calls are noted and not made, but for those that only work out sizes."""

    def __init__(self, world, real):
        self._world, self._real = world, real

    def __getattr__(self, name):
        if "bytes" in name or ("gguf" in name and "upload" not in name):
            return getattr(self._real, name)
        return lambda *a: self._world.launched.append((name, a)) or 0


class Waiting(Tensor):
    """A tensor whose value the host reads, which waits for the current stream."""

    def __getitem__(self, i):
        return self

    def item(self):
        self.world.waited.append(self.world.current)
        return 0


@pytest.fixture
def others(world, monkeypatch):
    real, size = _lib.load(), lambda s: (s,) if isinstance(s, int) else tuple(s)  # noqa: E731
    make = lambda shape, dtype=None, device=None: Waiting(world, size(shape), dtype, world.current)  # noqa: E731
    world.waited = []
    for name, value in (("empty", make), ("zeros", make), ("Tensor", Tensor),
                        ("empty_like", lambda t: make(t.shape, t.dtype)), ("as_tensor", lambda t: t)):
        monkeypatch.setattr(torch, name, value)
    monkeypatch.setattr(_lib, "load", lambda: Lib(world, real))
    return world


def strides_of(shape):
    out, n = [], 1
    for s in reversed(shape):
        out.insert(0, n)
        n *= s
    return tuple(out)


Tensor.stride = lambda self, i=None: strides_of(self.shape) if i is None else strides_of(self.shape)[i]
Tensor.to = lambda self, device=None, dtype=None: Tensor(self.world, self.shape, dtype, self.world.current)
Tensor.contiguous = lambda self: self
Q8 = qk.Q8_0


def plain_calls(w):
    f = lambda *s: Tensor(w, s, torch.float32)  # noqa: E731
    i = lambda *s: Tensor(w, s, torch.int32)  # noqa: E731
    b = lambda n: Tensor(w, (n,), torch.uint8)  # noqa: E731
    big = b(1 << 22)
    return {
        "gemm_q": (lambda **kw: qk.gemm_q(Q8, big, f(2, 256), 256, 256, **kw), 2),
        "gemm_q_ex": (lambda **kw: qk.gemm_q_ex(Q8, big, f(2, 256), 256, 256, **kw), 2),
        "gemm_q_chain": (lambda **kw: qk.gemm_q_chain(Q8, big, 256, 256, 2, x=f(2, 256), **kw), 1),
        "mlp_forward_": (lambda **kw: qk.mlp_forward_(Q8, big, Q8, big, f(2, 256), 256, 256, **kw), 1),
        "pack_weights": (lambda **kw: qk.pack_weights(Q8, big, 256, 256, **kw), 1),
        "pack_weights_gated": (lambda **kw: qk.pack_weights_gated(Q8, big, 256, 256, **kw), 1),
        "dequant": (lambda **kw: qk.dequant(Q8, big, 4096, **kw), 1),
        "rmsnorm": (lambda **kw: qk.rmsnorm(f(2, 256), **kw), 1),
        "synth_blocks": (lambda **kw: qk.synth_blocks(Q8, 7, 8, **kw), 1),
        "synth_gaussian": (lambda **kw: qk.synth_gaussian(7, 256, **kw), 1),
        "stream_read": (lambda **kw: qk.stream_read(big, **kw), 1),
        "silu_mul": (lambda **kw: qk.silu_mul(f(2, 512), 256, **kw), 1),
        "softmax_sample": (lambda **kw: sampler.softmax_sample(f(2, 5000), f(2), top_k=4, **kw), 2),
        "apply_penalties_": (lambda **kw: sampler.apply_penalties_(f(2, 5000), i(3), **kw), 1),
        "softmax_stats": (lambda **kw: sp.softmax_stats(f(2, 5000), 0.8, **kw), 3),
        "spec_accept": (lambda **kw: sp.spec_accept(f(2, 5, 5000), f(2, 4, 5000), i(2, 4), 0.8, f(2, 4), f(2), f(2), **kw), 3),
        "greedy_verify": (lambda **kw: sp.greedy_verify(f(2, 5, 5000), i(2, 4), **kw), 3),
        "mtp_verify_step": (lambda **kw: sp.mtp_verify_step(f(2, 5, 5000), i(2, 4), **kw), 3),
        "tree_accept": (lambda **kw: sp.tree_accept(f(6, 500), f(6, 500), i(6), i(6), 0.8, f(6), **kw), 3),
    }


PLAIN = ["gemm_q", "gemm_q_ex", "gemm_q_chain", "mlp_forward_", "pack_weights", "pack_weights_gated", "dequant", "rmsnorm",
         "synth_blocks", "synth_gaussian", "stream_read", "silu_mul", "softmax_sample", "apply_penalties_", "softmax_stats",
         "spec_accept", "greedy_verify", "mtp_verify_step", "tree_accept"]


@pytest.mark.parametrize("name", PLAIN)
@pytest.mark.parametrize("stream", [None, HERE, THERE])
def test_other_calls(others, name, stream):
    """Every tensor that a call makes is made, filled and waited for on the stream of its kernels, and what it returns is
    known to the current one."""
    call, n = plain_calls(others)[name]
    on = stream or HERE
    got = call(**({} if stream is None else {"stream": Stream(stream)}))
    assert len(others.launched) == 1 and on in others.launched[0][1]
    assert [t.made for t in others.made] == [on] * n and others.current == HERE
    assert others.waited == ([on] if name in ("mtp_verify_step", "tree_accept") else [])
    for t in got if isinstance(got, tuple) else [got]:
        if t in others.made:
            assert t.recorded == ([HERE] if on == THERE else [])


@pytest.mark.parametrize("stream", [HERE, THERE])
def test_gguf_upload(others, stream, tmp_path):
    path = str(tmp_path / "m.gguf")
    gguf.write_gguf(path, [], [("w", (256,), Q8, b"\0" * (34 * 8))])
    with gguf.read_gguf(path) as f:
        out = f.upload("w", stream=Stream(stream))
    assert out.made == stream and out.recorded == ([HERE] if stream == THERE else [])
