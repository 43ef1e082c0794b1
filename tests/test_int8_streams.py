"""Which stream the 8-bit calls' own tensors are made for, without a GPU: the wrappers run on the stand-ins for torch's tensors,
streams and the library."""
import pytest
import torch

from inferno_hip import _lib, int8

from test_call_streams import HERE, THERE, Lib, Stream, Tensor, Waiting, world  # noqa: F401


@pytest.fixture
def on8(world, monkeypatch):  # noqa: F811
    real = _lib.load()
    size = lambda s: (s,) if isinstance(s, int) else s  # noqa: E731
    made = lambda shape, dtype=None, device=None: Waiting(world, size(shape), dtype, world.current)  # noqa: E731
    for name, value in (("_i8", torch.int8), ("_u8", torch.uint8), ("_f32", torch.float32), ("_Tensor", Tensor),
                        ("_current_device", lambda: 0), ("_stream_of", lambda device: world.current),
                        ("_c_quantize", lambda *a: world.launched.append(("quantize", a)) or 0),
                        ("_c_gemm", lambda *a: world.launched.append(("gemm", a)) or 0)):
        monkeypatch.setattr(int8, name, value)
    monkeypatch.setattr(torch, "empty", made)
    monkeypatch.setattr(torch, "Tensor", Tensor)
    monkeypatch.setattr(_lib, "load", lambda: Lib(world, real))
    return world


def calls(w):
    f = lambda *s: Tensor(w, s, torch.float32)  # noqa: E731
    c = lambda *s: Tensor(w, s, torch.int8)  # noqa: E731
    assert int8.gemm_i8_ws_bytes(515, 1030, 12288)
    return {  # the call, what it returns, what it makes
        "quantize_i8": (lambda **kw: int8.quantize_i8(f(6, 64), **kw), 2, 2),
        "rmsnorm_i8": (lambda **kw: int8.rmsnorm_i8(f(6, 64), f(64), add=f(2, 6, 64), **kw), 2, 2),
        "silu_mul_i8": (lambda **kw: int8.silu_mul_i8(f(6, 128), **kw), 2, 2),
        "gemm_i8": (lambda **kw: int8.gemm_i8(c(515, 12288), f(515), c(1030, 12288), f(1030), **kw), 1, 2),
        "gemm_i8 without parts": (lambda **kw: int8.gemm_i8(c(1, 64), f(1), c(64, 64), f(64), **kw), 1, 1),
    }


NAMES = ["quantize_i8", "rmsnorm_i8", "silu_mul_i8", "gemm_i8", "gemm_i8 without parts"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("stream", [None, HERE, THERE, Stream(THERE)], ids=["none", "current", "handle", "object"])
def test_made_for_the_stream(on8, name, stream):
    """What a call makes, it makes on its kernels' stream; what it returns is known to the current one, its workspace is not."""
    call, returned, made = calls(on8)[name]
    got = call(stream=stream)
    got = got if isinstance(got, tuple) else (got,)
    there = THERE if stream is not None and stream is not HERE and getattr(stream, "cuda_stream", stream) == THERE else HERE
    assert len(got) == returned and len(on8.made) == made and [t.made for t in on8.made] == [there] * made
    assert len(on8.launched) == 1 and on8.launched[0][1][-1] == there and on8.current == HERE
    for t in on8.made:
        back = any(t is g for g in got)
        assert t.recorded == ([HERE] if back and there == THERE else [])


@pytest.mark.parametrize("stream", [None, THERE])
def test_weights(on8, stream, monkeypatch):
    w = Tensor(on8, (4 * 34 * 2,), torch.uint8)
    Tensor.view = lambda self, *s: self if s == (-1,) else Tensor(on8, s, self.dtype)
    Tensor.__getitem__ = lambda self, i: self
    monkeypatch.setattr(Waiting, "__getitem__", lambda self, i: self if not isinstance(i, tuple) else Waiting.cut(self, i))
    Waiting.cut = staticmethod(lambda t, i: setattr(t, "shape", torch.Size((t.shape[0], i[1].stop))) or t)
    try:
        int8.quantize_weights_i8(8, w, 4, 64, stream=stream)
    finally:
        del Tensor.view, Tensor.__getitem__, Waiting.cut
    assert [n for n, _ in on8.launched] == ["ihip_dequant", "quantize"]
    there = HERE if stream is None else THERE
    assert [t.made for t in on8.made] == [there] * 3
    assert all(a[-1] == there or getattr(a[-1], "value", None) == there for _, a in on8.launched)


def test_other_device(on8, monkeypatch):
    """Tensors that are not on the current device, or not on one, are refused by name before any launch."""
    f = lambda *s: Tensor(on8, s, torch.float32)  # noqa: E731
    c = lambda *s: Tensor(on8, s, torch.int8)  # noqa: E731
    far = lambda t: (setattr(t, "get_device", lambda: 1), setattr(t, "device", "cuda:1"), t)[-1]  # noqa: E731
    bad = [lambda: int8.quantize_i8(far(f(2, 64))), lambda: int8.rmsnorm_i8(f(2, 64), far(f(64))),
           lambda: int8.rmsnorm_i8(f(2, 64), add=far(f(2, 64))), lambda: int8.quantize_i8(f(2, 64), out=far(c(2, 64))),
           lambda: int8.quantize_i8(f(2, 64), scales=far(f(2))),
           lambda: int8.gemm_i8(far(c(2, 64)), f(2), c(3, 64), f(3)), lambda: int8.gemm_i8(c(2, 64), far(f(2)), c(3, 64), f(3)),
           lambda: int8.gemm_i8(c(2, 64), f(2), far(c(3, 64)), f(3)), lambda: int8.gemm_i8(c(2, 64), f(2), c(3, 64), far(f(3))),
           lambda: int8.gemm_i8(c(2, 64), f(2), c(3, 64), f(3), out=far(f(2, 3))),
           lambda: int8.gemm_i8(c(2, 64), f(2), c(3, 64), f(3), ws=far(Tensor(on8, (64,), torch.uint8))),
           lambda: int8.quantize_weights_i8(8, far(Tensor(on8, (4 * 68,), torch.uint8)), 4, 64)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert not on8.launched
