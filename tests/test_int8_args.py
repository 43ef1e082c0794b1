"""The 8-bit projections' argument checks, without a GPU (calls that fail before any launch)."""
import ctypes as C

import pytest

from inferno_hip import _lib as L


@pytest.fixture(scope="module")
def lib():
    return L.load()


BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 63) & ~63


def quant(lib, x=P, ldx=64, act=0, norm_w=None, eps=1e-6, add=None, n_add=0, stride=0, m=2, k=64, q=P, ldq=64, scale=P):
    a = L.GemmInput(x, ldx, act, norm_w, eps, add, n_add, stride)
    return lib.ihip_quantize_i8(C.byref(a), m, k, q, ldq, scale, None)


@pytest.mark.parametrize("kw,rc", [
    ({"x": None}, -14), ({"q": None}, -14), ({"scale": None}, -14),
    ({"act": 3}, -22), ({"act": -1}, -22), ({"m": 0}, -22), ({"m": (1 << 23) + 1}, -22),
    ({"k": 0}, -22), ({"k": 8}, -22), ({"k": 40, "ldx": 40}, -22), ({"k": 65552, "ldx": 65552, "ldq": 65552}, -22),
    ({"ldq": 48}, -22), ({"ldq": 72}, -22), ({"q": P + 4}, -22), ({"scale": P + 2}, -22),
    ({"ldx": 60}, -22), ({"ldx": 66}, -22), ({"x": P + 4}, -22), ({"act": 2, "ldx": 124}, -22),
    ({"act": 1, "eps": -1.0}, -22), ({"act": 1, "eps": float("nan")}, -22), ({"act": 1, "norm_w": P + 4}, -22),
    ({"add": P, "n_add": 0}, -22), ({"add": P, "n_add": 2, "stride": 64}, -22), ({"add": P + 4, "n_add": 1}, -22),
    ({"add": P, "n_add": 2, "stride": 130}, -22), ({"add": P, "n_add": 1, "act": 2, "ldx": 128}, -22),
    ({"x": None, "add": P, "n_add": 2, "ldx": 80, "stride": 128}, -22)])
def test_quantize_refusals(lib, kw, rc):
    assert quant(lib, **kw) == rc, kw
    assert b"ihip_quantize_i8" in lib.ihip_last_error()


def gemm(lib, x=P, ldx=64, xs=P, w=P, ldw=64, ws=P, y=P, ldy=8, m=4, n=8, k=64, flags=0, space=None, size=0):
    return lib.ihip_gemm_i8(x, ldx, xs, w, ldw, ws, y, ldy, m, n, k, flags, space, size, None)


@pytest.mark.parametrize("kw,rc", [
    ({"x": None}, -14), ({"xs": None}, -14), ({"w": None}, -14), ({"ws": None}, -14), ({"y": None}, -14),
    ({"m": 0}, -22), ({"n": 0}, -22), ({"m": -3}, -22), ({"m": (1 << 23) + 1}, -22), ({"n": (1 << 23) + 1, "ldy": 1 << 24}, -22),
    ({"m": 1 << 20, "n": 1 << 20, "ldy": 1 << 20}, -22),
    ({"k": 0}, -22), ({"k": 24}, -22), ({"k": 65552, "ldx": 65552, "ldw": 65552}, -22),
    ({"ldx": 48}, -22), ({"ldw": 48}, -22), ({"ldx": 72}, -22), ({"ldw": 72}, -22), ({"x": P + 8}, -22), ({"w": P + 8}, -22),
    ({"ldy": 7}, -22), ({"y": P + 1}, -22), ({"xs": P + 1}, -22), ({"ws": P + 2}, -22),
    ({"flags": 1}, -22), ({"flags": 8}, -22), ({"flags": 4 | 32}, -22)])
def test_gemm_refusals(lib, kw, rc):
    assert gemm(lib, **kw) == rc, kw
    assert b"ihip_gemm_i8" in lib.ihip_last_error()


def test_ws_bytes(lib):
    nb = C.c_size_t(7)
    assert lib.ihip_gemm_i8_ws_bytes(5, 100, 256, 0, None) == -14
    for bad in ((0, 1, 64, 0), (1, 0, 64, 0), (1, 1, 20, 0), (1, 1, 64, 2)):
        assert lib.ihip_gemm_i8_ws_bytes(*bad, C.byref(nb)) == -22
    for m, n, k in ((1, 1, 16), (5, 4096, 12288), (515, 4096, 4096), (4096, 24576, 4096), (1 << 23, 1, 16)):
        assert lib.ihip_gemm_i8_ws_bytes(m, n, k, 4, C.byref(nb)) == 0 and nb.value < 1 << 32
        if nb.value:  # a workspace short of that, or none, is refused before any launch
            ld = (k + 15) // 16 * 16
            assert gemm(lib, ldx=ld, ldw=ld, ldy=n, m=m, n=n, k=k, flags=4, space=P, size=nb.value - 1) == -12
            assert gemm(lib, ldx=ld, ldw=ld, ldy=n, m=m, n=n, k=k, flags=4) == -14


def test_python_refusals():
    """Host tensors and other types are refused by name before the library is reached."""
    import torch

    import inferno_hip as ih
    x, q, s = torch.zeros(2, 64), torch.zeros((2, 64), dtype=torch.int8), torch.zeros(2)
    for f in (ih.quantize_i8, ih.rmsnorm_i8, ih.silu_mul_i8):
        with pytest.raises(ValueError, match="x must be a GPU tensor"):
            f(x)
        with pytest.raises(ValueError, match="rows"):
            f(x[0])
    with pytest.raises(ValueError, match="65 columns"):
        ih.silu_mul_i8(torch.zeros(2, 65))
    with pytest.raises(ValueError, match="q must be a GPU tensor"):
        ih.gemm_i8(q, s, q, s)
    with pytest.raises(ValueError, match="q must be a torch tensor"):
        ih.gemm_i8(None, s, q, s)
    with pytest.raises(ValueError, match="whole blocks"):
        ih.quantize_weights_i8(12, q, 2, 64)
    assert ih.gemm_i8_ws_bytes(1, 16, 64) >= 0
