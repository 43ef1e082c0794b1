"""The 8-bit projections of prompts and single tokens: rows of the residual
stream, of [gate | up] or of the mixers' output as 8-bit codes with a scale for
each row (the RMSNorm, gating and residual adds of src/ModelCPU.jl:110-122,
:447-473, :870-891), and their products with 8-bit weights (:284-378), past the
64 rows that gemm_q takes. (Up to those, gemm_q on GGUF weights is about as fast
or faster and more exact; these calls take any number of rows.)

Kernels run on `stream` (default: torch's current one). What a call allocates
itself (codes, scales, out, ws) is made for that stream; its inputs have to be
ready there, and other streams wait for it before they read its outputs. A
workspace that is given serves one call at a time.
"""
from __future__ import annotations

import ctypes as C
from struct import Struct

from . import _lib
from .formats import BLOCK_BYTES, BLOCK_ELEMS
from .mixers import _device_of, _refuse, _rows, _torch, _whole, _workspace
from .quantized_kernels import ACT_PLAIN, ACT_RMSNORM, ACT_SILU_MUL, GEMM_ACCUM, _raw_stream, check_tensor, dequant, made_for

_i8 = _u8 = _f32 = _Tensor = _current_device = _stream_of = _c_quantize = _c_gemm = None
_INPUT = Struct("@PiiPfPiq").pack  # ihip_gemm_input (host time is most of a small call: a ctypes Structure takes longer)


def _names():
    """torch's and the library's names, looked up once."""
    global _i8, _u8, _f32, _Tensor, _current_device, _stream_of, _c_quantize, _c_gemm
    import torch
    _torch()
    lib = _lib.load()
    _c_quantize, _c_gemm = lib.ihip_quantize_i8, lib.ihip_gemm_i8
    _current_device, _stream_of, _Tensor = torch.cuda.current_device, _raw_stream(), torch.Tensor
    _u8, _f32 = torch.uint8, torch.float32
    _i8 = torch.int8  # (last: what the calls look at)


def _on(stream, dev: int) -> int:
    return _stream_of(dev) if stream is None else getattr(stream, "cuda_stream", stream)


def _refuse_codes(t, name: str, rows, k, dev: int):
    if not isinstance(t, _Tensor) or t.dtype is not _i8 or t.get_device() != dev:
        _refuse(t, name, _i8, None, False, dev)
    raise ValueError(f"{name} must be [{'rows' if rows is None else rows}, {'k' if k is None else f'>= {k}'}] int8 with "
                     f"unit column stride, got {tuple(t.shape)} of strides {t.stride()}")


def _codes(t, name: str, rows: int | None, k: int | None, dev: int):
    """t as int8 [rows, k or more] with unit column stride on device dev; its address, rows, columns and row stride."""
    if not isinstance(t, _Tensor) or t.dtype is not _i8 or t.get_device() != dev or t.dim() != 2:
        _refuse_codes(t, name, rows, k, dev)
    m, n = t.shape
    ld, one = t.stride()
    if one != 1 or m < 1 or (rows is not None and m != rows) or n < (k or 1):
        _refuse_codes(t, name, rows, k, dev)
    return t.data_ptr(), m, n, ld if m > 1 else (n + 15) // 16 * 16


def _quantize(x, act: int, norm_w, eps: float, add, out, scales, stream):
    if _i8 is None:
        _names()
    if not isinstance(x, _Tensor) or x.dim() != 2:
        raise ValueError("rows must be a float32 GPU tensor [M, K]")
    rows, k = x.shape
    if act == ACT_SILU_MUL:
        if k % 2:
            raise ValueError(f"gate_up has {k} columns: gate, then up")
        k //= 2
    dev = x.get_device()
    if dev < 0 or dev != _current_device():
        _device_of(x, "x")
    ldx, one = x.stride()
    if x.dtype is not _f32 or one != 1 or rows < 1 or k < 1 or ldx > 0x7fffffff:
        _rows(x, "x", k, None, dev)
        raise ValueError(f"x of strides {x.stride()}: unit column stride, rows up to 2^31 values apart")
    if rows == 1:
        ldx = x.shape[1]
    wp = 0 if norm_w is None else _whole(norm_w, "norm_w", _f32, (k,), dev)
    if add is None:
        ap, n = 0, 0
    else:
        if isinstance(add, _Tensor) and add.dim() == 2:
            n, shape = 1, (rows, k)
        else:
            n = add.shape[0] if isinstance(add, _Tensor) and add.dim() == 3 else 1
            shape = (n, rows, k)
        ap = _whole(add, "add", _f32, shape, dev)
    if out is None:
        out = made_for(stream, x.new_empty, (rows, k), dtype=_i8)
    if scales is None:
        scales = made_for(stream, x.new_empty, rows)
    try:
        (m, kq), (ldq, q1) = out.shape, out.stride()
        fine = (out.dtype is _i8 and m == rows and kq >= k and q1 == 1 and out.get_device() == dev and scales.dtype is _f32
                and scales.shape == (rows,) and scales.get_device() == dev and scales.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        fine = False
    if not fine:  # (which of them is not, by name)
        _, _, kq, ldq = _codes(out, "out", rows, k, dev)
        _whole(scales, "scales", _f32, (rows,), dev)
    if rows == 1:  # (a single row's stride has no meaning)
        ldq = (kq + 15) // 16 * 16
    rc = _c_quantize(_INPUT(x.data_ptr(), ldx, act, wp, eps, ap, n, rows * k), rows, k, out.data_ptr(), ldq, scales.data_ptr(),
                     _stream_of(dev) if stream is None else _on(stream, dev))
    if rc:
        _lib.check(rc)
    return out, scales


def quantize_i8(x, out=None, scales=None, stream=None):
    """Rows x [M, K] float32 (unit column stride, K a multiple of 16) as int8
    codes [M, K] and float32 scales [M]: scales[m] = max |x[m]| / 127, codes
    the nearest, ties to even. A row of zeros has scale 0, one with a value
    that is not finite scale NaN, both codes 0."""
    return _quantize(x, ACT_PLAIN, None, 0.0, None, out, scales, stream)


def rmsnorm_i8(x, norm_w=None, eps: float = 1e-6, add=None, out=None, scales=None, stream=None):
    """RMSNorm(x) * norm_w of rows x [M, K] as codes and scales. add, [M, K] or
    [n, M, K]: the slices are added to x first, in place."""
    return _quantize(x, ACT_RMSNORM, norm_w, eps, add, out, scales, stream)


def silu_mul_i8(gate_up, out=None, scales=None, stream=None):
    """silu(gate) * up of rows [gate | up] (gate_up [M, 2 K]) as codes [M, K] and scales."""
    return _quantize(gate_up, ACT_SILU_MUL, None, 0.0, None, out, scales, stream)


def quantize_weights_i8(qtype: int, w_dev, n: int, k: int, stream=None):
    """A GGUF matrix [n, k] on the device as int8 codes [n, k] and a scale a
    channel, once at load time: its rows dequantized, 64 Mi values at a time,
    then quantize_i8. The codes' rows begin at multiples of 128 bytes, which
    gemm_i8 reads fastest (512 x 4096 x 2880: 14.5 us, with rows of 2880 bytes 16.0)."""
    import torch
    if _i8 is None:
        _names()
    if qtype not in BLOCK_ELEMS or k % BLOCK_ELEMS[qtype]:
        raise ValueError(f"qtype {qtype}, k={k}: not rows of whole blocks")
    row = k // BLOCK_ELEMS[qtype] * BLOCK_BYTES[qtype]
    if n < 1:
        raise ValueError(f"n={n} channels")
    check_tensor(w_dev, "w_dev", torch.uint8, min_numel=n * row)
    _device_of(w_dev, "w_dev")
    codes = made_for(stream, torch.empty, (n, (k + 127) // 128 * 128), dtype=torch.int8, device=w_dev.device)[:, :k]
    scales = made_for(stream, torch.empty, n, dtype=torch.float32, device=w_dev.device)
    step = max(1, (64 << 20) // k)
    flat = w_dev.view(-1)
    for i in range(0, n, step):
        rows = min(step, n - i)
        x = dequant(qtype, flat[i * row:(i + rows) * row], rows * k, stream=stream).view(rows, k)
        quantize_i8(x, out=codes[i:i + rows], scales=scales[i:i + rows], stream=stream)
    return codes, scales


@_lib.kept_by_size
def _ws_bytes(m: int, n: int, k: int, flags: int) -> int:
    nb = C.c_size_t()
    _lib.check(_lib.load().ihip_gemm_i8_ws_bytes(m, n, k, flags, C.byref(nb)))
    return int(nb.value)


def gemm_i8_ws_bytes(m: int, n: int, k: int, accum: bool = False) -> int:
    """Workspace bytes of gemm_i8 (0: none)."""
    return _ws_bytes(m, n, k, GEMM_ACCUM if accum else 0)


def gemm_i8(q, scales, w, w_scales, accum: bool = False, out=None, ws=None, stream=None):
    """out [M, N] float32 = scales[m] * w_scales[n] * sum_k q[m, k] w[n, k], or
    with accum that added to out (which is then given). q int8 [M, K or more
    columns], w int8 [N, K] (unit column stride, rows a multiple of 16 values
    apart, K a multiple of 16), scales float32 [M] and [N]. Any M and N."""
    if _i8 is None:
        _names()
    try:
        (n, k), (m, kq), (ldw, w1), (ldq, q1) = w.shape, q.shape, w.stride(), q.stride()
        dev = q.get_device()
        fine = (dev >= 0 and dev == _current_device() and q.dtype is _i8 and w.dtype is _i8 and w1 == 1 and q1 == 1
                and kq >= k > 0 and w.get_device() == dev and m > 0 and n > 0 and scales.dtype is _f32 and scales.shape == (m,)
                and scales.get_device() == dev and scales.is_contiguous() and w_scales.dtype is _f32 and w_scales.shape == (n,)
                and w_scales.get_device() == dev and w_scales.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        fine = False
    if not fine:  # (which of them is not, by name)
        dev = _device_of(q, "q")
        _, n, k, ldw = _codes(w, "w", None, None, dev)
        _, m, _, ldq = _codes(q, "q", None, k, dev)
        _whole(scales, "scales", _f32, (m,), dev)
        _whole(w_scales, "w_scales", _f32, (n,), dev)
    if m == 1:  # (a single row's stride has no meaning)
        ldq = (k + 15) // 16 * 16
    if n == 1:
        ldw = (k + 15) // 16 * 16
    if out is None:
        if accum:
            raise ValueError("accum adds to out: pass it")
        out = made_for(stream, scales.new_empty, (m, n))
    yp, _, ldy = _rows(out, "out", n, m, dev)
    flags = GEMM_ACCUM if accum else 0
    if ws is None:
        need = _ws_bytes(m, n, k, flags)
        ws = made_for(stream, scales.new_empty, need, dtype=_u8, returned=False) if need else None
    tp, tn = (None, 0) if ws is None else _workspace(ws, dev)
    rc = _c_gemm(q.data_ptr(), ldq, scales.data_ptr(), w.data_ptr(), ldw, w_scales.data_ptr(), yp, ldy, m, n, k, flags, tp, tn,
                 _stream_of(dev) if stream is None else _on(stream, dev))
    if rc:
        _lib.check(rc)
    return out
