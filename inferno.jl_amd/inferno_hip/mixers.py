"""What stands between the projections of a decoder layer: rotary positions
and the KV-cache append (the reference's partial RoPE and cache write,
src/ModelCPU.jl:125-258), attention of a batch's new tokens over a shared
prefix and their own cached entries (:730-856), and the gated delta rule of
the recurrent layers (:476-700).

They take the fp32 rows the matmuls of quantized_kernels leave and give fp32
rows to the next matmul; lengths and states are read and written on the
device, so that a step of them can be captured in a HIP graph between
speculative.advance_len_ and speculative.commit_state_.

Kernels run on `stream` (default: torch's current one). What a call allocates
itself (out, ws) is made for that stream; its inputs have to be ready there,
and other streams wait for it before they read its outputs. A workspace that is
given serves one call at a time.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .quantized_kernels import _ptr, _raw_stream, check_tensor, made_for

F16, BF16 = 1, 30
ROPE_PLAIN, ROPE_LINEAR, ROPE_BY_PARTS = 0, 1, 2
DELTA_L2NORM = 1
_SCALINGS = {"none": ROPE_PLAIN, "linear": ROPE_LINEAR, "by_parts": ROPE_BY_PARTS}


# The per-call checks are kept to a few attribute reads a tensor (a call's host time is most of a one-token call's); what
# they refuse goes to _refuse for the message.
_f32 = _i32 = _i64 = _u8 = _current_device = _stream_of = _Tensor = None


def _torch():
    """torch's names, looked up once (the package itself does not import it)."""
    global _f32, _i32, _i64, _u8, _current_device, _stream_of, _Tensor
    import torch
    _current_device, _stream_of = torch.cuda.current_device, _raw_stream()
    _i32, _i64, _u8, _Tensor = torch.int32, torch.int64, torch.uint8, torch.Tensor
    _f32 = torch.float32  # (last: what the calls look at)


def _refuse(t, name: str, dtype, shape=None, contiguous: bool = True, dev: int | None = None):
    """The ValueError for a tensor that is not as it should be."""
    check_tensor(t, name, dtype, shape, contiguous)
    if dev is not None and t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{dev}")
    raise ValueError(f"{name}: strides {t.stride()} of {tuple(t.shape)}")


def _device_of(t, name: str) -> int:
    """The device of a GPU tensor, which is the current one."""
    dev = t.get_device() if isinstance(t, _Tensor) else -1
    if dev < 0:
        check_tensor(t, name)
    if dev != _current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{_current_device()}")
    return dev


def _on(stream, dev: int) -> int:
    """The stream's handle; without one that of torch's current stream."""
    return _stream_of(dev) if stream is None else getattr(stream, "cuda_stream", stream)


def _call(name: str):
    """A bound function of the library."""
    return getattr(_lib._lib or _lib.load(), name)


def _whole(t, name: str, dtype, shape, dev: int):
    """A contiguous tensor of exactly this type and shape on device dev; its address."""
    if not isinstance(t, _Tensor) or t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _refuse(t, name, dtype, shape, True, dev)
    return t.data_ptr()


def _workspace(ws, dev: int):
    if not isinstance(ws, _Tensor) or ws.dtype is not _u8 or ws.get_device() != dev or not ws.is_contiguous():
        _refuse(ws, "ws", _u8, None, True, dev)
    return ws.data_ptr(), ws.numel()


def _rows(t, name: str, width: int, rows: int | None, dev: int):
    """t as fp32 [rows, >= width] with unit column stride on device dev; its address, rows and row stride."""
    if not isinstance(t, _Tensor) or t.dtype is not _f32 or t.get_device() != dev:
        _refuse(t, name, _f32, None, False, dev)
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[1] < width or shape[0] < 1 or (rows is not None and shape[0] != rows) \
            or (stride[1] != 1 and shape[1] > 1):
        raise ValueError(f"{name} must be [{'rows' if rows is None else rows}, >= {width}] float32 with unit column "
                         f"stride, got {tuple(shape)} of strides {stride}")
    return t.data_ptr(), shape[0], stride[0] if shape[0] > 1 else max(stride[0], shape[1])


class RopeParams:
    """ihip_rope: rotary positions of heads of head_dim values, rot_dim of
    them rotated (default: all), in pairs (i, i + rot_dim / 2) or, interleaved,
    (2 i, 2 i + 1). scaling "none", "linear" (theta / factor) or "by_parts"
    (pairs that turn more than beta_fast times over orig_len keep their
    frequency, those below beta_slow are divided by factor, a ramp between);
    attn_scale multiplies the rotated values; freq_factors: a float32 GPU
    tensor [rot_dim / 2] that divides the frequencies."""

    def __init__(self, head_dim: int, rot_dim: int | None = None, interleaved: bool = False, base: float = 10000.0,
                 scaling: str = "none", factor: float = 1.0, orig_len: float = 0.0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attn_scale: float = 1.0, freq_factors=None):
        import torch
        if scaling not in _SCALINGS:
            raise ValueError(f"scaling {scaling!r}: one of {', '.join(_SCALINGS)}")
        rot_dim = head_dim if rot_dim is None else rot_dim
        if freq_factors is not None:
            check_tensor(freq_factors, "freq_factors", torch.float32, (rot_dim // 2,))
        self.head_dim, self.rot_dim, self.freq_factors = head_dim, rot_dim, freq_factors
        self._c = _lib.Rope()
        _lib.check(_lib.load().ihip_rope_init(C.byref(self._c), head_dim, rot_dim, int(interleaved), base,
                                              _SCALINGS[scaling], factor, orig_len, beta_fast, beta_slow, attn_scale,
                                              None if freq_factors is None else _ptr(freq_factors)))
        self._ref = C.byref(self._c)

    def _on(self, dev: int):
        if self.freq_factors is not None and self.freq_factors.get_device() != dev:
            raise ValueError(f"freq_factors are on {self.freq_factors.device}, the current device is cuda:{dev}")
        return self._ref


class KVCache:
    """ihip_kv over two float16 or bfloat16 GPU tensors k and v of shape
    [sequences, capacity, heads, head_dim] and equal strides (any order of the
    two middle axes in memory, each entry's values contiguous). The tensors
    are kept; their storage must stay where it is."""

    def __init__(self, k, v):
        import torch
        for t, name in ((k, "k"), (v, "v")):
            check_tensor(t, name, k.dtype if isinstance(k, torch.Tensor) else None, contiguous=False)
        if k.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a KV cache is float16 or bfloat16, got {k.dtype}")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.device != v.device or k.stride(3) != 1 \
                or k.numel() == 0:
            raise ValueError("k and v must be [sequences, capacity, heads, head_dim] of equal shapes and strides, "
                             "each entry's values contiguous")
        self.k, self.v = k, v
        self.n_seq, self.capacity, self.n_kv, self.head_dim = k.shape
        self._c = _lib.Kv(F16 if k.dtype == torch.float16 else BF16, self.n_seq, self.n_kv, self.head_dim,
                          self.capacity, _ptr(k), _ptr(v), k.stride(0), k.stride(1), k.stride(2))
        self._ref, self._dev = C.byref(self._c), k.get_device()

    def _on(self, dev: int):
        if self._dev != dev:
            raise ValueError(f"the cache is on cuda:{self._dev}, the current device is cuda:{dev}")
        return self._ref


def rope(x, positions, n_heads: int, params: RopeParams, out=None, stream=None):
    """x [tokens, n_heads * head_dim] float32 (unit column stride) with each
    head rotated to its row's position (int32 [tokens]); out may be x."""
    if _f32 is None:
        _torch()
    dev = _device_of(x, "x")
    width = n_heads * params.head_dim
    xp, rows, ldx = _rows(x, "x", width, None, dev)
    pp = _whole(positions, "positions", _i32, (rows,), dev)
    if out is None:
        out = made_for(stream, x.new_empty, (rows, width))
    yp, _, ldy = _rows(out, "out", width, rows, dev)
    _lib.check(_call("ihip_rope_apply")(params._on(dev), xp, ldx, yp, ldy, n_heads, pp, rows, _on(stream, dev)))
    return out


def rope_append(qkv, n_q: int, cache: KVCache, lengths, params: RopeParams, positions=None, pos0: int = 0, out=None,
                stream=None):
    """The new tokens' rows qkv [sequences * M, >= (n_q + 2 n_kv) * head_dim]
    (q heads, k heads, v heads): q rotated into out [sequences * M, n_q *
    head_dim] (returned; may be qkv itself), k rotated and v as it is into the
    cache's entries lengths[s] + m. positions int32 [sequences * M], or pos0 +
    lengths[s] + m. lengths int32 [sequences]: below 0 an idle sequence (left
    as it was); where M entries do not fit, NaN rows and the cache as it was."""
    if _f32 is None:
        _torch()
    dev = _device_of(qkv, "qkv")
    d, s = params.head_dim, cache.n_seq
    xp, rows, ld = _rows(qkv, "qkv", (n_q + 2 * cache.n_kv) * d, None, dev)
    if rows % s:
        raise ValueError(f"{rows} rows for {s} sequences")
    lp = _whole(lengths, "lengths", _i32, (s,), dev)
    pp = None if positions is None else _whole(positions, "positions", _i32, (rows,), dev)
    if out is None:
        out = made_for(stream, qkv.new_empty, (rows, n_q * d))
    yp, _, ldq = _rows(out, "out", n_q * d, rows, dev)
    _lib.check(_call("ihip_rope_append")(params._on(dev), xp, ld, yp, ldq, n_q, cache._on(dev), lp, pp, pos0, rows // s,
                                         _on(stream, dev)))
    return out


def attn_prefix_ws_bytes(n_q: int, m: int, cache: KVCache, prefix: KVCache | None = None) -> int:
    """Workspace bytes of attn_prefix for m new tokens a sequence."""
    nb = C.c_size_t()
    _lib.check(_lib.load().ihip_attn_prefix_ws_bytes(n_q, m, cache._ref, None if prefix is None else prefix._ref,
                                                     C.byref(nb)))
    return int(nb.value)


def attn_prefix(q, n_q: int, cache: KVCache, lengths, prefix: KVCache | None = None, scale: float | None = None,
                tree_mask=None, out=None, ws=None, stream=None):
    """Attention of q [sequences * M, >= n_q * head_dim] over prefix (one
    sequence that all share, whole), each sequence's entries [0, lengths[s])
    and its M new ones, already appended at lengths[s] ..: causal, or bit j of
    tree_mask (int64 [sequences, M], M <= 64) for new entry j. scale: default
    head_dim ** -0.5. A row that sees nothing is zero; lengths below 0 leave a
    sequence's rows as they were, and one past its capacity gets NaN rows."""
    if _f32 is None:
        _torch()
    dev = _device_of(q, "q")
    d, n = cache.head_dim, cache.n_seq
    qp, rows, ldq = _rows(q, "q", n_q * d, None, dev)
    if rows % n:
        raise ValueError(f"{rows} rows for {n} sequences")
    m = rows // n
    lp = _whole(lengths, "lengths", _i32, (n,), dev)
    mp = None if tree_mask is None else _whole(tree_mask, "tree_mask", _i64, (n, m), dev)
    if out is None:
        out = made_for(stream, q.new_empty, (rows, n_q * d))
    op, _, ldo = _rows(out, "out", n_q * d, rows, dev)
    if ws is None:
        ws = made_for(stream, q.new_empty, attn_prefix_ws_bytes(n_q, m, cache, prefix), dtype=_u8, returned=False)
    wp, wn = _workspace(ws, dev)
    _lib.check(_call("ihip_attn_prefix")(qp, ldq, op, ldo, n_q, m, cache._on(dev), lp,
                                         None if prefix is None else prefix._on(dev), mp,
                                         d ** -0.5 if scale is None else scale, wp, wn, _on(stream, dev)))
    return out


@_lib.kept_by_size
def _delta_ws_bytes(n_seq: int, t: int, n_k: int, n_v: int, dk: int, dv: int, snapshots: int) -> int:
    nb = C.c_size_t()
    _lib.check(_lib.load().ihip_delta_ws_bytes(n_seq, t, n_k, n_v, dk, dv, snapshots, C.byref(nb)))
    return int(nb.value)


def gated_delta_rule_ws_bytes(n_seq: int, t: int, n_k: int, n_v: int, dk: int, dv: int, snapshots: bool = False) -> int:
    """Workspace bytes of gated_delta_rule for t tokens a sequence."""
    return _delta_ws_bytes(n_seq, t, n_k, n_v, dk, dv, int(bool(snapshots)))


def _heads(t, name: str, s: int, n: int, h: int, d: int, dev: int):
    """t as fp32 [sequences, tokens, heads, values] (values 0: [sequences, tokens, heads]) on device dev, each token's heads
    side by side, the tokens' rows evenly spaced over all sequences; its address and the row stride."""
    shape = (s, n, h, d) if d else (s, n, h)
    if not isinstance(t, _Tensor) or t.dtype is not _f32 or t.shape != shape or t.get_device() != dev:
        _refuse(t, name, _f32, shape, False, dev)
    st = t.stride()
    w = h * d if d else h
    ld = st[1] if n > 1 else st[0] if s > 1 else w
    if (st[-1] != 1 and shape[-1] > 1) or (d and h > 1 and st[2] != d) or (s > 1 and n > 1 and st[0] != n * ld) or ld < w:
        raise ValueError(f"{name} {shape} of strides {st}: the heads of a token must be contiguous and the rows of all "
                         "tokens evenly spaced")
    return t.data_ptr(), ld


def gated_delta_rule(q, k, v, g, beta, state, new_state=None, snapshots=None, lengths=None, l2norm: bool = False,
                     scale: float | None = None, out=None, ws=None, stream=None):
    """The gated delta rule over T tokens of each sequence: q, k [sequences, T,
    n_k, dk], v [sequences, T, n_v, dv], g (log decay) and beta [sequences, T,
    n_v], all float32 (views of projection rows allowed: evenly spaced rows);
    state [sequences, n_v, dk, dv], or None for zeros. Per head: S = e^g S; S
    += k (beta (v - S^T k))^T; o = scale S^T q (scale: default dk ** -0.5),
    with unit q and k where l2norm is set. new_state receives the last state
    (may be `state`), snapshots [sequences, T, n_v, dk, dv] the state after
    every token (T <= 64; commit_state_ picks from them). lengths int32
    [sequences]: tokens of each, rows past them left as they were. Value head
    h reads key head h // (n_v // n_k). out overlaps none of the inputs.
    Returns out [sequences, T, n_v, dv]."""
    if _f32 is None:
        _torch()
    dev = _device_of(q, "q")
    for x, name in ((k, "k"), (v, "v")):
        if not isinstance(x, _Tensor) or x.dim() != 4 or x.numel() == 0:
            raise ValueError(f"{name} must be a float32 GPU tensor [sequences, tokens, heads, values] with something in it")
    s, t, n_k, dk = k.shape
    n_v, dv = v.shape[2], v.shape[3]
    a = _lib.Delta()
    a.q, a.ldq = _heads(q, "q", s, t, n_k, dk, dev)
    a.k, a.ldk = _heads(k, "k", s, t, n_k, dk, dev)
    a.v, a.ldv = _heads(v, "v", s, t, n_v, dv, dev)
    a.g, a.ldg = _heads(g, "g", s, t, n_v, 0, dev)
    a.beta, a.ldb = _heads(beta, "beta", s, t, n_v, 0, dev)
    if out is None:
        out = made_for(stream, v.new_empty, (s, t, n_v, dv))
    a.o, a.ldo = _heads(out, "out", s, t, n_v, dv, dev)
    if state is not None:
        a.state_in = _whole(state, "state", _f32, (s, n_v, dk, dv), dev)
    if new_state is not None:
        a.state_out = _whole(new_state, "new_state", _f32, (s, n_v, dk, dv), dev)
    if snapshots is not None:
        a.snap_out = _whole(snapshots, "snapshots", _f32, (s, t, n_v, dk, dv), dev)
    if lengths is not None:
        a.len = _whole(lengths, "lengths", _i32, (s,), dev)
    if ws is None:
        ws = made_for(stream, v.new_empty, gated_delta_rule_ws_bytes(s, t, n_k, n_v, dk, dv, snapshots is not None),
                      dtype=_u8, returned=False)
    wp, wn = _workspace(ws, dev)
    a.n_seq, a.T, a.n_k, a.n_v, a.dk, a.dv = s, t, n_k, n_v, dk, dv
    a.scale = dk ** -0.5 if scale is None else scale
    a.flags = DELTA_L2NORM if l2norm else 0
    _lib.check(_call("ihip_gated_delta_rule")(C.byref(a), wp, wn, _on(stream, dev)))
    return out
