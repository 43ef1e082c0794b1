"""What stands between the projections of a decoder layer: rotary positions
and the KV-cache append (the reference's partial RoPE and cache write,
src/ModelCPU.jl:125-258), attention of a batch's new tokens over a shared
prefix and their own cached entries (:730-856), and the gated delta rule of
the recurrent layers (:476-700).

They take the fp32 rows the matmuls of quantized_kernels leave and give fp32
rows to the next matmul; lengths and states are read and written on the
device, so that a step of them can be captured in a HIP graph between
speculative.advance_len_ and speculative.commit_state_.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .quantized_kernels import _ptr, _stream, check_tensor

F16, BF16 = 1, 30
ROPE_PLAIN, ROPE_LINEAR, ROPE_BY_PARTS = 0, 1, 2
DELTA_L2NORM = 1
_SCALINGS = {"none": ROPE_PLAIN, "linear": ROPE_LINEAR, "by_parts": ROPE_BY_PARTS}


def _here(*tensors):
    """The tensors are on the current device, whose stream the call takes."""
    import torch
    at = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"a tensor is on {t.device}, the current device is cuda:{at}")


def _rows(t, name: str, width: int, rows: int | None = None):
    """t as fp32 [rows, >= width] with unit column stride; its row stride."""
    import torch
    check_tensor(t, name, torch.float32, contiguous=False)
    if t.dim() != 2 or t.shape[1] < width or (rows is not None and t.shape[0] != rows) or t.shape[0] < 1 \
            or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be [{'rows' if rows is None else rows}, >= {width}] float32 with unit column "
                         f"stride, got {tuple(t.shape)}")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


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
        self._ref = C.byref(self._c)


def rope(x, positions, n_heads: int, params: RopeParams, out=None, stream=None):
    """x [tokens, n_heads * head_dim] float32 (unit column stride) with each
    head rotated to its row's position (int32 [tokens]); out may be x."""
    import torch
    width = n_heads * params.head_dim
    ldx = _rows(x, "x", width)
    if x.shape[1] != width:
        x = x[:, :width]
    check_tensor(positions, "positions", torch.int32, (x.shape[0],))
    if out is None:
        out = torch.empty((x.shape[0], width), dtype=torch.float32, device=x.device)
    ldo = _rows(out, "out", width, x.shape[0])
    _here(x, positions, out, params.freq_factors)
    _lib.check(_lib.load().ihip_rope_apply(params._ref, _ptr(x), ldx, _ptr(out), ldo, n_heads, _ptr(positions),
                                           x.shape[0], _stream(stream)))
    return out


def rope_append(qkv, n_q: int, cache: KVCache, lengths, params: RopeParams, positions=None, pos0: int = 0, out=None,
                stream=None):
    """The new tokens' rows qkv [sequences * M, >= (n_q + 2 n_kv) * head_dim]
    (q heads, k heads, v heads): q rotated into out [sequences * M, n_q *
    head_dim] (returned; may be qkv itself), k rotated and v as it is into the
    cache's entries lengths[s] + m. positions int32 [sequences * M], or pos0 +
    lengths[s] + m. lengths int32 [sequences]: below 0 an idle sequence (left
    as it was); where M entries do not fit, NaN rows and the cache as it was."""
    import torch
    d = params.head_dim
    ld = _rows(qkv, "qkv", (n_q + 2 * cache.n_kv) * d)
    rows = qkv.shape[0]
    if rows % cache.n_seq:
        raise ValueError(f"{rows} rows for {cache.n_seq} sequences")
    check_tensor(lengths, "lengths", torch.int32, (cache.n_seq,))
    if positions is not None:
        check_tensor(positions, "positions", torch.int32, (rows,))
    if out is None:
        out = torch.empty((rows, n_q * d), dtype=torch.float32, device=qkv.device)
    ldq = _rows(out, "out", n_q * d, rows)
    _here(qkv, cache.k, lengths, positions, out, params.freq_factors)
    _lib.check(_lib.load().ihip_rope_append(params._ref, _ptr(qkv), ld, _ptr(out), ldq, n_q, cache._ref, _ptr(lengths),
                                            None if positions is None else _ptr(positions), pos0, rows // cache.n_seq,
                                            _stream(stream)))
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
    import torch
    d = cache.head_dim
    ldq = _rows(q, "q", n_q * d)
    rows = q.shape[0]
    if rows % cache.n_seq:
        raise ValueError(f"{rows} rows for {cache.n_seq} sequences")
    m = rows // cache.n_seq
    check_tensor(lengths, "lengths", torch.int32, (cache.n_seq,))
    if tree_mask is not None:
        check_tensor(tree_mask, "tree_mask", torch.int64, (cache.n_seq, m))
    if out is None:
        out = torch.empty((rows, n_q * d), dtype=torch.float32, device=q.device)
    ldo = _rows(out, "out", n_q * d, rows)
    if ws is None:
        ws = torch.empty(attn_prefix_ws_bytes(n_q, m, cache, prefix), dtype=torch.uint8, device=q.device)
    check_tensor(ws, "ws", torch.uint8)
    _here(q, cache.k, None if prefix is None else prefix.k, lengths, tree_mask, out, ws)
    _lib.check(_lib.load().ihip_attn_prefix(_ptr(q), ldq, _ptr(out), ldo, n_q, m, cache._ref, _ptr(lengths),
                                            None if prefix is None else prefix._ref,
                                            None if tree_mask is None else _ptr(tree_mask),
                                            d ** -0.5 if scale is None else scale, _ptr(ws), ws.numel(),
                                            _stream(stream)))
    return out


@_lib.kept_by_size
def _delta_ws_bytes(n_seq: int, t: int, n_k: int, n_v: int, dk: int, dv: int, snapshots: int) -> int:
    nb = C.c_size_t()
    _lib.check(_lib.load().ihip_delta_ws_bytes(n_seq, t, n_k, n_v, dk, dv, snapshots, C.byref(nb)))
    return int(nb.value)


def gated_delta_rule_ws_bytes(n_seq: int, t: int, n_k: int, n_v: int, dk: int, dv: int, snapshots: bool = False) -> int:
    """Workspace bytes of gated_delta_rule for t tokens a sequence."""
    return _delta_ws_bytes(n_seq, t, n_k, n_v, dk, dv, int(bool(snapshots)))


def _heads(t, name: str, shape):
    """t as fp32 [sequences, tokens, heads, values], each token's heads side by side, the tokens' rows evenly spaced
    over all sequences; the row stride."""
    import torch
    check_tensor(t, name, torch.float32, shape, contiguous=False)
    s, n, h, d = t.shape
    st = t.stride()
    ld = st[1] if n > 1 else st[0] if s > 1 else h * d
    if (d > 1 and st[3] != 1) or (h > 1 and st[2] != d) or (s > 1 and n > 1 and st[0] != n * ld) or ld < h * d:
        raise ValueError(f"{name} {tuple(t.shape)} of strides {st}: the heads of a token must be contiguous and the "
                         "rows of all tokens evenly spaced")
    return ld


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
    [sequences]: tokens of each, rows past them left as they were. Returns
    out [sequences, T, n_v, dv]."""
    import torch
    check_tensor(k, "k", torch.float32, (None, None, None, None), contiguous=False)
    check_tensor(v, "v", torch.float32, (None, None, None, None), contiguous=False)
    s, t, n_k, dk = k.shape
    n_v, dv = v.shape[2], v.shape[3]
    if 0 in k.shape or 0 in v.shape:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)}: nothing to do")
    ldq, ldk = _heads(q, "q", (s, t, n_k, dk)), _heads(k, "k", (s, t, n_k, dk))
    ldv = _heads(v, "v", (s, t, n_v, dv))
    for x, name in ((g, "g"), (beta, "beta")):
        check_tensor(x, name, torch.float32, (s, t, n_v), contiguous=False)
    ldg, ldb = (_heads(x.unsqueeze(3), name, (s, t, n_v, 1)) for x, name in ((g, "g"), (beta, "beta")))
    if out is None:
        out = torch.empty((s, t, n_v, dv), dtype=torch.float32, device=v.device)
    ldo = _heads(out, "out", (s, t, n_v, dv))
    for x, name in ((state, "state"), (new_state, "new_state")):
        if x is not None:
            check_tensor(x, name, torch.float32, (s, n_v, dk, dv))
    if snapshots is not None:
        check_tensor(snapshots, "snapshots", torch.float32, (s, t, n_v, dk, dv))
    if lengths is not None:
        check_tensor(lengths, "lengths", torch.int32, (s,))
    if ws is None:
        ws = torch.empty(gated_delta_rule_ws_bytes(s, t, n_k, n_v, dk, dv, snapshots is not None), dtype=torch.uint8,
                         device=v.device)
    check_tensor(ws, "ws", torch.uint8)
    _here(q, k, v, g, beta, state, new_state, snapshots, lengths, out, ws)
    p = lambda x: None if x is None else _ptr(x)  # noqa: E731
    a = _lib.Delta(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), ldq, ldk, ldv, ldg, ldb, _ptr(out), ldo, p(state),
                   p(new_state), p(snapshots), p(lengths), s, t, n_k, n_v, dk, dv,
                   dk ** -0.5 if scale is None else scale, DELTA_L2NORM if l2norm else 0)
    _lib.check(_lib.load().ihip_gated_delta_rule(C.byref(a), _ptr(ws), ws.numel(), _stream(stream)))
    return out
