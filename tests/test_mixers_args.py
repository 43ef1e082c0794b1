"""The token mixers' argument checks and descriptors, without a GPU (calls that fail before any launch, and
ihip_rope_init, which is host arithmetic)."""
import ctypes as C
import math

import pytest

import _mixref as R
from inferno_hip import _lib as L


@pytest.fixture(scope="module")
def lib():
    return L.load()


BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 63) & ~63


def rope_of(lib, d=128, rot=128, inter=0, base=10000.0, scaling=0, factor=1.0, orig=0.0, fast=32.0, slow=1.0, ms=1.0, ff=None):
    r = L.Rope()
    return lib.ihip_rope_init(C.byref(r), d, rot, inter, base, scaling, factor, orig, fast, slow, ms, ff), r


def kv(type=1, n_seq=2, n_kv=2, d=128, cap=16, k=P, v=P, strides=None):
    st = strides or (cap * n_kv * d, n_kv * d, d)
    return L.Kv(type, n_seq, n_kv, d, cap, k, v, *st)


@pytest.mark.parametrize("scaling,kw", [(0, {}), (1, {"factor": 8.0}),
                                        (2, {"factor": 4.0, "orig": 8192.0, "fast": 32.0, "slow": 1.0})])
def test_rope_table(lib, scaling, kw):
    """Turns per position of each pair, to a few units of fp64."""
    rc, r = rope_of(lib, 256, 64, base=1000000.0, scaling=scaling, **kw)
    assert rc == 0
    names = {"factor": "factor", "orig": "orig_len", "fast": "beta_fast", "slow": "beta_slow"}
    th = R.theta(64, 1000000.0, ("none", "linear", "by_parts")[scaling], **{names[k]: v for k, v in kw.items()})
    for i in range(32):
        assert abs(r.turns[i] * 2 * math.pi - th[i]) <= 8 * 2.0 ** -53 * th[i]
    assert list(r.turns[32:]) == [0.0] * 96


def test_rope_refusals(lib):
    assert lib.ihip_rope_init(None, 128, 128, 0, 1e4, 0, 1.0, 0.0, 32.0, 1.0, 1.0, None) == -14
    for kw in ({"rot": 127}, {"rot": 0}, {"rot": 130}, {"d": 512, "rot": 258}, {"base": 0.0}, {"base": float("inf")},
               {"scaling": 3}, {"scaling": 1, "factor": 0.0}, {"scaling": 1, "factor": float("nan")},
               {"scaling": 2, "factor": 4.0}, {"scaling": 2, "factor": 4.0, "orig": 100.0, "fast": 1.0, "slow": 1.0},
               {"scaling": 2, "factor": 4.0, "orig": 100.0, "ff": P}, {"ms": float("nan")}):
        assert rope_of(lib, **kw)[0] == -22, kw
    _, r = rope_of(lib)
    ref = C.byref(r)
    assert lib.ihip_rope_apply(ref, None, 128, P, 128, 1, P, 1, None) == -14
    assert lib.ihip_rope_apply(None, P, 128, P, 128, 1, P, 1, None) == -14
    assert lib.ihip_rope_apply(ref, P, 127, P, 128, 1, P, 1, None) == -22
    assert lib.ihip_rope_apply(ref, P, 128, P, 100, 1, P, 1, None) == -22
    assert lib.ihip_rope_apply(ref, P, 128, P, 128, 0, P, 1, None) == -22
    assert lib.ihip_rope_apply(ref, P, 128, P, 128, 1, P, 0, None) == -22
    assert lib.ihip_rope_apply(ref, P, 256, P, 128, 1, P, 1, None) == -22  # in place, other row stride


def test_append_refusals(lib):
    _, r = rope_of(lib)
    ref = C.byref(r)
    call = lambda c, ld=1024, ldq=512, n_q=4, M=1, x=P, q=P + 64, n=P: lib.ihip_rope_append(  # noqa: E731
        ref, x, ld, q, ldq, n_q, None if c is None else C.byref(c), n, None, 0, M, None)
    assert call(None) == -14 and call(kv(), x=None) == -14 and call(kv(), n=None) == -14 and call(kv(k=None)) == -14
    assert call(kv(), ld=1023) == -22 and call(kv(), ldq=511) == -22 and call(kv(), M=0) == -22 and call(kv(), n_q=0) == -22
    assert call(kv(), q=P) == -22  # in place, other row stride
    assert call(kv(d=64)) == -22 and b"head_dim" in lib.ihip_last_error()
    assert call(kv(), M=1 << 23) == -22  # more tokens than a launch holds
    for bad in (kv(type=0), kv(n_seq=0), kv(n_kv=0), kv(cap=0), kv(k=P + 8), kv(strides=(4096, 256, 132)),
                kv(strides=(4095 * 8, 128, 128)), kv(strides=(2048, 256, 128)), kv(strides=(-4096, 256, 128)),
                kv(strides=(1 << 62, 1 << 61, 1 << 60), cap=1 << 30)):
        assert call(bad) == -22, list(bad.strides if hasattr(bad, "strides") else [bad.seq_stride, bad.tok_stride])


def test_attn_refusals(lib):
    nb = C.c_size_t()
    ws = lambda c, n_q=4, M=1, pre=None: lib.ihip_attn_prefix_ws_bytes(  # noqa: E731
        n_q, M, C.byref(c), None if pre is None else C.byref(pre), C.byref(nb))
    one = kv(n_seq=1, cap=100)
    assert ws(kv()) == 0 and nb.value > 0 and ws(kv(), pre=one) == 0
    assert lib.ihip_attn_prefix_ws_bytes(4, 1, C.byref(kv()), None, None) == -14
    assert ws(kv(), M=1 << 20) == -22 and b"query rows" in lib.ihip_last_error()  # more than a launch holds
    assert ws(kv(d=96)) == -22 and ws(kv(), n_q=3) == -22 and ws(kv(), n_q=0) == -22 and ws(kv(), M=0) == -22
    for bad in (kv(n_seq=2), kv(n_seq=1, type=30), kv(n_seq=1, n_kv=1), kv(n_seq=1, d=64)):
        assert ws(kv(), pre=bad) == -22
    c = kv()
    ws(c)
    call = lambda q=P, ldq=512, out=P, ldo=512, n_q=4, M=1, n=P, mask=None, scale=0.1, w=P, wb=1 << 40: (  # noqa: E731
        lib.ihip_attn_prefix(q, ldq, out, ldo, n_q, M, C.byref(c), n, None, mask, scale, w, wb, None))
    assert call(q=None) == -14 and call(n=None) == -14 and call(w=None) == -14
    assert call(ldq=508) == -22 and call(ldo=514) == -22 and call(q=P + 4) == -22 and call(out=P + 8) == -22
    assert call(M=65, mask=P) == -22 and call(scale=float("nan")) == -22 and call(w=P + 8) == -22
    assert call(wb=nb.value - 1) == -12


def test_delta_refusals(lib):
    nb = C.c_size_t()
    for bad in ((0, 1, 1, 1, 64, 64), (1, 0, 1, 1, 64, 64), (1, 1, 2, 3, 64, 64), (1, 1, 0, 1, 64, 64), (1, 1, 1, 1, 96, 64),
                (1, 1, 1, 1, 64, 30), (1, 1, 1, 1, 64, 516), (65536, 1, 1, 1, 64, 64), (60000, 1, 1, 128, 64, 64)):
        assert lib.ihip_delta_ws_bytes(*bad, 0, C.byref(nb)) == -22, bad
    assert lib.ihip_delta_ws_bytes(1, 1, 1, 1, 64, 64, 0, None) == -14
    assert lib.ihip_delta_ws_bytes(2, 9, 1, 2, 64, 64, 0, C.byref(nb)) == 0 and nb.value > 0

    def call(wb=1 << 40, **kw):
        a = dict(q=P, k=P, v=P, g=P, beta=P, ldq=64, ldk=64, ldv=128, ldg=2, ldb=2, o=P, ldo=128, state_in=P, state_out=P,
                 snap_out=None, len=None, n_seq=2, T=9, n_k=1, n_v=2, dk=64, dv=64, scale=0.1, flags=0)
        a.update(kw)
        return lib.ihip_gated_delta_rule(C.byref(L.Delta(**a)), P, wb, None)

    assert lib.ihip_gated_delta_rule(None, P, 1 << 40, None) == -14
    for kw in ({"q": None}, {"o": None}, {"beta": None}):
        assert call(**kw) == -14, kw
    for kw in ({"ldq": 60}, {"ldk": 66}, {"ldv": 124}, {"ldo": 130}, {"ldg": 1}, {"ldb": 0}, {"q": P + 4}, {"state_out": P + 8},
               {"snap_out": P + 4}, {"snap_out": P, "T": 65}, {"flags": 2}, {"scale": float("inf")}, {"dk": 80}, {"n_seq": 0}):
        assert call(**kw) == -22, kw
    assert call(wb=nb.value - 1) == -12


def test_wrappers_refuse_host_tensors():
    """The Python entry points check what the C ABI cannot see."""
    import torch

    import inferno_hip as ih
    t = torch.zeros(4, 512)
    with pytest.raises(ValueError):
        ih.KVCache(torch.zeros(1, 4, 2, 64, dtype=torch.float16), torch.zeros(1, 4, 2, 64, dtype=torch.float16))
    with pytest.raises(ValueError):
        ih.RopeParams(128, scaling="other")
    with pytest.raises(ih.HipError):
        ih.RopeParams(128, 129)
    with pytest.raises(ValueError):
        ih.rope(t, torch.zeros(4, dtype=torch.int32), 4, ih.RopeParams(128))
    with pytest.raises(ValueError):
        ih.gated_delta_rule(*(torch.zeros(1, 2, 1, 64),) * 3, torch.zeros(1, 2, 1), torch.zeros(1, 2, 1), None)
