"""Workspaces of the token mixers: their sizes where tokens go in chunks, and calls that stay inside them."""
import ctypes as C

import pytest

import _mixref as R
from inferno_hip import _lib as L
from test_gpu_attn_prefix import Case, trees
from test_gpu_delta import check, ih, make  # noqa: F401  (ih: the fixture)

BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 63) & ~63


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("s,t,n_k,n_v", [(1, 65, 1, 1), (3, 333, 2, 6), (7, 64, 3, 3), (2, 63, 1, 5)])
def test_chunked_workspace(s, t, n_k, n_v, dk):
    """A chunk of 64 tokens keeps two fp16 limbs of q, k and (a value head) W, six 16 x 32 blocks of P T in two limbs, six
    factors a token and 16 more; a call with less is refused before any launch."""
    lib, nb = L.load(), C.c_size_t()
    assert lib.ihip_delta_ws_bytes(s, t, n_k, n_v, dk, 48, 0, C.byref(nb)) == 0
    rows = 2 * 64 * dk * 2
    assert nb.value == s * ((t + 63) // 64) * (n_k * 2 * rows + n_v * (rows + 6 * 2 * 16 * 32 * 2 + (6 * 64 + 16) * 4))
    a = L.Delta(q=P, k=P, v=P, g=P, beta=P, ldq=n_k * dk, ldk=n_k * dk, ldv=n_v * 48, ldg=n_v, ldb=n_v, o=P, ldo=n_v * 48,
                state_in=None, state_out=P, snap_out=None, len=None, n_seq=s, T=t, n_k=n_k, n_v=n_v, dk=dk, dv=48, scale=0.1, flags=0)
    assert lib.ihip_gated_delta_rule(C.byref(a), P, nb.value - 1, None) == -12 and b"workspace" in lib.ihip_last_error()


class Fenced:
    """A workspace of n bytes between two fences of a pattern."""
    EDGE = 1 << 20

    def __init__(self, n):
        import torch
        self.all = torch.full((n + 2 * self.EDGE,), 0xA5, dtype=torch.uint8, device="cuda")
        self.ws = self.all[self.EDGE:self.EDGE + n]
        self.after = self.EDGE + n

    def check(self):
        assert bool((self.all[:self.EDGE] == 0xA5).all()) and bool((self.all[self.after:] == 0xA5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 14, 1, 1, 64, 4), (3, 333, 2, 6, 64, 36), (2, 65, 1, 3, 128, 20), (5, 130, 3, 3, 128, 16),
                                   (1, 1000, 2, 2, 64, 512), (2, 5, 1, 2, 64, 32)])
def test_delta_stays_inside(ih, shape):  # noqa: F811
    import torch
    s, t, hk, hv, dk, dv = shape
    q, k, v, g, b, st = make(*shape, seed=3)
    f = Fenced(ih.gated_delta_rule_ws_bytes(*shape))
    o, _, last = R.delta(q, k, v, g, b, st)
    new = torch.empty_like(st)
    check(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, ws=f.ws), o, "o")
    check(new, last, "state")
    f.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("s,m,hq,hkv,d,p,lens,tree", [
    (1, 1, 1, 1, 64, 0, [0], False), (1, 1, 4, 1, 128, 40000, [5], False), (3, 7, 10, 2, 64, 333, [31, 0, 64], False),
    (1, 1, 2, 1, 256, 0, [9000], False), (1, 37, 8, 2, 256, 100, [5], True), (5, 3, 6, 2, 128, 130, [3, -1, 9, 0, 2], False)])
def test_attention_stays_inside(ih, s, m, hq, hkv, d, p, lens, tree, dtype):  # noqa: F811
    import torch
    c = Case(s, m, hq, hkv, d, p, lens, dtype=dtype, tree=trees(s, m, 3) if tree else None, seed=7)
    f = Fenced(ih.attn_prefix_ws_bytes(hq, m, ih.KVCache(c.k, c.v), ih.KVCache(c.pk, c.pv) if p else None))
    out = torch.full((s * m, hq * d), 3.0, device="cuda")
    c.check(c.run(ih, ws=f.ws, out=out))
    f.check()
