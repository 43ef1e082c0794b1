"""attn_prefix against the definition in 64 bits, entry by entry within the bound of fp32 arithmetic
(_mixref.attention_bound), and within the matmuls' fp32-accurate criterion (rel-L2 1e-5)."""
import numpy as np
import pytest

import _mixref as R
from _util import rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ih():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import inferno_hip
    assert inferno_hip.quant_kernels_available(), inferno_hip._lib.last_error()
    return inferno_hip


class Case:
    def __init__(self, s, m, hq, hkv, d, p, lens, dtype="float16", tree=None, seed=0, q_size=1.5, spare=3, head_major=False):
        import torch
        self.s, self.m, self.hq, self.hkv, self.d, self.p = s, m, hq, hkv, d, p
        dt = getattr(torch, dtype)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        r = lambda *a: torch.randn(a, generator=g, device="cuda")  # noqa: E731
        self.lens = np.asarray(lens, dtype=np.int32)
        cap = int(max(0, self.lens.max())) + m + spare
        self.q = q_size * r(s * m, hq * d)
        shape = (s, hkv, cap, d) if head_major else (s, cap, hkv, d)
        self.k, self.v = (r(*shape).to(dt) for _ in "kv")
        if head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.pk, self.pv = (r(1, max(p, 1), hkv, d).to(dt) for _ in "kv")
        for i in range(s):  # what lies behind a sequence's entries is nothing a row may see
            if self.lens[i] >= 0:
                self.k[i, self.lens[i] + m:] = float("nan")
                self.v[i, self.lens[i] + m:] = float("nan")
        self.mask = tree
        self.scale = d ** -0.5

    def tensors(self):
        import torch
        ln = torch.from_numpy(self.lens).cuda()
        mk = None if self.mask is None else torch.tensor([[b - (1 << 64) if b >> 63 else b for b in r] for r in self.mask],
                                                        dtype=torch.int64, device="cuda")
        return ln, mk

    def run(self, ih, **kw):
        ln, mk = self.tensors()
        return ih.attn_prefix(self.q, self.hq, ih.KVCache(self.k, self.v), ln,
                              prefix=ih.KVCache(self.pk, self.pv) if self.p else None, tree_mask=mk, **kw)

    def want(self):
        n = lambda t: t.float().cpu().numpy()  # noqa: E731
        return R.attention(n(self.q).reshape(self.s, self.m, self.hq, self.d), n(self.k), n(self.v),
                           n(self.pk)[0][: self.p], n(self.pv)[0][: self.p], self.lens.tolist(), self.scale, self.mask)

    def check(self, got):
        out, size, reach, seen = self.want()
        g = got.double().cpu().numpy().reshape(out.shape)
        live = self.lens >= 0
        err, tol = np.abs(g - out)[live], R.attention_bound(self.d, size, reach, seen)[live]
        assert np.isfinite(g[live]).all() and (err <= tol).all(), (float((err - tol).max()), float(err.max()))
        assert (g[(seen == 0).repeat(self.d, 3) & live[:, None, None, None]] == 0).all()
        if np.any(out[live]):
            assert rel_l2(g[live], out[live]) <= 1e-5


def trees(s, m, seed):
    rng = np.random.default_rng(seed)
    out = []
    for _ in range(s):
        bits = [1]
        for i in range(1, m):
            bits.append(bits[int(rng.integers(0, i))] | 1 << i)
        out.append(bits)
    return out


SHAPES = [  # s, m, hq, hkv, d, p, lens
    (1, 1, 4, 1, 128, 0, [0]),            # a first token: itself alone
    (1, 1, 32, 8, 128, 777, [150]),
    (1, 1, 1, 1, 64, 1, [0]),
    (3, 5, 8, 2, 128, 130, [0, 31, 64]),
    (2, 5, 10, 2, 64, 257, [33, 7]),
    (4, 1, 6, 2, 256, 63, [1, 2, 300, 5]),
    (9, 5, 16, 4, 64, 515, [3, 40, 0, 12, 99, 64, 1, 33, 32]),
    (2, 64, 4, 2, 128, 100, [17, 70]),
    (1, 64, 8, 2, 256, 129, [5]),
    (7, 3, 21, 7, 128, 0, [5, 0, 1, 255, 256, 257, 30]),
    (1, 150, 4, 4, 128, 0, [20]),         # a block of a prompt: causal, more than 64 tokens
    (1, 3, 8, 1, 128, 3000, [0]),
    (33, 2, 8, 2, 128, 300, list(range(33))),
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_causal(ih, shape, dtype):
    c = Case(*shape, dtype=dtype, seed=len(shape[6]))
    c.check(c.run(ih))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("s,m,hq,hkv,d,p,lens", [(1, 64, 16, 4, 256, 300, [77]), (3, 17, 8, 2, 128, 90, [0, 5, 40]),
                                                 (1, 7, 4, 4, 64, 0, [0]), (2, 33, 12, 4, 128, 0, [31, 100])])
def test_tree(ih, s, m, hq, hkv, d, p, lens, dtype):
    c = Case(s, m, hq, hkv, d, p, lens, dtype=dtype, tree=trees(s, m, s + m), seed=3)
    c.check(c.run(ih))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_rows_that_see_nothing(ih, dtype):
    """No prefix, no cached entries, masks without a bit (and bits past M, which name no entry)."""
    m = 5
    mask = [[0, 0b11, 0, 1 << 63 | 0b100, 1 << 40], [0] * m]
    c = Case(2, m, 4, 2, 128, 0, [0, 0], dtype=dtype, tree=mask, seed=9)
    got = c.run(ih)
    c.check(got)
    assert bool((got.view(2, m, 4, 128)[1] == 0).all()) and bool((got.view(2, m, 4, 128)[0, 0] == 0).all())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_unseen_entries_have_no_effect(ih, dtype):
    """NaN and infinite keys and values at a new entry that only some rows see: the others as without it."""
    import torch
    m = 6
    mask = [[0b1, 0b11, 0b101, 0b1001, 0b10011, 0b100101]]
    c = Case(1, m, 4, 2, 128, 40, [13], dtype=dtype, tree=mask, seed=4)
    clean = c.run(ih)
    for bad in (float("nan"), float("inf"), -float("inf")):
        k, v = c.k.clone(), c.v.clone()
        c.v[0, 13 + 1, :, ::3] = bad
        c.k[0, 13 + 2] = bad
        got = c.run(ih).view(m, 4, 128)
        for r in (0, 3):  # see neither
            assert torch.equal(got[r], clean.view(m, 4, 128)[r])
        for r in (1, 4):  # see the value: non-finite where it is, the rest as before
            assert not bool(torch.isfinite(got[r][:, ::3]).any())
            assert torch.equal(got[r][:, 1::3], clean.view(m, 4, 128)[r][:, 1::3])
        c.k, c.v = k, v


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_idle_and_full_sequences(ih, dtype):
    import torch
    c = Case(4, 3, 8, 2, 64, 50, [9, -1, 12, 4], dtype=dtype, seed=6, spare=0)
    full = Case(4, 3, 8, 2, 64, 50, [9, -1, 12, 4], dtype=dtype, seed=6, spare=0)
    out = torch.full((12, 8 * 64), 3.0, device="cuda")
    c.run(ih, out=out)
    c.check(out)
    assert bool((out.view(4, 3, -1)[1] == 3.0).all())
    full.lens = np.array([9, -1, 13, 4], dtype=np.int32)  # 13 + 3 entries of 15
    out2 = torch.full((12, 8 * 64), 3.0, device="cuda")
    full.run(ih, out=out2)
    assert bool(torch.isnan(out2.view(4, 3, -1)[2]).all())
    for i in (0, 1, 3):
        assert torch.equal(out2.view(4, 3, -1)[i], out.view(4, 3, -1)[i])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("q_size", [1e-6, 0.0, 30.0, 3000.0])
def test_score_sizes(ih, q_size, dtype):
    """Flat, zero and one-hot softmaxes; scores far past exp's range."""
    c = Case(2, 5, 8, 2, 128, 200, [40, 3], dtype=dtype, seed=8, q_size=q_size)
    c.check(c.run(ih))


def test_value_sizes(ih):
    """fp16 values of either end of the range, one head's tiny and another's large."""
    c = Case(2, 4, 8, 4, 128, 300, [20, 90], seed=12)
    for t in (c.v, c.pv):
        t[..., 0, :] *= 2.0 ** -13
        t[..., 1, :] *= 2.0 ** 12
    c.check(c.run(ih))


@pytest.mark.parametrize("head_major", [False, True])
def test_strides(ih, head_major):
    """Rows of q and out apart, caches of either order, a prefix that is a slice of another cache."""
    import torch
    c = Case(3, 5, 8, 2, 128, 90, [10, 0, 70], seed=2, head_major=head_major)
    plain = c.run(ih)
    wide = torch.randn(15, 8 * 128 + 64, device="cuda")
    wide[:, : 8 * 128] = c.q
    big_k, big_v = torch.randn(2, 200, 3, 128, device="cuda").half(), torch.randn(2, 200, 3, 128, device="cuda").half()
    big_k[1, 50:140, :2], big_v[1, 50:140, :2] = c.pk[0], c.pv[0]
    out = torch.full((15, 8 * 128 + 8), 5.0, device="cuda")
    ln, _ = c.tensors()
    ih.attn_prefix(wide, 8, ih.KVCache(c.k, c.v), ln, prefix=ih.KVCache(big_k[1:, 50:140, :2], big_v[1:, 50:140, :2]), out=out)
    assert torch.equal(out[:, : 8 * 128], plain) and bool((out[:, 8 * 128:] == 5.0).all())


def test_far_entries(ih):
    """Entries more than 2^31 values behind the cache's start."""
    import torch
    c = Case(2, 2, 4, 2, 64, 0, [9, 30], seed=21)
    gap = (1 << 31) + 8192
    flat = [torch.empty(gap + c.k[0].numel(), dtype=torch.float16, device="cuda") for _ in "kv"]
    far = [f.as_strided(tuple(c.k.shape), (gap, *c.k.stride()[1:])) for f in flat]
    far[0].copy_(c.k), far[1].copy_(c.v)
    ln, _ = c.tensors()
    assert torch.equal(ih.attn_prefix(c.q, 4, ih.KVCache(*far), ln), c.run(ih))


def test_repeats_streams_and_graph(ih):
    """The same bits each time: on another stream, from a workspace of other contents, and replayed from a graph while the
    lengths advance, with eager calls of other inputs between."""
    import torch
    c = Case(5, 5, 16, 4, 128, 400, [3, 60, 0, 200, 31], seed=31, spare=20)
    other = Case(5, 5, 16, 4, 128, 333, [9, 9, 9, 9, 9], seed=32, spare=40)
    c.k.nan_to_num_(0.5), c.v.nan_to_num_(0.5)
    ref = c.run(ih)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = c.run(ih)
    st.synchronize()
    assert torch.equal(again, ref)
    cache, prefix = ih.KVCache(c.k, c.v), ih.KVCache(c.pk, c.pv)
    ws = torch.full((ih.attn_prefix_ws_bytes(16, 5, cache, prefix),), 255, dtype=torch.uint8, device="cuda")
    ln, _ = c.tensors()
    step = torch.full((5,), 2, dtype=torch.int32, device="cuda")
    out = torch.empty_like(ref)
    first = ln.clone()
    with torch.cuda.stream(st):
        ih.attn_prefix(c.q, 16, cache, ln, prefix=prefix, out=out, ws=ws)
    st.synchronize()
    assert torch.equal(out, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        ih.attn_prefix(c.q, 16, cache, ln, prefix=prefix, out=out, ws=ws)
        ih.advance_len_(ln, step)
    for i in range(4):
        out.fill_(float("nan"))
        graph.replay()
        other.run(ih)
        torch.cuda.synchronize()
        want = ih.attn_prefix(c.q, 16, cache, first + 3 * i, prefix=prefix)
        assert torch.equal(out, want), i


BIG = [  # s, m, hq, hkv, d, p, lens: what takes each pair of block shapes (the prefix's, the sequences' own)
    (5, 55, 8, 2, 64, 300, [0, 3, 20, 70, 1]),           # 1100 rows share, 220 a sequence
    (5, 55, 8, 2, 128, 300, [0, 3, 20, 70, 1]),
    (1, 300, 8, 2, 64, 100, [40]),                       # 1200 rows of one
    (1, 300, 8, 2, 128, 100, [40]),
    (1, 300, 8, 2, 64, 28000, [0]),                      # and a long prefix
    (64, 4, 32, 8, 64, 8300, [i % 5 for i in range(64)]),
    (1, 1100, 32, 8, 64, 0, [900]),
    (9, 4, 16, 4, 256, 7500, [7] * 9),
    (1, 100, 16, 4, 256, 50, [2600]),
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", BIG)
def test_large(ih, shape, dtype):
    """(The definition in 64 bits on the GPU, a sequence and key head at a time: these are too many for the other.)"""
    import torch
    c = Case(*shape, dtype=dtype, seed=41)
    got = c.run(ih).double().view(c.s, c.m, c.hkv, -1, c.d)
    q = c.q.double().view(got.shape)
    diff = norm = 0.0
    for i in range(c.s):
        n = int(c.lens[i])
        last = c.p + n + torch.arange(c.m, device="cuda")[:, None, None]
        hides = torch.arange(c.p + n + c.m, device="cuda") > last  # [m, 1, keys]
        for g in range(c.hkv):
            k, v = (torch.cat([x[0, :c.p, g], y[i, :n + c.m, g]]).double() for x, y in ((c.pk, c.k), (c.pv, c.v)))
            z = (q[i, :, g] @ k.T * c.scale).masked_fill(hides, float("-inf"))
            w = torch.softmax(z, -1)
            out, size = w @ v, w @ v.abs()
            reach = (q[i, :, g].abs() @ k.abs().T * c.scale).masked_fill(hides, 0.0).amax(-1, keepdim=True)
            err = (got[i, :, g] - out).abs()
            bound = R.attention_bound(c.d, size, reach, (last + 1).double())
            assert bool((err <= bound).all()), (i, g, float((err - bound).max()))
            diff, norm = diff + float(err.square().sum()), norm + float(out.square().sum())
    assert diff <= 1e-10 * norm, (diff, norm)  # rel-L2 1e-5


@pytest.mark.parametrize("d,dtype", [(64, "float16"), (128, "float16"), (128, "bfloat16"), (256, "bfloat16")])
def test_tree_of_many_heads(ih, d, dtype):
    """So many query heads over a key head that a sequence's own entries are met in tall blocks."""
    c = Case(2, 64, 34, 2, d, 70, [30, 2050 if d == 256 else 5], dtype=dtype, tree=trees(2, 64, 3), seed=43)
    c.check(c.run(ih))


@pytest.mark.parametrize("d,dtype", [(64, "float16"), (64, "bfloat16"), (128, "bfloat16"), (256, "float16")])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_large_unseen_values(ih, d, dtype, value):
    """Tall blocks: an entry whose k and v are not finite reaches the rows that see it alone."""
    import torch
    m, n = 300, 1100 if d == 256 else 40
    c = Case(1, m, 8, 2, d, 100, [n], dtype=dtype, seed=47)
    good = c.run(ih)
    c.k[0, n + 200:n + m], c.v[0, n + 200:n + m] = value, value
    got = c.run(ih)
    assert torch.equal(got[:200], good[:200]) and not bool(torch.isfinite(got[200:]).any())
