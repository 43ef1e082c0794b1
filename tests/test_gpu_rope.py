"""Rotary positions and the KV-cache append against the definition in 64 bits.

Tolerance of a rotated value: the angle's fraction of a turn is rounded once to
fp32 (at most pi 2^-24 radians), sine and cosine are within two units (2 2^-24
each of a value up to 1), mscale, the two products and the sum round once each:
at most (pi + 2 + 1 + 3) 2^-24 < 10 2^-24 of |a| + |b|. A cache value is off by
half a step of its type more (and half the type's smallest subnormal)."""
import numpy as np
import pytest

import _mixref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ih():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import inferno_hip
    assert inferno_hip.quant_kernels_available(), inferno_hip._lib.last_error()
    return inferno_hip


def close(got, want, size, half_step=0.0, least=0.0):
    err = np.abs(got.double().cpu().numpy() - want)
    tol = 10 * U * size + half_step * np.abs(want) * (1 + 2 ** -10) + least
    assert (err <= tol).all(), float((err - tol).max())


STEP = {"float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 2.0 ** -134)}  # (finfo(t).eps / 2, half a subnormal)
SCALINGS = [("none", {}, 1.0), ("linear", {"factor": 8.0}, 1.0),
            ("by_parts", {"factor": 4.0, "orig_len": 8192.0, "beta_fast": 32.0, "beta_slow": 1.0}, 1.138)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (256, 64), (80, 20), (96, 24), (6, 4), (2, 2), (512, 256)])
@pytest.mark.parametrize("scaling", range(3))
def test_rope(ih, d, rot, interleaved, scaling):
    """Both layouts, part of the head, rows apart, every scaling, positions up to 2^31 - 1."""
    import torch
    name, kw, mscale = SCALINGS[scaling]
    heads, n = 3, 37
    rng = np.random.default_rng(d * 7 + rot + scaling)
    wide = torch.from_numpy(rng.standard_normal((n, heads * d + 12)).astype(np.float32)).cuda()
    x = wide[:, : heads * d]
    pos = np.concatenate([[0, 1, 2, 2 ** 31 - 1, 1000003], rng.integers(0, 200000, n - 5)]).astype(np.int32)
    rp = ih.RopeParams(d, rot, interleaved=interleaved, base=500000.0, scaling=name, attn_scale=mscale, **kw)
    y = ih.rope(x, torch.from_numpy(pos).cuda(), heads, rp)
    th = R.theta(rot, 500000.0, name, **kw)
    m32 = float(np.float32(mscale))
    xn = x.cpu().double().numpy().reshape(n, heads, d)
    close(y.view(n, heads, d), R.rotate(xn, pos, th, interleaved, m32), R.pair_size(xn, rot, interleaved, m32))
    keep = wide[:, heads * d:].clone()
    z = ih.rope(x, torch.from_numpy(pos).cuda(), heads, rp, out=x)  # in place, what lies beside the rows untouched
    assert torch.equal(z, y) and torch.equal(wide[:, heads * d:], keep)


def test_rope_frequency_factors_and_alignment(ih):
    """freq_factors divide the frequencies; rows that are no multiple of 16 bytes, and a view 4 bytes off."""
    import torch
    d, rot, heads, n = 64, 32, 2, 9
    rng = np.random.default_rng(5)
    ff = (1 + 7 * rng.random(rot // 2)).astype(np.float32)
    rp = ih.RopeParams(d, rot, base=10000.0, freq_factors=torch.from_numpy(ff).cuda())
    pos = rng.integers(0, 100000, n).astype(np.int32)
    buf = torch.from_numpy(rng.standard_normal(n * 131 + 1).astype(np.float32)).cuda()
    x = buf[1:].view(n, 131)[:, : heads * d]
    y = ih.rope(x, torch.from_numpy(pos).cuda(), heads, rp)
    xn = x.cpu().double().numpy().reshape(n, heads, d)
    close(y.view(n, heads, d), R.rotate(xn, pos, R.theta(rot, 10000.0, freq_factors=ff), False), R.pair_size(xn, rot, False))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("s,m,hq,hkv,d,rot", [(1, 1, 32, 8, 128, 128), (5, 3, 4, 2, 64, 16), (3, 17, 3, 1, 256, 64),
                                               (2, 700, 2, 2, 40, 40), (4, 1, 6, 2, 24, 12)])
def test_append(ih, dtype, head_major, s, m, hq, hkv, d, rot):
    """q, and the cache entries len .. len + m; the others as they were. One sequence idle, one without room."""
    import torch
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(s * 100 + m)
    cap = m + 50
    shape = (s, hkv, cap, d) if head_major else (s, cap, hkv, d)
    k0, v0 = (torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda().to(dt) for _ in "kv")
    k, v = k0.clone(), v0.clone()
    view = (lambda t: t.transpose(1, 2)) if head_major else (lambda t: t)
    lens = rng.integers(0, 50, s).astype(np.int32)
    if s > 2:
        lens[1], lens[2] = -1, 51
    qkv = torch.from_numpy(rng.standard_normal((s * m, (hq + 2 * hkv) * d + 4)).astype(np.float32)).cuda()
    rp = ih.RopeParams(d, rot, base=10000.0)
    out = torch.full((s * m, hq * d), 7.0, device="cuda")
    ln = torch.from_numpy(lens).cuda()
    ih.rope_append(qkv, hq, ih.KVCache(view(k), view(v)), ln, rp, pos0=11, out=out)
    x = qkv[:, : (hq + 2 * hkv) * d].cpu().double().numpy().reshape(s, m, hq + 2 * hkv, d)
    o = out.view(s, m, hq, d)
    th = R.theta(rot, 10000.0)
    half, least = STEP[dtype]
    for i in range(s):
        n = int(lens[i])
        mine = [view(t)[i].clone() for t in (k, v)]
        before = [view(t)[i] for t in (k0, v0)]
        if n < 0 or n + m > cap:
            assert torch.equal(mine[0], before[0]) and torch.equal(mine[1], before[1])
            assert bool((o[i] == 7.0).all()) if n < 0 else bool(torch.isnan(o[i]).all())
            continue
        turned = R.rotate(x[i], 11 + n + np.arange(m), th, False)
        size = R.pair_size(x[i], rot, False)
        close(o[i], turned[:, :hq], size[:, :hq])
        close(mine[0][n:n + m], turned[:, hq:hq + hkv], size[:, hq:hq + hkv], half, least)
        assert torch.equal(mine[1][n:n + m], torch.from_numpy(x[i][:, hq + hkv:]).to(torch.float32).to(dt).cuda())
        for t, b in zip(mine, before):
            assert torch.equal(t[:n], b[:n]) and torch.equal(t[n + m:], b[n + m:])
    # explicit positions, q in place: the same values
    posn = (11 + lens[:, None].astype(np.int64) + np.arange(m)).astype(np.int32).reshape(-1)
    k2, v2 = k0.clone(), v0.clone()
    ih.rope_append(qkv, hq, ih.KVCache(view(k2), view(v2)), ln, rp, positions=torch.from_numpy(posn).cuda(), out=qkv)
    for i in range(s):
        if lens[i] >= 0 and lens[i] + m <= cap:
            assert torch.equal(qkv[i * m:(i + 1) * m, : hq * d], out[i * m:(i + 1) * m])
    assert torch.equal(k2, k) and torch.equal(v2, v)


def test_append_far_sequences(ih):
    """Sequences whose entries lie more than 2^31 values apart."""
    import torch
    s, cap, hkv, d = 2, 8, 2, 64
    gap = (1 << 31) + 4096
    flat = [torch.empty(gap + cap * hkv * d, dtype=torch.float16, device="cuda") for _ in "kv"]
    k, v = (f.as_strided((s, cap, hkv, d), (gap, hkv * d, d, 1)) for f in flat)
    k.zero_(), v.zero_()
    qkv = torch.randn(s, (2 + 2 * hkv) * d, device="cuda")
    lens = torch.tensor([3, 5], dtype=torch.int32, device="cuda")
    q = ih.rope_append(qkv, 2, ih.KVCache(k, v), lens, ih.RopeParams(d))
    k2, v2 = torch.zeros(s, cap, hkv, d, dtype=torch.float16, device="cuda"), torch.zeros(s, cap, hkv, d, dtype=torch.float16, device="cuda")
    q2 = ih.rope_append(qkv, 2, ih.KVCache(k2, v2), lens, ih.RopeParams(d))
    assert torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(v, v2) and bool((k2[1, 5] != 0).any())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(256, 64), (128, 128)])
def test_many_rows_are_as_few(ih, d, rot, interleaved):
    """More rows than the caches hold (their loads and stores pass them by): the same bits as a few at a time."""
    import torch
    n, hq, hkv = 2300, 16, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(n, (hq + 2 * hkv) * d + 8, generator=g, device="cuda")[:, :(hq + 2 * hkv) * d]
    rp = ih.RopeParams(d, rot, interleaved=interleaved, base=1e6)
    def caches():
        return [torch.full((1, n + 3, hkv, d), 7.0, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    k, v = caches()
    q = ih.rope_append(x, hq, ih.KVCache(k, v), torch.tensor([2], dtype=torch.int32, device="cuda"), rp, pos0=11)
    k1, v1 = caches()
    c1 = ih.KVCache(k1, v1)
    for at in range(0, n, 500):
        m = min(500, n - at)
        part = ih.rope_append(x[at:at + m], hq, c1, torch.tensor([2 + at], dtype=torch.int32, device="cuda"), rp, pos0=11)
        assert torch.equal(part, q[at:at + m]), at
    assert torch.equal(k, k1) and torch.equal(v, v1)
    pos = 13 + torch.arange(n, dtype=torch.int32, device="cuda")
    assert torch.equal(ih.rope(x, pos, hq + 2 * hkv, rp)[:, :hq * d], q)
