"""The 8-bit projections where their kernels and their values end."""
import numpy as np
import pytest

import _i8ref as R
from _i8plans import PLANS, TILE128X2
from test_gpu_int8 import cu, ih, operands, rng, rows, same  # noqa: F401  (ih: the fixture)

pytestmark = pytest.mark.gpu


def bits(t):
    import torch
    return t.contiguous().view(torch.int32)


def rounded(q, s, w, ws):
    """The product's steps one by one in fp32, which round as the kernels do: the whole sum, then the two scales."""
    with np.errstate(under="ignore", over="ignore"):
        return (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32) * s[:, None] * ws


@pytest.mark.parametrize("m,n,k", [(1, 37, 272), (5, 300, 272), (16, 302, 8208), (33, 301, 144), (300, 257, 144), (300, 2001, 8208)])
def test_signs_of_zero(ih, m, n, k):  # noqa: F811
    """Products that are zero or underflow keep their sign in every kernel and column, as the three steps have it."""
    r = rng(30, m, n)
    q, s, w, ws = operands(r, m, n, k)
    s[::2] *= -1  # sums of zero become -0, in a row of zeros for every channel
    q[0] = 0
    ws[1::5] *= -1
    s[min(1, m - 1)] = 0.0  # (a scale of zero with codes that are not)
    s[min(2, m - 1)] = np.float32(-1e-44)  # (most of its products underflow)
    w[::7] = 0
    want = rounded(q, s, w, ws)
    assert (np.signbit(want) & (want == 0)).any()
    got = ih.gemm_i8(*map(cu, (q, s, w, ws))).cpu().numpy()
    bad = np.argwhere(got.view(np.int32) != want.view(np.int32))
    assert not len(bad), (len(bad), bad[:4].tolist())


@pytest.mark.parametrize("k", [16160, 16384, 16400, 65536])
def test_scales_past_fp32(ih, k):  # noqa: F811
    """A norm's scale can pass fp32 where neither the row's largest value nor its sum of squares is out of the ordinary: one value
    that is not zero, eps 0 and a large weight. Such a row has scale NaN and codes 0, its neighbours what they have."""
    x = np.zeros((6, k), np.float32)
    x[0, 5], x[1, k - 9], x[4, 5] = 1e-13, -1e-10, 2e-15
    x[3, 77], x[5, 77] = 1e-13, -1e-3
    x[2] = rows(rng(31, k), 1, k)[0]
    w = np.ones(k, np.float32)
    w[[5, k - 9]] = np.finfo(np.float32).max  # (sqrt(K) / 127 of it: past fp32 from K = 16130 on)
    w[77] = 1e30
    want = R.rmsnorm(x, w, 0.0)
    past = np.isin(np.arange(6), (0, 1, 4))
    assert np.isnan(want[1][past]).all() and np.isfinite(want[1][~past]).all()
    same(ih.rmsnorm_i8(cu(x), cu(w), 0.0), want, R.norm_tol(k))


@pytest.mark.parametrize("m,k", [(3, 512), (300, 1040), (2, 16400)])
def test_gates_below_the_normal_numbers(ih, m, k):  # noqa: F811
    """Gates whose half is a subnormal number, with ups so large that their product is an ordinary one."""
    r = rng(32, m, k)
    for gate, up in ((1e-42, 1e25), (1e-40, 1e37), (3e-38, 1e20), (1e-44, 5e37), (1e-39, 1e9)):
        g, u = (r.uniform(-1, 1, (m, k)) * gate).astype(np.float32), (r.standard_normal((m, k)) * up).astype(np.float32)
        g[0, 3:], u[m - 1, 0] = 0, 0
        gu = np.concatenate([g, u], 1)
        same(ih.silu_mul_i8(cu(gu)), R.quantize(R.silu_mul(gu)), 2 * R.HALF)


@pytest.mark.parametrize("far", [-89.0, -1e3, -9e5, -2e6, -1e12, -1e30, -3e38])
@pytest.mark.parametrize("m,k", [(3, 512), (300, 1040), (2, 16400)])
def test_gates_far_below_zero(ih, m, k, far):  # noqa: F811
    """A finite gate far below zero has a product of nothing, beside products of any size."""
    r = rng(33, m, k)
    for up in (1.0, 1e-3, 1e-16, 1e4, 1e12):
        gu = (2 * r.standard_normal((m, 2 * k))).astype(np.float32)
        gu[:, k:] *= up
        gu[:, 1:k:9] = far
        gu[m - 1, k + 1::9] *= 1e3
        same(ih.silu_mul_i8(cu(gu)), R.quantize(R.silu_mul(gu)), 2 * R.HALF)


@pytest.mark.parametrize("m,n,k,accum,kernel,parts", PLANS)
def test_every_kernel_and_number_of_parts(ih, m, n, k, accum, kernel, parts):  # noqa: F811
    """Products that end inside the tiles of each kernel, over K of several times its places in LDS, into rows that begin at any
    value: the bits of the sum's rounding, the two scales' and the addition's. What lies beside the results stays."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(35 + m + k)
    codes = lambda *s: torch.randint(-128, 128, s, dtype=torch.int8, device="cuda", generator=g)  # noqa: E731
    scale = lambda c: torch.rand(c, device="cuda", generator=g) + 0.01  # noqa: E731
    # (rows beside K: operands lie in wider ones, whose other values count for nothing)
    q, w, s, ws = codes(m, k + 48)[:, 16:16 + k], codes(n, k + 16)[:, :k], scale(m), scale(n)
    sums = torch.empty((m, n), device="cuda")
    wt = w.double().T.contiguous()
    for i in range(0, m, 512):
        sums[i:i + 512] = (q[i:i + 512].double() @ wt).float()  # (whole numbers below 2^53: exact)
    y = 1e4 * torch.randn((m + 2, n + 5), device="cuda", generator=g)
    want = y.clone()
    steps = sums * s[:, None] * ws
    want[1:m + 1, 1:n + 1] = steps + y[1:m + 1, 1:n + 1] if accum else steps
    space = torch.full((ih.gemm_i8_ws_bytes(m, n, k, accum) + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    ih.gemm_i8(q, s, w, ws, accum=accum, out=y[1:m + 1, 1:n + 1], ws=space[:-256])
    assert (space.numel() > 256) == (parts > 1) and bool((space[-256:] == 0x5a).all())
    bad = (bits(y) != bits(want)).nonzero()
    assert not len(bad), (len(bad), bad[0].tolist(), bad[-1].tolist())


def test_rows_alone_and_from_the_large_tiles(ih):  # noqa: F811
    """A row's and a channel's results in tiles of 128 and 256 are the bits of calls on them alone."""
    import torch
    for m, n, k, accum, kernel, parts in PLANS:
        if kernel < TILE128X2 or accum:
            continue
        q, s, w, ws = (cu(v) for v in operands(rng(36, m, k), m, n, k))
        y = ih.gemm_i8(q, s, w, ws)
        for i, j in ((1, n), (5, 700), (64, 1030), (300, 333), (m, 1)):
            got = ih.gemm_i8(q[m - i:], s[m - i:], w[n - j:], ws[n - j:])
            assert torch.equal(bits(got), bits(y[m - i:, n - j:])), (m, n, k, i, j)


@pytest.mark.parametrize("m,k,weight", [(4200, 4112, True), (4200, 4112, False), (1027, 16384, True), (8200, 2064, True)])
def test_norm_past_the_caches(ih, m, k, weight):  # noqa: F811
    """The residual's addition and the norm of so many rows that they are read and written past the caches: every row's sums,
    codes and scales. Among them rows whose values lie next to a tie, and rows whose largest products are equal in fp32 and not
    in truth, made of halves that only the sum puts together."""
    import torch
    assert m * k >= 16 << 20
    r = rng(34, m, k)
    w = (1 + 0.3 * r.standard_normal(k)).astype(np.float32)
    w[np.abs(w) < 0.05] = 1
    if not weight:
        w[:] = 1
    x = rows(r, m, k)
    add = r.standard_normal((m, k), dtype=np.float32)
    planted = np.arange(3, m, m // 60)
    for i in planted:
        if i % 2:
            top = np.float32(r.uniform(0.5, 200.0))
            y = ((r.integers(-127, 127, k) + 0.5) * np.float64(top) / 127.0 / w).astype(np.float32)
            y += (r.integers(-2, 3, k) * np.spacing(np.abs(y))).astype(np.float32)
            y[7] = top / w[7]
        else:
            y = (np.float32(3.0) / w).astype(np.float32) * (r.integers(0, 2, k) * 2 - 1).astype(np.float32)
        x[i] = add[i] = y / 2
    xd, wd = cu(x), cu(w)
    want_x = torch.from_numpy(x + add).cuda()
    q, s = ih.rmsnorm_i8(xd, wd if weight else None, 1e-5, add=cu(add))
    assert torch.equal(bits(xd), bits(want_x))
    for i in range(0, m, 512):
        t = want_x[i:i + 512].double()
        factor = 1.0 / torch.sqrt((t * t).mean(-1) + 1e-5)
        t = t * wd.double()
        top = t.abs().amax(-1)
        code = torch.round(t * 127.0 / top[:, None])
        bad = (code != q[i:i + 512]).nonzero()
        assert not len(bad), (len(bad), bad[0].tolist(), (bad[0] + torch.tensor([i, 0], device="cuda")).tolist())
        scale = top / 127.0 * factor
        assert bool(((s[i:i + 512].double() - scale).abs() <= R.norm_tol(k) * scale).all()), i
