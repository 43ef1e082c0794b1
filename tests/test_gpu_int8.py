"""The 8-bit projections on the GPU against their definitions in 64 bits: codes are equal, scales and products within the
roundings that they have."""
import numpy as np
import pytest

import _i8ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ih():
    import inferno_hip
    return inferno_hip


def cu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rng(*seed):
    return np.random.default_rng(seed)


def rows(r, m, k):
    """Rows with channels of several sizes, a few far larger."""
    size = np.exp(0.5 * r.standard_normal(k)).astype(np.float32)
    size[:: max(1, k // 3)] *= 12
    return (r.standard_normal((m, k)).astype(np.float32) * size).astype(np.float32)


def same(got, want, tol):
    """Codes equal, scales within tol (relative; where the scale is below fp32's normal numbers, half of its last step)."""
    (q, s), (rq, rs) = got, want
    q, s = q.cpu().numpy(), s.cpu().numpy().astype(np.float64)
    bad = np.argwhere(q != rq)
    assert bad.size == 0, f"{len(bad)} codes differ, the first at {bad[0]}: {q[tuple(bad[0])]} for {rq[tuple(bad[0])]}"
    assert np.array_equal(np.isnan(s), np.isnan(rs))
    off = np.abs(s - rs)[~np.isnan(rs)] - 2.0 ** -149
    assert (off <= tol * np.abs(rs[~np.isnan(rs)])).all(), float((off / np.abs(rs[~np.isnan(rs)])).max())


KS = [16, 48, 256, 1008, 4096, 4112, 6144, 12288, 16384, 16400, 40000, 65536]


@pytest.mark.parametrize("m", [1, 3, 257])
@pytest.mark.parametrize("k", KS)
def test_plain(ih, m, k):
    m = m if k < 20000 else min(m, 3)
    x = rows(rng(1, m, k), m, k)
    same(ih.quantize_i8(cu(x)), R.quantize(x), R.HALF)


@pytest.mark.parametrize("weight,add", [(True, 0), (False, 1), (True, 1), (True, 3), (False, 0)])
@pytest.mark.parametrize("m,k", [(1, 16), (2, 4096), (5, 2048), (300, 272), (300, 4096), (3, 12288), (2, 16400), (1, 65536)])
def test_rmsnorm(ih, m, k, weight, add):
    r = rng(2, m, k, add)
    x, w = rows(r, m, k), (1 + 0.2 * r.standard_normal(k)).astype(np.float32) if weight else None
    slices = r.standard_normal((add, m, k)).astype(np.float32)
    want = x.copy()
    if add:
        total = slices[0]
        for s in slices[1:]:
            total = total + s
        want = x + total
    xd = cu(x)
    got = ih.rmsnorm_i8(xd, None if w is None else cu(w), 1e-5, add=None if not add else cu(slices) if add > 1 else cu(slices[0]))
    assert np.array_equal(xd.cpu().numpy(), want)
    same(got, R.rmsnorm(want, w, 1e-5), R.norm_tol(k))


@pytest.mark.parametrize("m,k", [(1, 16), (5, 12288), (3, 4096), (259, 1040), (300, 6144), (2, 16400), (1, 65536)])
def test_silu_mul(ih, m, k):
    gu = 2.5 * rng(3, m, k).standard_normal((m, 2 * k)).astype(np.float32)
    same(ih.silu_mul_i8(cu(gu)), R.quantize(R.silu_mul(gu)), R.HALF)


def test_near_ties(ih):
    """Values within a few units of fp32 of a tie, on either side and on it, fall where the exact quotient does."""
    k = 4096
    r = rng(4)
    x = np.empty((64, k), np.float32)
    for i in range(64):
        top = np.float32(r.uniform(0.5, 200.0) if i else 127.0)
        half = (r.integers(-127, 127, k) + 0.5) * np.float64(top) / 127.0
        v = half.astype(np.float32)
        step = r.integers(-2, 3, k)
        x[i] = v + step * np.spacing(np.abs(v))
        x[i, 7] = top
    same(ih.quantize_i8(cu(x)), R.quantize(x), R.HALF)
    w = (1 + 0.3 * r.standard_normal(k)).astype(np.float32)
    w[np.abs(w) < 0.05] = 1
    y = (x / w).astype(np.float32)
    same(ih.rmsnorm_i8(cu(y), cu(w)), R.rmsnorm(y, w), R.norm_tol(k))
    assert (np.abs(np.abs(x[0] - np.rint(x[0]))) == 0.5).any()


def test_several_largest(ih):
    """Products that are equal in fp32 and not in truth: the largest of them sets the codes of the others."""
    k = 1024
    r = rng(5)
    w = (1 + r.random(k)).astype(np.float32)
    x = (np.float32(3.0) / w).astype(np.float32)
    x = np.stack([x, -x, x * (r.integers(0, 2, k) * 2 - 1).astype(np.float32)])
    same(ih.rmsnorm_i8(cu(x), cu(w)), R.rmsnorm(x, w), R.norm_tol(k))


@pytest.mark.parametrize("scale", [0.0, 1e-45, 1e-40, 1e-30, 1e-21, 1e-19, 1e-10, 1e18, 1e25, 1e31, 3e37])
def test_sizes_of_values(ih, scale):
    """Rows from the smallest to the largest numbers that fp32 holds."""
    r = rng(6)
    x = (r.uniform(-1, 1, (3, 512)) * scale).astype(np.float32)
    x[1, 5:] = 0
    same(ih.quantize_i8(cu(x)), R.quantize(x), R.HALF)
    w = (1 + 0.2 * r.standard_normal(512)).astype(np.float32)
    same(ih.rmsnorm_i8(cu(x), cu(w), 1e-6), R.rmsnorm(x, w), R.norm_tol(512))
    gu = np.concatenate([r.standard_normal((3, 512)).astype(np.float32) * 3, x], 1)
    same(ih.silu_mul_i8(cu(gu)), R.quantize(R.silu_mul(gu)), R.HALF)
    gu = np.concatenate([-85 - 30 * np.abs(r.standard_normal((3, 512))).astype(np.float32), x], 1)
    same(ih.silu_mul_i8(cu(gu)), R.quantize(R.silu_mul(gu)), 2 * R.HALF)


def test_zero_eps_and_weights(ih):
    """eps 0, weights of zero, rows of zeros."""
    r = rng(7)
    x = r.standard_normal((4, 256)).astype(np.float32)
    x[2] = 0
    w = np.zeros(256, np.float32)
    w[9] = -2
    x[3, 9] = 0
    same(ih.rmsnorm_i8(cu(x), cu(w), 0.0), R.rmsnorm(x, w, 0.0), R.norm_tol(256))
    same(ih.rmsnorm_i8(cu(x), None, 0.0), R.rmsnorm(x, None, 0.0), R.norm_tol(256))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("k", [512, 16400])
def test_not_finite(ih, bad, k):
    """A row with such a value: codes 0, scale NaN; the others as they are."""
    r = rng(8)
    x = r.standard_normal((4, k)).astype(np.float32)
    x[1, k - 3] = bad
    x[3, 0] = bad
    want = R.quantize(x[[0, 2]])
    for f, tol in ((ih.quantize_i8, R.HALF), (ih.rmsnorm_i8, R.norm_tol(k))):
        q, s = f(cu(x))
        assert not q[1].any() and not q[3].any() and s[[1, 3]].isnan().all()
        same((q[[0, 2]], s[[0, 2]]), want if f is ih.quantize_i8 else R.rmsnorm(x[[0, 2]]), tol)
    gu = r.standard_normal((4, 2 * k)).astype(np.float32)
    gu[1, 3], gu[2, 2 * k - 1] = bad, bad
    q, s = ih.silu_mul_i8(cu(gu))
    assert not q[1:3].any() and s[1:3].isnan().all()
    same((q[[0, 3]], s[[0, 3]]), R.quantize(R.silu_mul(gu[[0, 3]])), R.HALF)


def test_strides_and_what_lies_beside(ih):
    """Rows inside wider ones: inputs as views, codes into a wider buffer whose other columns stay."""
    import torch
    r = rng(9)
    wide = cu(r.standard_normal((6, 1200)).astype(np.float32))
    x = wide[:, 8:8 + 512]
    out = torch.full((6, 640), 77, dtype=torch.int8, device="cuda")
    scales = torch.empty(6, device="cuda")
    before = wide.clone()
    q, s = ih.quantize_i8(x, out=out[:, 64:576], scales=scales)
    assert q.data_ptr() == out.data_ptr() + 64 and s is scales
    same((q, s), R.quantize(x.cpu().numpy()), R.HALF)
    assert bool((out[:, :64] == 77).all()) and bool((out[:, 576:] == 77).all()) and torch.equal(wide, before)
    add = cu(r.standard_normal((6, 512)).astype(np.float32))
    ih.rmsnorm_i8(x, add=add, out=out[:, 64:576], scales=scales)
    before[:, 8:520] += add
    assert torch.equal(wide, before)
    same((out[:, 64:576], scales), R.rmsnorm(x.cpu().numpy()), R.norm_tol(512))


def test_slices_as_input(ih):
    """The partials of a deferred product, without x: their sum in slice order is the input."""
    import ctypes as C

    import torch
    from inferno_hip import _lib as L
    r = rng(10)
    sl = r.standard_normal((3, 5, 1040)).astype(np.float32)
    total = sl[0] + sl[1] + sl[2]
    d = cu(sl)
    for act, k, want, tol in ((0, 1024, R.quantize(total[:, :1024]), R.HALF), (1, 1024, R.rmsnorm(total[:, :1024]), R.norm_tol(1024)),
                              (2, 512, R.quantize(R.silu_mul(total[:, :1024])), R.HALF)):
        q, s = torch.empty((5, k), dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
        a = L.GemmInput(None, 1040, act, None, 1e-6, d.data_ptr(), 3, 5 * 1040)
        L.check(L.load().ihip_quantize_i8(C.byref(a), 5, k, q.data_ptr(), k, s.data_ptr(), torch.cuda.current_stream().cuda_stream))
        same((q, s), want, tol)


# ---------------------------------------------------------------- products

def operands(r, m, n, k):
    q = r.integers(-127, 128, (m, k)).astype(np.int8)
    w = r.integers(-127, 128, (n, k)).astype(np.int8)
    return q, (0.01 + r.random(m)).astype(np.float32), w, (0.001 + r.random(n)).astype(np.float32)


def near(got, want, extra=0.0):
    got = got.cpu().numpy().astype(np.float64)
    off = np.abs(got - want) - R.PRODUCT_TOL * np.abs(want) - extra
    assert (off <= 0).all(), (np.argwhere(off > 0)[:3], float(off.max()))


MS = [1, 2, 5, 8, 16, 17, 33, 64, 65, 128, 130, 255, 256, 300]
NK = [(1, 16), (3, 48), (16, 128), (100, 144), (130, 1024), (257, 2064), (1040, 512)]


@pytest.mark.parametrize("n,k", NK)
@pytest.mark.parametrize("m", MS)
def test_product(ih, m, n, k):
    a = operands(rng(11, m, n, k), m, n, k)
    near(ih.gemm_i8(*map(cu, a)), R.product(*a))


@pytest.mark.parametrize("n,k", [(5, 32), (257, 2064), (640, 4096)])
@pytest.mark.parametrize("m", [1, 7, 20, 64, 100, 259])
def test_product_added(ih, m, n, k):
    r = rng(12, m, n, k)
    a = operands(r, m, n, k)
    y = (1e4 * r.standard_normal((m, n))).astype(np.float32)
    want = R.product(*a)
    out = cu(y)
    assert ih.gemm_i8(*map(cu, a), accum=True, out=out) is out
    total = want + y
    near(out, total, R.PRODUCT_TOL * np.abs(want) + R.HALF * np.abs(total))  # (the product's roundings, then the sum's)


@pytest.mark.parametrize("m,n,k", [(1, 24576, 4096), (5, 4096, 12288), (3, 20000, 256), (64, 12288, 2048), (515, 4096, 4096),
                                   (700, 1000, 8192), (2050, 1030, 512), (1, 151936, 64), (4000, 17, 128)])
def test_product_large(ih, m, n, k):
    a = operands(rng(13, m, n, k), m, n, k)
    near(ih.gemm_i8(*map(cu, a)), R.product(*a))


@pytest.mark.parametrize("n", [1, 3, 70])
def test_product_of_a_million_tokens(ih, n):
    """More tokens than 65535 groups of 16, few channels."""
    a = operands(rng(20, n), 16 * 65535 + 19, n, 16)
    near(ih.gemm_i8(*map(cu, a)), R.product(*a))


@pytest.mark.parametrize("m", [1, 40, 130])
def test_largest_sums(ih, m):
    """K = 65536 of the extreme codes, -128 among them: sums up to 2^30."""
    import torch
    k, n = 65536, 40
    q, w = np.full((m, k), -127, np.int8), np.full((n, k), 127, np.int8)
    q[0], w[1], w[2, ::2], w[3] = -128, -128, -127, 0
    one = lambda c: np.ones(c, np.float32)  # noqa: E731
    got = ih.gemm_i8(cu(q), cu(one(m)), cu(w), cu(one(n)))
    want = q.astype(np.int64).sum(-1)  # (rows of w are one value, but the third)
    exact = np.stack([want * 127] * n, 1)
    exact[:, 1] = want * -128
    exact[:, 2] = (q.astype(np.int64) @ w[2].astype(np.int64))
    exact[:, 3] = 0
    assert torch.equal(got.cpu(), torch.from_numpy(exact).float())


@pytest.mark.parametrize("m,n,k", [(3, 50, 96), (70, 131, 272), (300, 257, 144)])
def test_product_strides(ih, m, n, k):
    """Operands and results inside wider buffers, rows of odd length; what lies beside the results stays."""
    import torch
    r = rng(14, m, n, k)
    q, s, w, ws = operands(r, m, n, k)
    qd, wd = cu(r.integers(-128, 128, (m, k + 80)).astype(np.int8)), cu(r.integers(-128, 128, (n, k + 48)).astype(np.int8))
    qd[:, 32:32 + k], wd[:, 16:16 + k] = cu(q), cu(w)
    for ld, at in ((n + 5, 1), (n + 8 - n % 4, 4)):
        out = torch.full((m + 2, ld), 5.0, device="cuda")
        view = out[1:m + 1, at:at + n]
        ih.gemm_i8(qd[:, 32:32 + k], cu(s), wd[:, 16:16 + k], cu(ws), out=view)
        near(view, R.product(q, s, w, ws))
        rest = out.clone()
        rest[1:m + 1, at:at + n] = 5.0
        assert bool((rest == 5.0).all())


def test_a_rows_results_are_its_own(ih):
    """The same bits for a row and a channel from every kernel, alone or among others, added to y or not."""
    import torch
    q, s, w, ws = (cu(v) for v in operands(rng(26), 700, 1540, 8208))
    y = ih.gemm_i8(q, s, w, ws)
    for m, n in ((1, 1540), (5, 1540), (64, 1540), (130, 700), (300, 1540), (700, 16), (700, 1)):
        assert torch.equal(ih.gemm_i8(q[:m], s[:m], w[:n], ws[:n]), y[:m, :n]), (m, n)
        out = torch.ones((m, n), device="cuda")
        assert torch.equal(ih.gemm_i8(q[:m], s[:m], w[:n], ws[:n], accum=True, out=out), y[:m, :n] + 1), (m, n)


@pytest.mark.parametrize("m,n,k", [(5, 300, 272), (491, 668, 32), (385, 1923, 2576), (1012, 1860, 176), (300, 2001, 8208), (700, 1540, 8208)])
def test_added_after_its_rounding(ih, m, n, k):
    """The product's roundings, then that of the addition, each by itself: the same bits as the four steps one by one."""
    import torch
    q, s, w, ws = (cu(v) for v in operands(rng(27, m), m, n, k))
    y = cu(rng(28, m).standard_normal((m, n)).astype(np.float32)) * 1e4
    want = torch.from_numpy(R.product(*(a.cpu().numpy() for a in (q, s, w, ws)))).cuda()
    steps = (q.double() @ w.double().T).float() * s[:, None] * ws
    near(steps, want.cpu().numpy())
    assert torch.equal(ih.gemm_i8(q, s, w, ws), steps)
    want = steps + y
    assert torch.equal(ih.gemm_i8(q, s, w, ws, accum=True, out=y), want)


def test_scales_not_finite(ih):
    """A row of scale NaN is NaN, the others are not."""
    m, n, k = 70, 40, 64
    q, s, w, ws = operands(rng(15), m, n, k)
    s[3] = np.nan
    got = ih.gemm_i8(cu(q), cu(s), cu(w), cu(ws))
    assert got[3].isnan().all()
    keep = np.arange(m) != 3
    near(got[cu(keep)], R.product(q, s, w, ws)[keep])


@pytest.mark.parametrize("m", [1, 40, 300])
def test_other_stream_and_capture(ih, m):
    """On a given stream, and captured: replays with other inputs in the same buffers, eager calls between them."""
    import torch
    n, k = 520, 1024
    r = rng(16, m)
    side = torch.cuda.Stream()
    x, add = cu(rows(r, m, k)), cu(r.standard_normal((m, k)).astype(np.float32))
    w, ws = ih.quantize_i8(cu(r.standard_normal((n, k)).astype(np.float32)))
    side.wait_stream(torch.cuda.current_stream())
    xs = x.clone()
    side.wait_stream(torch.cuda.current_stream())
    q, s = ih.rmsnorm_i8(xs, add=add, stream=side)
    y = ih.gemm_i8(q, s, w, ws, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    want = ih.gemm_i8(*ih.rmsnorm_i8(x, add=add), w, ws)
    assert torch.equal(y, want) and torch.equal(x, xs)
    q, s = torch.empty((m, k), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    out = torch.zeros((m, n), device="cuda")
    space = torch.empty(max(16, ih.gemm_i8_ws_bytes(m, n, k, True)), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ih.rmsnorm_i8(x, add=add, out=q, scales=s)
        ih.gemm_i8(q, s, w, ws, accum=True, out=out, ws=space)
    for i in range(4):
        x0 = rows(rng(17, i), m, k)
        y0 = r.standard_normal((m, n)).astype(np.float32)
        x.copy_(cu(x0)), out.copy_(cu(y0)), space.random_()
        g.replay()
        torch.cuda.synchronize()
        xe, ye = cu(x0), cu(y0)
        ih.gemm_i8(*ih.rmsnorm_i8(xe, add=add), w, ws, accum=True, out=ye)
        assert torch.equal(x, xe) and torch.equal(out, ye), i


def test_repeats_are_equal(ih):
    import torch
    for m, n, k in ((5, 4096, 12288), (64, 1000, 4096), (515, 1030, 4096)):
        a = [cu(v) for v in operands(rng(18, m), m, n, k)]
        first = ih.gemm_i8(*a)
        for _ in range(5):
            assert torch.equal(ih.gemm_i8(*a), first)


def in_parts(ih):
    """Products whose K goes in parts through a workspace."""
    shapes = ((515, 1030, 12288), (700, 1000, 8192), (300, 2001, 8208), (500, 1500, 16400), (100, 2050, 16400), (200, 2048, 16384))
    found = [s for s in shapes if ih.gemm_i8_ws_bytes(*s)]  # (2 to 8 parts)
    assert len(found) >= 3
    return found


@pytest.mark.parametrize("accum", [False, True])
def test_workspace_ends(ih, accum):
    """A workspace of just its size, any bytes in it, with bytes behind it that stay; rows of y of any length."""
    import torch
    for m, n, k in in_parts(ih):
        r = rng(21, m, n, k)
        a = operands(r, m, n, k)
        need = ih.gemm_i8_ws_bytes(m, n, k, accum)
        space = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
        space[:need].random_()
        y = r.standard_normal((m, n + 3)).astype(np.float32)
        out = cu(y)
        ih.gemm_i8(*map(cu, a), accum=accum, out=out[:, 1:n + 1], ws=space[:need])
        want = R.product(*a)
        total = want + y[:, 1:n + 1] if accum else want
        near(out[:, 1:n + 1], total, R.PRODUCT_TOL * np.abs(want) + R.HALF * np.abs(total) if accum else 0.0)
        assert bool((space[need:] == 0x5a).all())
        out = out.cpu().numpy()
        assert np.array_equal(out[:, 0], y[:, 0]) and np.array_equal(out[:, n + 1:], y[:, n + 1:])
        with pytest.raises(ih.HipError):
            ih.gemm_i8(*map(cu, a), ws=space[:need - 1] if not accum else space[:16])


def test_two_streams_at_once(ih):
    """Calls that overlap in time, each with its own workspace or one that it makes itself."""
    import torch
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for m, n, k in in_parts(ih):
        ops = [[cu(v) for v in operands(rng(22, m, i), m, n, k)] for i in range(2)]
        want = [ih.gemm_i8(*o) for o in ops]
        outs = [[], []]
        for side in sides:
            side.wait_stream(torch.cuda.current_stream())
        for _ in range(8):
            for i in range(2):
                outs[i].append(ih.gemm_i8(*ops[i], stream=sides[i]))
        for side in sides:
            torch.cuda.current_stream().wait_stream(side)
        for i in range(2):
            assert all(torch.equal(o, want[i]) for o in outs[i])


def test_captured_with_its_own_workspace(ih):
    """Two graphs of calls that make codes, scales, results and workspace themselves, replayed in turn with eager calls between."""
    import torch
    (m, n, k), (m2, n2, k2) = in_parts(ih)[:2]
    r = rng(23)
    w, w2 = (ih.quantize_i8(cu(r.standard_normal(s).astype(np.float32))) for s in ((n, k), (n2, k2)))
    x, x2 = (torch.zeros(s, device="cuda") for s in ((m, k), (m2, k2)))
    graphs, outs = [], []
    for a, b in ((x, w), (x2, w2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ih.gemm_i8(*ih.quantize_i8(a), *b))
        graphs.append(g)
    for i in range(3):
        x.copy_(cu(rows(r, m, k))), x2.copy_(cu(rows(r, m2, k2)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b, o in ((x, w, outs[0]), (x2, w2, outs[1])):
            assert torch.equal(o, ih.gemm_i8(*ih.quantize_i8(a), *b)), i


def test_single_rows_of_any_stride(ih):
    """A single token's, a single channel's row: its stride has no meaning."""
    r = rng(24)
    a = operands(r, 1, 1, 48)
    q, s, w, ws = map(cu, a)
    near(ih.gemm_i8(q.as_strided((1, 48), (1, 1)), s, w.as_strided((1, 48), (7, 1)), ws), R.product(*a))
    x = rows(r, 1, 48)
    same(ih.quantize_i8(cu(x).as_strided((1, 48), (5, 1))), R.quantize(x), R.HALF)


def test_offsets_past_32_bits(ih):
    """Codes, weights, rows and results of more than 2^32 bytes or 2^31 values: the last rows are those of a call on them alone."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(25)
    codes = lambda m, k: torch.randint(-127, 128, (m, k), dtype=torch.int8, device="cuda", generator=g)  # noqa: E731
    ones = lambda m: torch.rand(m, device="cuda", generator=g)  # noqa: E731
    big, small, sb, ss = codes(600000, 8192), codes(40, 8192), ones(600000), ones(40)  # 4.9 GB
    y = ih.gemm_i8(small[:3], ss[:3], big, sb)
    assert torch.equal(y[:, -70:], ih.gemm_i8(small[:3], ss[:3], big[-70:].clone(), sb[-70:].clone()))
    y = ih.gemm_i8(big, sb, small, ss)
    assert torch.equal(y[-70:], ih.gemm_i8(big[-70:].clone(), sb[-70:].clone(), small, ss))
    del big, y
    q, w, s, ws = codes(80000, 64), codes(30001, 64), ones(80000), ones(30001)
    y = ih.gemm_i8(q, s, w, ws)  # 2.4e9 values
    assert torch.equal(y[-70:], ih.gemm_i8(q[-70:].clone(), s[-70:].clone(), w, ws))
    before = y[-70:].clone()
    ih.gemm_i8(q, s, w, ws, accum=True, out=y)
    assert torch.equal(y[-70:], before + before)
    del y
    x = torch.randn((300000, 8192), device="cuda", generator=g)  # 2.5e9 values
    # (a norm's sum of squares is added in an order that depends on the number of rows: each of the two scales is within
    # norm_tol of the exact one, so they are within twice that of each other)
    alike = lambda s, rs: bool(((s[-70:].double() - rs).abs() <= 2 * R.norm_tol(8192) * rs).all())  # noqa: E731
    for call in (ih.quantize_i8, ih.silu_mul_i8, ih.rmsnorm_i8):
        (c, s), (rc, rs) = call(x), call(x[-70:].clone())
        assert torch.equal(c[-70:], rc) and (alike(s, rs) if call is ih.rmsnorm_i8 else torch.equal(s[-70:], rs))
    add = torch.full_like(x, 0.5)
    last = x[-70:] + 0.5
    c, s = ih.rmsnorm_i8(x, add=add)
    rc, rs = ih.rmsnorm_i8(last.clone())
    assert torch.equal(x[-70:], last) and torch.equal(c[-70:], rc) and alike(s, rs)


def test_python_refusals(ih):
    import torch
    x = torch.zeros((4, 64), device="cuda")
    q, s = ih.quantize_i8(x)
    w, ws = torch.zeros((8, 64), dtype=torch.int8, device="cuda"), torch.zeros(8, device="cuda")
    for bad in (lambda: ih.quantize_i8(x.double()), lambda: ih.quantize_i8(x.t()), lambda: ih.quantize_i8(x, out=q.float()),
                lambda: ih.quantize_i8(x, scales=s[:3]), lambda: ih.rmsnorm_i8(x, ws), lambda: ih.rmsnorm_i8(x, add=x[:, :32]),
                lambda: ih.gemm_i8(q, s, w, ws, accum=True), lambda: ih.gemm_i8(q, s[:3], w, ws), lambda: ih.gemm_i8(q, s, w, ws[:5]),
                lambda: ih.gemm_i8(q[:, :48], s, w, ws), lambda: ih.gemm_i8(x, s, w, ws), lambda: ih.gemm_i8(q.t(), s, w, ws),
                lambda: ih.gemm_i8(q, s, w, ws, out=torch.zeros((4, 7), device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ih.quantize_i8(x[:, :40]), lambda: ih.quantize_i8(x[:, 1:49]), lambda: ih.gemm_i8(q[:, 8:56], s, w[:, :48], ws)):
        with pytest.raises(ih.HipError):
            bad()


# ---------------------------------------------------------------- as they are used

@pytest.mark.parametrize("name", ["Q4_K", "Q6_K", "Q8_0"])
def test_weights(ih, name):
    """A GGUF matrix as codes: those of its dequantized rows."""
    from inferno_hip import formats as F, synth
    n, k, qt = 300, 512, getattr(F, name)
    w = synth.matrix(qt, n, k, synth.stream_for(0x1F3E0001, "int8.w"))
    d = cu(w)
    codes, scales = ih.quantize_weights_i8(qt, d, n, k)
    same((codes, scales), R.quantize(ih.dequant(qt, d, n * k).view(n, k).cpu().numpy()), R.HALF)


@pytest.mark.parametrize("name,k", [("Q6_K", 768), ("Q8_0", 32 * 27)])
def test_weights_of_several_pieces(ih, name, k):
    """More values than are dequantized at a time; pieces whose blocks begin at any 2 bytes, rows not a multiple of 128."""
    from inferno_hip import formats as F
    from inferno_hip.quantized_kernels import synth_blocks
    qt, step = getattr(F, name), (64 << 20) // k
    n, row = step + 300, k // F.BLOCK_ELEMS[getattr(F, name)] * F.BLOCK_BYTES[getattr(F, name)]
    d = synth_blocks(qt, 0x1F3E0002, n * row // F.BLOCK_BYTES[qt])
    codes, scales = ih.quantize_weights_i8(qt, d, n, k)
    assert codes.shape == (n, k) and codes.stride(0) % 128 == 0
    for i in (0, step - 40, n - 40):
        x = ih.dequant(qt, d[i * row:(i + 40) * row].clone(), 40 * k).view(40, k).cpu().numpy()
        same((codes[i:i + 40], scales[i:i + 40]), R.quantize(x), R.HALF)
    for i in range(0, n, 1 << 15):  # (the rows between: no code differs from those of the whole matrix in one piece)
        j = min(n, i + (1 << 15))
        q, s = ih.quantize_i8(ih.dequant(qt, d[i * row:j * row].clone(), (j - i) * k).view(j - i, k))
        assert bool((q == codes[i:j]).all()) and bool((s == scales[i:j]).all())


@pytest.mark.parametrize("m,start", [(150, 0), (1, 37), (5, 3)])
def test_layer(ih, m, start):
    """A decoder layer's prompt (or next tokens) on codes, from the residual stream to the residual stream: each step against
    its definition on what the step before left."""
    import torch
    H, NQ, NKV, D, F = 256, 4, 2, 64, 528
    r = rng(19, m)
    weight = lambda n, k: ih.quantize_i8(cu((r.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)))  # noqa: E731
    wqkv, wo, wgu, wdown = weight((NQ + 2 * NKV) * D, H), weight(H, NQ * D), weight(2 * F, H), weight(H, F)
    n1, n2 = (cu((1 + 0.1 * r.standard_normal(H)).astype(np.float32)) for _ in range(2))
    cache = ih.KVCache(*(cu(r.standard_normal((1, 256, NKV, D)).astype(np.float16)) for _ in "kv"))
    lengths = torch.tensor([start], dtype=torch.int32, device="cuda")
    x = cu(rows(r, m, H) * 0.2)

    def product(codes, w, out=None):
        before = None if out is None else out.cpu().numpy()
        y = ih.gemm_i8(*codes, *w, accum=out is not None, out=out)
        want = R.product(*(t.cpu().numpy() for t in (*codes, *w)))
        if out is None:
            near(y, want)
        else:
            near(y, want + before, R.PRODUCT_TOL * np.abs(want) + R.HALF * np.abs(want + before))
        return y

    codes = ih.rmsnorm_i8(x, n1)
    same(codes, R.rmsnorm(x.cpu().numpy(), n1.cpu().numpy()), R.norm_tol(H))
    qkv = product(codes, wqkv)
    q = ih.rope_append(qkv, NQ, cache, lengths, ih.RopeParams(D))
    o = ih.attn_prefix(q, NQ, cache, lengths)
    codes = ih.quantize_i8(o)
    same(codes, R.quantize(o.cpu().numpy()), R.HALF)
    product(codes, wo, out=x)
    codes = ih.rmsnorm_i8(x, n2)
    same(codes, R.rmsnorm(x.cpu().numpy(), n2.cpu().numpy()), R.norm_tol(H))
    gu = product(codes, wgu)
    codes = ih.silu_mul_i8(gu)
    same(codes, R.quantize(R.silu_mul(gu.cpu().numpy())), R.HALF)
    product(codes, wdown, out=x)
    assert bool(x.isfinite().all())
