"""The 8-bit projections where their kernels and their values end."""
import numpy as np
import pytest

import _i8ref as R
from test_gpu_int8 import cu, ih, operands, rng, rows, same  # noqa: F401  (ih: the fixture)

pytestmark = pytest.mark.gpu


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
