"""The 8-bit projections where their kernels and their values end."""
import numpy as np
import pytest

from test_gpu_int8 import cu, ih, operands, rng  # noqa: F401  (ih: the fixture)

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
