"""attn_prefix at scores far from zero. The scale is the fp32 number next to ln 2, whose product with log2 e rounds to 1: scores
in powers of two are then the dot products themselves. Queries, keys and so scores are chosen to be exact in fp32 and in the
limbs, so weights are exact powers of two and the outputs are off by the limbs of q and P and by sums alone: 2^-20 of the
values' size."""
import numpy as np
import pytest

from test_gpu_delta import ih  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
LN2 = float(np.float32(np.log(2.0)))
assert np.float32(LN2) * np.float32(1.44269504088896341) == np.float32(1.0)


def attend(ih, q, key_a, key_b, period, p, d, dtype, own, hide=False):
    """One query row over p entries: key_a in the first `period` of each 2 period, key_b in the others. Returns the output, the
    sums of either's values in 64 bits, their numbers, and the largest value. hide: the new entry of a sequence that has
    nothing else of its own (score and value 0) is not seen."""
    import torch
    dt = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.zeros(1, p, 1, d, device="cuda", dtype=dt)
    a = (torch.arange(p, device="cuda") // period % 2 == 0)
    for key, at in ((key_a, a), (key_b, ~a)):
        for i, x in enumerate(key):
            k[0, at, 0, i] = x
    v = torch.randn(1, p, 1, d, generator=gen, device="cuda").to(dt)
    x = torch.zeros(1, d, device="cuda")
    for i, y in enumerate(q):
        x[0, i] = y
    if own:  # the entries are the sequence's own, the last of them the new one
        got = ih.attn_prefix(x, 1, ih.KVCache(k, v), torch.tensor([p - 1], dtype=torch.int32, device="cuda"), scale=LN2)
    else:
        z = torch.zeros(1, 1, 1, d, device="cuda", dtype=dt)
        got = ih.attn_prefix(x, 1, ih.KVCache(z, z.clone()), torch.zeros(1, dtype=torch.int32, device="cuda"),
                             prefix=ih.KVCache(k, v), scale=LN2,
                             tree_mask=torch.zeros(1, 1, dtype=torch.int64, device="cuda") if hide else None)
    v = v.double()[0, :, 0]
    return got.double()[0], v[a].sum(0), v[~a].sum(0), int(a.sum()), int((~a).sum()), float(v.abs().max())


def check(got, sa, sb, na, nb, size, wb):
    want = (sa + wb * sb) / (na + wb * nb)
    assert bool((abs(got - want) <= 2.0 ** -20 * size).all()), (got[:4].tolist(), want[:4].tolist())


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("exponent", [10, 20, 23, 24, 25])
def test_a_score_a_little_above_a_far_one(ih, exponent, d, dtype, own):  # noqa: F811
    """The largest score so far is 2^exponent, a later one 8 above it: the reference has to follow, also where fp32's numbers are
    2 and 4 apart."""
    half = exponent // 2
    q, a, b = [2.0 ** (exponent - half), 1.0], [2.0 ** half, 0.0], [2.0 ** half, 8.0]
    check(*attend(ih, q, a, b, 128, 65536, d, dtype, own), wb=256.0)


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("period", [128, 16384])
def test_scores_where_numbers_are_16_apart(ih, period, d, dtype, own):  # noqa: F811
    """Scores of 3 2^26 and 16 more, in the same ranges of keys and in ranges of their own: a reference 8 below is between two
    fp32 numbers."""
    q, a, b = [3 * 2.0 ** 13, 1.0], [2.0 ** 13, 0.0], [2.0 ** 13, 16.0]
    check(*attend(ih, q, a, b, period, 65536, d, dtype, own), wb=65536.0)
    check(*attend(ih, q, b, b, period, 65536, d, dtype, own), wb=1.0)
    low = [-y for y in q]
    check(*attend(ih, low, a, b, period, 65536, d, dtype, own, hide=True), wb=2.0 ** -16)
    if not own:  # (the new entry's score of 0 is then far above all others)
        assert bool((attend(ih, low, a, b, period, 65536, d, dtype, own)[0] == 0).all())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("exponent", [-120, -104, 100, 112, 118, 122])
def test_queries_of_any_size(ih, exponent, dtype):  # noqa: F811
    """Queries of 2^exponent over small keys: scores that fp32 holds, of which the larger takes everything (or, where they are
    tiny, an equal share)."""
    q, a, b = [2.0 ** exponent], [2.0 ** -9], [2.0 ** -10]
    got, sa, sb, na, nb, size = attend(ih, q, a, b, 128, 8192, 64, dtype, False, hide=True)
    check(got, sa, sb, na, nb, size, wb=0.0 if exponent > 0 else 1.0)
    check(*attend(ih, q, [0.0], [0.0], 128, 8192, 64, dtype, False, hide=True), wb=1.0)
