"""The gated delta rule at sizes far from one: a state that is tiny when a large write comes, keys and queries whose squares
leave fp32's range. Against the recurrence in 64 bits, chunk by chunk, within test_gpu_delta's tolerance of the chunk's norm."""
import pytest

import _mixref as R
from test_gpu_delta import TOL, check, ih, make  # noqa: F401  (ih: the fixture)

pytestmark = pytest.mark.gpu
# The chunks' kernel brings a column of the state to at least 2^11 by a power of two of up to 2^80, and takes it as two fp16
# limbs, the last place of the second 2^-24: off by up to 2^-25 2^-80 a value where the power is at its end (columns below
# 2^-69). A unit query's product with a column is off by up to sqrt(dk) times that, below 2^-101, besides TOL.
FLOOR = 2.0 ** -101


def check_chunks(out, o, what):
    for at in range(0, o.shape[1], 64):
        got, want = out[:, at:at + 64].double().cpu(), o[:, at:at + 64]
        diff = float((got - want).norm())
        allowed = TOL * float(want.norm()) + FLOOR * want.numel() ** 0.5
        assert diff <= allowed, (what, at, diff, allowed)


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("state,write", [(1e-20, 1e6), (1e-25, 1e5), (1e-30, 1e15), (1e-20, 1e15), (1e-12, 1e20), (0.0, 1e20)])
def test_a_large_write_meets_a_tiny_state(ih, dk, state, write):  # noqa: F811
    """Nothing is written to a tiny state for a chunk, then large values are."""
    import torch
    q, k, v, g, b, st = make(2, 250, 2, 4, dk, 64, seed=61, rate=0.02)
    st.mul_(state)
    b[:, :64] = 0.0
    v.mul_(write)
    o, _, last = R.delta(q, k, v, g, b, st)
    new = torch.empty_like(st)
    check_chunks(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new), o, "o")
    check(new, last, "state")


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("write", [1e5, 1e15])
def test_a_large_write_meets_a_faded_state(ih, dk, write):  # noqa: F811
    """The state fades by e^-64 in a chunk that writes nothing, then large values are written; part of the key heads' values
    stays zero, so that a part of the state's rows takes nothing of them."""
    import torch
    q, k, v, g, b, st = make(2, 250, 2, 4, dk, 64, seed=67, rate=0.02)
    g[:, :64] = -1.0
    b[:, :64] = 0.0
    k[..., : dk // 2] = 0.0
    v.mul_(write)
    o, _, last = R.delta(q, k, v, g, b, st)
    new = torch.empty_like(st)
    check_chunks(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new), o, "o")
    check(new, last, "state")


@pytest.mark.parametrize("dk", [64, 128])
def test_a_large_state_is_cleared_for_small_writes(ih, dk):  # noqa: F811
    """The state's power of two comes from far below one to far above it in a step."""
    import torch
    q, k, v, g, b, st = make(2, 250, 2, 4, dk, 64, seed=71, rate=0.02)
    st.mul_(1e20)
    b[:, :64] = 0.0
    g[:, 63] = float("-inf")
    b[:, 64:128] = 0.0
    b[:, 63] = 1.0
    v[:, 63].mul_(1e-15)
    v[:, 64:].mul_(1e-10)
    o, _, last = R.delta(q, k, v, g, b, st)
    new = torch.empty_like(st)
    out = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new)
    # (the first chunk's outputs are of the large state but for its last token's, which is not judged beside them)
    check_chunks(out[:, 64:], o[:, 64:], "o")
    check(new, last, "state")


@pytest.mark.parametrize("t", [1, 5, 100])
@pytest.mark.parametrize("keys,queries", [(2.0 ** 60, 1.0), (2.0 ** 64, 2.0 ** 64), (2.0 ** 70, 1.0), (1.0, 2.0 ** 75),
                                          (2.0 ** 86, 2.0 ** 86), (2.0 ** 21, 2.0 ** -70)])
@pytest.mark.parametrize("dk,state", [(64, 1.0), (128, 2.0 ** 40)])
def test_norms_of_large_keys_and_queries(ih, t, keys, queries, dk, state):  # noqa: F811
    """l2norm takes keys and queries whose squares, and products with each other and the state, leave fp32's range: what comes
    of them is of ordinary size. (Random normal values below 16: 2^86 times them stay below 2^90.)"""
    import torch
    q, k, v, g, b, st = make(2, t, 2, 4, dk, 64, seed=73, unit=False, rate=0.05)
    q.mul_(queries), k.mul_(keys), st.mul_(state)
    o, _, last = R.delta(q, k, v, g, b, st, l2norm=True)
    new = torch.empty_like(st)
    check_chunks(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, l2norm=True), o, "o")
    check(new, last, "state")


@pytest.mark.parametrize("t", [5, 100])
def test_one_large_key_among_ordinary_ones(ih, t):  # noqa: F811
    """A single token's key and query past the range, tokens and heads beside them as without."""
    import torch
    q, k, v, g, b, st = make(2, t, 2, 4, 128, 64, seed=79, unit=False, rate=0.05)
    plain = ih.gated_delta_rule(q, k, v, g, b, st, l2norm=True)
    k[1, t // 2, 1] *= 2.0 ** 80
    q[1, t // 2, 1] *= 2.0 ** 80
    o, _, last = R.delta(q, k, v, g, b, st, l2norm=True)
    new = torch.empty_like(st)
    got = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, l2norm=True)
    check(got, o, "o")
    check(new, last, "state")
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1, :, :2], plain[1, :, :2])


@pytest.mark.parametrize("t", [5, 100, 250])
@pytest.mark.parametrize("values,states,keys,queries", [(75, 75, 0, 0), (75, -40, 0, 0), (-40, 75, 0, 0), (30, 30, 36, 36)])
def test_sizes_up_to_the_limits(ih, t, values, states, keys, queries):  # noqa: F811
    """v, state, keys and queries times these powers of two (beta such that beta k.k stays): all at their ends at once. Chunk 0 of
    a small state beside large values and the other way round is a sum of both, judged by its norm. (Values of 2^75 with keys of
    2^-40 and such a beta are beyond them: beta v is 2^155 and k (beta v) 2^115, the first of which no fp32 number holds.)"""
    import torch
    q, k, v, g, b, st = make(2, t, 2, 4, 128, 64, seed=83, rate=0.05)
    v.mul_(2.0 ** values), st.mul_(2.0 ** states), k.mul_(2.0 ** keys), q.mul_(2.0 ** queries), b.mul_(2.0 ** (-2 * keys))
    o, _, last = R.delta(q, k, v, g, b, st)
    new = torch.empty_like(st)
    check_chunks(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new), o, "o")
    check(new, last, "state")
