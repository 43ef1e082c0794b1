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
