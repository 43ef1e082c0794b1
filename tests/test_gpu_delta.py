"""The gated delta rule against the recurrence in 64 bits.

Tolerance: a token's contribution to the state is a few sums of dk products, off by about sqrt(dk) 2^-24 of its size, and
the rule does not enlarge what older tokens left (|I - beta k k^T| <= 1 for unit keys and beta in [0, 1], decay <= 1), so
the errors of T tokens stay independent parts of a state that is itself their sum: about sqrt(128) 2^-24 = 7e-7 relative,
in the 2-norm; eight times that is allowed."""
import numpy as np
import pytest

import _mixref as R
from _util import rel_l2

pytestmark = pytest.mark.gpu
TOL = 8 * 128 ** 0.5 * 2.0 ** -24


@pytest.fixture(scope="module")
def ih():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import inferno_hip
    assert inferno_hip.quant_kernels_available(), inferno_hip._lib.last_error()
    return inferno_hip


def make(s, t, hk, hv, dk, dv, seed=0, unit=True, rate=1.0):
    """Inputs on the GPU; keys of unit length where the rule is not asked to make them so."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    r = lambda *a: torch.randn(a, generator=g, device="cuda")  # noqa: E731
    q, k, v = r(s, t, hk, dk), r(s, t, hk, dk) + 0.5, r(s, t, hv, dv)
    if unit:
        q, k = (torch.nn.functional.normalize(x, dim=-1) for x in (q, k))
    decay = -rate * torch.nn.functional.softplus(r(s, t, hv))
    return q, k, v, decay, torch.sigmoid(r(s, t, hv)), 0.3 * r(s, hv, dk, dv)


def check(got, want, what):
    """Within TOL of the norm, and what fp32 cannot hold: with e^g < 1 and no writes a state of any size falls below the
    smallest normal number 2^-126 after enough tokens (0.3 e^(-0.7 200) = 1e-61), where fp32 keeps less than 24 bits or
    zero, so each value may be off by up to 2^-126 besides."""
    diff = float((got.double().cpu() - want).norm())
    allowed = TOL * float(want.norm()) + 2.0 ** -126 * want.numel() ** 0.5
    assert diff <= allowed, (what, diff, allowed, float(want.norm()))


SHAPES = [(1, 1, 1, 1, 64, 4), (1, 1, 16, 32, 128, 128), (2, 5, 2, 4, 128, 128), (3, 2, 1, 3, 64, 36), (1, 63, 2, 2, 64, 64),
          (1, 64, 2, 4, 128, 128), (2, 65, 2, 2, 128, 96), (1, 128, 1, 1, 128, 16), (1, 130, 4, 4, 64, 20),
          (3, 333, 2, 4, 128, 128), (2, 1000, 1, 2, 64, 132), (1, 257, 1, 1, 128, 512), (20, 70, 1, 1, 64, 64)]


@pytest.mark.parametrize("l2norm", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rule(ih, shape, l2norm):
    """o and the last state; the state replaced in place gives the same."""
    import torch
    s, t, hk, hv, dk, dv = shape
    q, k, v, g, b, st = make(*shape, seed=t, unit=not l2norm, rate=0.2)
    o, _, last = R.delta(q, k, v, g, b, st, l2norm=l2norm)
    new = torch.empty_like(st)
    got = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, l2norm=l2norm)
    check(got, o, "o")
    check(new, last, "state")
    st2 = st.clone()
    got2 = ih.gated_delta_rule(q, k, v, g, b, st2, new_state=st2, l2norm=l2norm)
    assert torch.equal(got2, got) and torch.equal(st2, new)


@pytest.mark.parametrize("shape", [(1, 7, 1, 2, 64, 32), (2, 200, 2, 2, 128, 64)])
def test_no_state_and_scale(ih, shape):
    """state None is zeros; a scale of one's own; the last state not kept."""
    import torch
    q, k, v, g, b, _ = make(*shape, seed=3)
    o, _, last = R.delta(q, k, v, g, b, None, scale=0.37)
    new = torch.empty(shape[0], shape[3], shape[4], shape[5], device="cuda")
    got = ih.gated_delta_rule(q, k, v, g, b, None, new_state=new, scale=0.37)
    check(got, o, "o")
    check(new, last, "state")
    assert torch.equal(ih.gated_delta_rule(q, k, v, g, b, None, scale=0.37), got)


@pytest.mark.parametrize("shape", [(1, 1, 2, 4, 128, 128), (3, 5, 2, 4, 128, 128), (2, 9, 1, 1, 64, 36), (1, 64, 1, 2, 128, 64)])
def test_snapshots(ih, shape):
    """The state after every token; commit_state_ picks one; the given state is left alone."""
    import torch
    s, t, hk, hv, dk, dv = shape
    q, k, v, g, b, st = make(*shape, seed=5)
    o, kept, last = R.delta(q, k, v, g, b, st)
    snap, new, was = torch.full((s, t, hv, dk, dv), float("nan"), device="cuda"), torch.empty_like(st), st.clone()
    got = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, snapshots=snap)
    check(got, o, "o")
    check(snap, kept, "snapshots")
    assert torch.equal(snap[:, -1], new) and torch.equal(st, was)
    n = torch.arange(s, dtype=torch.int32, device="cuda") % t
    ih.commit_state_(st, snap, n)
    for i in range(s):
        assert torch.equal(st[i], snap[i, i % t])


@pytest.mark.parametrize("t", [6, 150])
def test_lengths(ih, t):
    """Fewer tokens in some sequences (none, a negative number, more than there are): rows past them as they were, the state
    that of their own last token."""
    import torch
    shape = (6, t, 2, 2, 128, 64)
    lens = [0, t, 1, -3, t + 9, t // 2]
    q, k, v, g, b, st = make(*shape, seed=11)
    for x in (q, k, v, g, b):  # nothing past a sequence's tokens may matter
        for i, n in enumerate(lens):
            x[i, max(0, n):] = float("nan")
    clip = [min(max(n, 0), t) for n in lens]
    o, _, last = R.delta(*(x.nan_to_num(0.0) for x in (q, k, v, g, b)), st, lens=clip)
    out, new = torch.full((6, t, 2, 64), 9.0, device="cuda"), torch.empty_like(st)
    ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"), out=out)
    check(new, last, "state")
    for i, n in enumerate(clip):
        if n:
            check(out[i, :n], o[i, :n], f"o of sequence {i}")
        assert bool((out[i, n:] == 9.0).all()), i
    assert torch.equal(new[0], st[0]) and torch.equal(new[3], st[3])


@pytest.mark.parametrize("t", [5, 200])
@pytest.mark.parametrize("what", ["keep", "forget", "fade_far", "one_key", "no_write", "zero_key", "mixed"])
def test_borders(ih, t, what):
    """No decay at all, all forgotten in a token, decays whose product leaves fp32's range, one key for every token with
    beta 1 (the system's inverse is then a difference, its powers are huge), beta 0, keys of zeros."""
    import torch
    shape = (1, t, 1, 2, 128, 64)
    q, k, v, g, b, st = make(*shape, seed=13)
    if what == "keep":
        g.zero_()
    elif what == "forget":
        g.fill_(-200.0)
    elif what == "fade_far":
        g.fill_(-3.0)
    elif what == "one_key":
        k[:] = k[:, :1].clone()
        b.fill_(1.0)
        g.fill_(-0.001)
    elif what == "no_write":
        b.zero_()
    elif what == "zero_key":
        k.zero_()
    else:
        g[:, ::7] = -60.0
        g[:, 3::7] = 0.0
    o, _, last = R.delta(q, k, v, g, b, st, l2norm=what != "zero_key")
    new = torch.empty_like(st)
    got = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, l2norm=what != "zero_key")
    check(got, o, "o")
    check(new, last, "state")


@pytest.mark.parametrize("t", [3, 100])
def test_views_of_projection_rows(ih, t):
    """q, k, v as parts of one projection's rows, g and beta of another's, o into rows apart."""
    import torch
    s, hk, hv, dk, dv = 2, 2, 4, 64, 32
    q, k, v, g, b, st = make(s, t, hk, hv, dk, dv, seed=17)
    want = ih.gated_delta_rule(q, k, v, g, b, st)
    wide = torch.randn(s * t, 2 * hk * dk + hv * dv + 8, device="cuda")
    x = wide.view(s, t, -1)
    q2, k2 = (x[..., i * hk * dk:(i + 1) * hk * dk].unflatten(-1, (hk, dk)) for i in (0, 1))
    v2 = x[..., 2 * hk * dk:2 * hk * dk + hv * dv].unflatten(-1, (hv, dv))
    gb = torch.randn(s, t, 2 * hv + 1, device="cuda")
    q2.copy_(q), k2.copy_(k), v2.copy_(v), gb[..., :hv].copy_(g), gb[..., hv:2 * hv].copy_(b)
    out = torch.full((s, t, hv * dv + 12), 4.0, device="cuda")
    ih.gated_delta_rule(q2, k2, v2, gb[..., :hv], gb[..., hv:2 * hv], st, out=out[..., : hv * dv].unflatten(-1, (hv, dv)))
    assert torch.equal(out[..., : hv * dv].reshape(s, t, hv, dv), want) and bool((out[..., hv * dv:] == 4.0).all())


def test_split_calls(ih):
    """A long run in one call and in pieces of odd lengths, the state carried."""
    import torch
    q, k, v, g, b, st = make(1, 300, 2, 2, 128, 128, seed=19, rate=0.05)
    new = torch.empty_like(st)
    whole = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new)
    cur, at, parts = st.clone(), 0, []
    for n in (1, 70, 5, 129, 95):
        part = [x[:, at:at + n] for x in (q, k, v, g, b)]
        parts.append(ih.gated_delta_rule(*part, cur, new_state=cur))
        at += n
    assert rel_l2(torch.cat(parts, 1).cpu().numpy(), whole.cpu().numpy()) <= 2 * TOL
    assert rel_l2(cur.cpu().numpy(), new.cpu().numpy()) <= 2 * TOL


@pytest.mark.parametrize("t", [5, 200])
def test_repeats_streams_and_graph(ih, t):
    """The same bits on another stream and from a graph replayed with eager work between, the state carried in place."""
    import torch
    q, k, v, g, b, st = make(2, t, 2, 4, 128, 128, seed=23)
    o2 = make(2, t, 2, 4, 128, 128, seed=24)
    first = st.clone()
    eager, states = [], []
    for _ in range(4):
        eager.append(ih.gated_delta_rule(q, k, v, g, b, st, new_state=st))
        states.append(st.clone())
    st.copy_(first)
    ws = torch.full((ih.gated_delta_rule_ws_bytes(2, t, 2, 4, 128, 128),), 255, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ih.gated_delta_rule(q, k, v, g, b, st, new_state=st, out=out, ws=ws)
    s.synchronize()
    assert torch.equal(out, eager[0]) and torch.equal(st, states[0])
    st.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ih.gated_delta_rule(q, k, v, g, b, st, new_state=st, out=out, ws=ws)
    st.copy_(first)
    for i in range(4):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]) and torch.equal(st, states[i]), i
        ih.gated_delta_rule(*o2[:5], o2[5])


@pytest.mark.parametrize("t", [5, 200])
@pytest.mark.parametrize("far", [float("-inf"), -3e38, -1e6, -150.0])
def test_a_decay_that_clears_the_state(ih, t, far):
    """A token whose decay leaves nothing of the state (where documents are packed one behind the other): the tokens behind
    it are those of a fresh state, with all their digits."""
    import torch
    at = t // 2
    q, k, v, g, b, st = make(2, t, 2, 4, 64, 64, seed=17)
    g[0, at] = far
    g[1, 1], g[1, t - 2] = far, far
    o, _, last = R.delta(q, k, v, g, b, st)
    new = torch.empty_like(st)
    check(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new), o, "o")
    check(new, last, "state")
    fresh, _, alone = R.delta(*(x[:1, at:] for x in (q, k, v, g, b)), torch.zeros_like(st[:1]))
    check(new[:1], alone, "state after the cleared one")


@pytest.mark.parametrize("t,at", [(5, 2), (100, 0), (100, 17), (100, 50), (100, 63), (100, 64), (100, 99), (300, 150)])
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_bad_token_spoils_no_earlier_one(ih, t, at, what, value):
    """One token's q, k, v, g or beta is not finite: the tokens before it, the heads that do not share it, and for v the
    other columns, are as without it; what it reaches is not finite (q: its own row; else every later row, and the state)."""
    import torch
    if what == "g" and value > 0:
        value = float("nan")  # (e^inf times a state is infinite or not a number, which of them is not fixed)
    q, k, v, g, b, st = make(2, t, 2, 4, 128, 64, seed=19)
    o, _, last = R.delta(q, k, v, g, b, st)
    {"q": q, "k": k, "v": v, "g": g, "beta": b}[what][(1, at, 1) + ((5,) if what in ("q", "k", "v") else ())] = value
    new = torch.empty_like(st)
    out = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new)
    bad = torch.zeros(out.shape, dtype=torch.bool)
    gone = torch.zeros(new.shape, dtype=torch.bool)
    if what == "q":
        bad[1, at, 2:] = True
    elif what == "k":
        bad[1, at:, 2:], gone[1, 2:] = True, True
    elif what == "v":
        bad[1, at:, 1, 5], gone[1, 1, :, 5] = True, True
    else:
        bad[1, at:, 1], gone[1, 1] = True, True
    out, new = out.cpu(), new.cpu()
    assert not bool(torch.isfinite(out[bad]).any()) and not bool(torch.isfinite(new[gone]).any())
    check(torch.where(bad, 0.0, out), torch.where(bad, 0.0, o.cpu().double()), "o")
    check(torch.where(gone, 0.0, new), torch.where(gone, 0.0, last.cpu().double()), "state")


@pytest.mark.parametrize("dk,dv", [(64, 32), (128, 128)])
@pytest.mark.parametrize("t", [13, 14, 15, 16, 17, 31, 32, 33, 47])
def test_few_tokens(ih, t, dk, dv):
    """Around the lengths where the recurrence gives way to a chunk, which is then mostly empty."""
    import torch
    q, k, v, g, b, st = make(2, t, 2, 4, dk, dv, seed=23)
    o, _, last = R.delta(q, k, v, g, b, st, l2norm=True)
    new = torch.empty_like(st)
    check(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, l2norm=True), o, "o")
    check(new, last, "state")


@pytest.mark.parametrize("shape", [(64, 65, 4, 12, 64, 8), (64, 65, 4, 8, 128, 16), (1, 4200, 8, 16, 64, 16), (64, 50, 8, 8, 128, 128)])
def test_many_chunks(ih, shape):
    """So many chunks that a key head's value heads (two, three, one) are prepared one after the other, and more columns than
    the GPU carries at once."""
    import torch
    q, k, v, g, b, st = make(*shape, seed=29)
    o, _, last = R.delta(q, k, v, g, b, st, l2norm=True)
    new = torch.empty_like(st)
    check(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, l2norm=True), o, "o")
    check(new, last, "state")


@pytest.mark.parametrize("t", [100])
@pytest.mark.parametrize("size", [1e-12, 1e-6, 1e6, 1e12])
@pytest.mark.parametrize("what", ["v", "state", "q", "k"])
def test_sizes_far_from_one(ih, t, size, what):
    """Values, states, queries of another size than the rest, and keys of one that the rule's own norm undoes: each has a
    scale of its own."""
    import torch
    q, k, v, g, b, st = make(1, t, 1, 2, 128, 64, seed=31)
    l2 = what == "k"
    if what != "k" or size > 1:  # (the square of a small key would meet the norm's own 1e-6)
        {"v": v, "state": st, "q": q, "k": k}[what].mul_(size)
    o, _, last = R.delta(q, k, v, g, b, st, l2norm=l2)
    new = torch.empty_like(st)
    check(ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, l2norm=l2), o, "o")
    check(new, last, "state")


def test_writes_stop_while_the_state_fades(ih):
    """The last tokens of a chunk decay and write nothing: what is left of the state is small beside what the chunk wrote, and
    as exact. Their outputs, sum_j (P T)_rj R_j with R_j = 0 from there on, shrink under the row's other entries, so they are
    allowed what the operand's limbs leave of those: P's row and T's column are brought to below 2^14 (at least 2^13), their
    product is kept times 2^-19 as an fp16 pair, whose last place is 2^-24, so (P T)_rj is off by up to
    2^-25 2^19 2^-13 2^-13 max|P_r| max|T_j| = 2^-32 max|P_r| max|T_j| besides its 22 bits; for unit keys, queries and beta in
    [0, 1] max|P_r| <= 128^-1/2, max|T_j| <= 1 and |R_j| <= |v_j| + |S| of the column."""
    import torch
    q, k, v, g, b, st = make(2, 128, 2, 2, 128, 64, seed=37)
    g.fill_(-1.0)
    b[:, 40:64] = 0.0
    b[:, 100:] = 0.0
    o, kept, last = R.delta(q, k, v, g, b, st)
    new = torch.empty_like(st)
    out = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new)
    check(new, last, "state")
    for i in range(0, 128, 8):
        first = i // 64 * 64
        before = st.double().cpu() if first == 0 else kept[:, first - 1]
        size = v[:, first:first + 64].double().cpu().abs().sum(1) + 64 * before.norm(dim=2)
        allowed = TOL * float(o[:, i:i + 8].norm()) + 2.0 ** -32 * 128 ** -0.5 * 8 ** 0.5 * float(size.norm())
        diff = float((out[:, i:i + 8].double().cpu() - o[:, i:i + 8]).norm())
        assert diff <= allowed, (i, diff, allowed)


def test_two_calls_in_two_graphs(ih):
    """A chunked call and one token by token, each captured with a workspace of its own, replayed beside each other."""
    import torch
    cases, graphs = [], []
    for seed, t in ((53, 300), (59, 7)):
        q, k, v, g, b, st = make(2, t, 2, 4, 128, 64, seed=seed)
        o, _, last = R.delta(q, k, v, g, b, st)
        ws = torch.empty(ih.gated_delta_rule_ws_bytes(2, t, 2, 4, 128, 64), dtype=torch.uint8, device="cuda")
        out, new = torch.empty_like(v), torch.empty_like(st)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, out=out, ws=ws, stream=stream)
        cases.append((o, last, out, new, (q, k, v, g, b, st, ws)))
        graphs.append((graph, stream))
    for turn in range(4):
        for _, _, out, new, _ in cases:
            out.fill_(3.0)
            new.fill_(3.0)
        torch.cuda.synchronize()
        for graph, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o, last, out, new, _ in cases:
            check(out, o, ("o", turn))
            check(new, last, ("state", turn))
