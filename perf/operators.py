"""Cases of the token mixers of a hybrid decoder layer, for timing and for comparing outputs.

A case is a dict of plain values whose "kind" says which operator it takes:

* append  rotary positions applied to the q and k heads of the [q; k; v] rows of
          each sequence's new tokens; k and v go to the KV cache behind its length;
* rope    rotary positions of one tensor's heads, no cache;
* attn    attention of each sequence's m new tokens over a prefix that all
          sequences share, its own cached tokens and the new ones (causal, or
          the ancestors in a draft tree);
* delta   the gated delta rule over a batch of sequences, key heads shared by
          value heads, from a given state; "snap" keeps the state after every
          token, as a verify step does.

Where `own` is false, run() computes them in plain torch operations.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64  # tokens that the plain gated delta rule takes at a time


def listed():
    return [
        # the next token of one conversation: the time is latency
        {"name": "append_s1_m1", "kind": "append", "s": 1, "m": 1, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "cap": 1024, "type": "f16", "pairs": "half", "scaling": "none", "len": 700},
        # a prompt's tokens into the cache: wide heads of which a quarter rotates, positions scaled for a long context
        {"name": "append_prompt_8190", "kind": "append", "s": 1, "m": 8190, "hq": 16, "hkv": 4, "d": 256, "rot": 64,
         "cap": 9000, "type": "bf16", "pairs": "half", "scaling": "by_parts", "len": 513},
        # the q rows of a 64-node draft tree, far positions, interleaved pairs
        {"name": "rope_tree_64", "kind": "rope", "n": 64, "h": 32, "d": 128, "rot": 128, "pairs": "interleaved",
         "scaling": "linear", "pos": 900001},
        # one conversation's next token over its system prompt and its own turns
        {"name": "attn_s1_m1_p777", "kind": "attn", "s": 1, "m": 1, "hq": 32, "hkv": 8, "d": 128, "p": 777, "len": 150,
         "type": "f16", "tree": False},
        # a very long document and one question: reading the cache is all there is
        {"name": "attn_s1_m1_p131072", "kind": "attn", "s": 1, "m": 1, "hq": 32, "hkv": 8, "d": 128, "p": 131072,
         "len": 33, "type": "f16", "tree": False},
        # a 64-node draft tree of one sequence, wide heads
        {"name": "attn_tree_64_p6001", "kind": "attn", "s": 1, "m": 64, "hq": 16, "hkv": 4, "d": 256, "p": 6001,
         "len": 200, "type": "bf16", "tree": True},
        # a verify step of 9 sequences of a small model, an odd prefix
        {"name": "attn_s9_m5_p4099", "kind": "attn", "s": 9, "m": 5, "hq": 16, "hkv": 4, "d": 64, "p": 4099, "len": 301,
         "type": "bf16", "tree": False},
        # the largest: 64 sequences' verify step over a shared document
        {"name": "attn_s64_m5_p16384", "kind": "attn", "s": 64, "m": 5, "hq": 32, "hkv": 8, "d": 128, "p": 16384,
         "len": 512, "type": "f16", "tree": False},
        # the next token of one conversation
        {"name": "delta_s1_t1", "kind": "delta", "s": 1, "t": 1, "hk": 16, "hv": 32, "dk": 128, "dv": 128, "snap": False},
        # a verify step (1 accepted + 4 drafted tokens) of 16 sequences, the states kept after each token
        {"name": "delta_s16_t5_snap", "kind": "delta", "s": 16, "t": 5, "hk": 16, "hv": 32, "dk": 128, "dv": 128,
         "snap": True},
        # a long prompt of one sequence
        {"name": "delta_prompt_4096", "kind": "delta", "s": 1, "t": 4096, "hk": 16, "hv": 32, "dk": 128, "dv": 128,
         "snap": False},
        # short prompts of several sequences, a small model's heads, an odd length
        {"name": "delta_s6_t333", "kind": "delta", "s": 6, "t": 333, "hk": 8, "hv": 8, "dk": 64, "dv": 96, "snap": False},
    ]


def _spread(rng, lo, hi, step=1):
    """A whole number in [lo, hi], spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + step)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    kind = rng.choice(["append", "rope", "attn", "attn", "attn", "delta", "delta", "delta"])
    d = rng.choice([64, 128, 128, 256])
    if kind == "rope":
        return {"kind": kind, "n": _spread(rng, 1, 4000), "h": rng.choice([4, 8, 16, 20, 32]), "d": d,
                "rot": rng.choice([d, d // 2, d // 4]), "pairs": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "by_parts"]), "pos": _spread(rng, 100, 1000000)}
    if kind == "append":
        hkv = rng.choice([2, 4, 8])
        s = _spread(rng, 1, 64)
        m = _spread(rng, 1, 8000 // s)
        n = _spread(rng, 1, 2000)
        return {"kind": kind, "s": s, "m": m, "hq": hkv * rng.choice([1, 2, 4]), "hkv": hkv, "d": d,
                "rot": rng.choice([d, d // 2, d // 4]), "cap": n + m + rng.randint(0, 100), "type": rng.choice(list(TYPES)),
                "pairs": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "by_parts"]), "len": n}
    if kind == "attn":
        hkv = rng.choice([2, 4, 8] if d < 256 else [2, 4])
        s = _spread(rng, 1, 64)
        m = rng.choice([1, 1, 2, 3, 5, 5, 8, 16]) if s > 4 else rng.choice([1, 3, 5, 8, 31, 64])
        hq = hkv * rng.choice([1, 2, 4, 5])
        rows = s * m * hq
        top = min(65536 if rows <= 512 else 24000, 80_000_000 // rows)
        return {"kind": kind, "s": s, "m": m, "hq": hq, "hkv": hkv, "d": d,
                "p": _spread(rng, 200, max(400, top)), "len": _spread(rng, 2, 512),
                "type": rng.choice(list(TYPES)), "tree": m > 2 and rng.random() < 0.4}
    hk = rng.choice([2, 4, 8, 16])
    hv = hk * rng.choice([1, 2, 3]) if hk < 16 else 32
    dk = rng.choice([64, 128, 128])
    form = rng.choice(["token", "verify", "prompt", "prompt"])
    s = _spread(rng, 1, 64 if form == "token" else 24 if form == "verify" else 8)
    t = 1 if form == "token" else rng.randint(2, 9) if form == "verify" else _spread(rng, 40, 4000 // s)
    if form == "verify":
        s = max(1, min(s, 160 * 32 // (2 * t * hv)))
    return {"kind": kind, "s": s, "t": t, "hk": hk, "hv": hv, "dk": dk, "dv": rng.choice([64, 96, 128]),
            "snap": form == "verify"}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _lengths(case, g):
    """Sequence lengths between half the case's length and all of it, each sequence's by the seed."""
    n = torch.linspace(case["len"] // 2 if case["s"] > 1 else case["len"], case["len"], case["s"], device="cuda")
    return n.to(torch.int32)[torch.randperm(case["s"], generator=g, device="cuda")]


def _parents_mask(m, s, g):
    """Ancestor bits of s random draft trees of m nodes (node 0 the root, a node's parent earlier than it)."""
    up = (torch.rand((s, m), generator=g, device="cuda") * torch.arange(m, device="cuda")).long().cpu()
    rows = []
    for t in range(s):
        bits = [1]
        for i in range(1, m):
            bits.append(bits[int(up[t, i])] | 1 << i)
        rows.append([b - (1 << 64) if b >> 63 else b for b in bits])
    return torch.tensor(rows, dtype=torch.int64, device="cuda")


def _inputs(case, seed):
    g = _gen(seed)
    if case["kind"] == "rope":
        x = _randn(g, case["n"], case["h"] * case["d"])
        pos = torch.randint(max(0, case["pos"] - 64), case["pos"] + 64, (case["n"],), generator=g, device="cuda", dtype=torch.int32)
        return {"case": case, "x": x, "pos": pos}
    if case["kind"] == "append":
        s, m, d = case["s"], case["m"], case["d"]
        qkv = _randn(g, s * m, (case["hq"] + 2 * case["hkv"]) * d)
        k, v = (torch.zeros((s, case["cap"], case["hkv"], d), dtype=TYPES[case["type"]], device="cuda") for _ in "kv")
        return {"case": case, "qkv": qkv, "k": k, "v": v, "len": _lengths(case, g)}
    if case["kind"] == "attn":
        s, m, d, hkv, t = case["s"], case["m"], case["d"], case["hkv"], TYPES[case["type"]]
        q = 1.7 * _randn(g, s * m, case["hq"] * d)  # (scores of standard deviation 1.7: some keys count far more than others)
        pk, pv = (_randn(g, 1, case["p"], hkv, d).to(t) for _ in "kv")
        k, v = (_randn(g, s, case["len"] + m + 7, hkv, d).to(t) for _ in "kv")
        n = _lengths(case, g)
        mask = _parents_mask(m, s, g) if case["tree"] else None
        return {"case": case, "q": q, "pk": pk, "pv": pv, "k": k, "v": v, "len": n, "mask": mask}
    s, t, hk, hv, dk, dv = (case[x] for x in ("s", "t", "hk", "hv", "dk", "dv"))
    # keys and queries behind a convolution and an activation: mostly small, some large, a common direction
    q, k = (torch.nn.functional.silu(_randn(g, s, t, hk, dk) + 0.3 * _randn(g, 1, 1, hk, dk)) for _ in "qk")
    v = torch.nn.functional.silu(_randn(g, s, t, hv, dv))
    # decays from almost none to a half a token, by head; write strengths around a half
    rate = torch.exp(torch.empty(hv, device="cuda").uniform_(-6.0, 0.0, generator=g))
    decay = -rate * torch.nn.functional.softplus(_randn(g, s, t, hv))
    beta = torch.sigmoid(_randn(g, s, t, hv))
    state = 0.1 * _randn(g, s, hv, dk, dv)
    return {"case": case, "q": q, "k": k, "v": v, "g": decay, "beta": beta, "state": state}


def _scaling(case):
    return {"none": {}, "linear": {"scaling": "linear", "factor": 8.0},
            "by_parts": {"scaling": "by_parts", "factor": 4.0, "orig_len": 32768, "beta_fast": 32.0, "beta_slow": 1.0,
                         "attn_scale": 0.1 * math.log(4.0) + 1.0}}[case["scaling"]]


BASE = 1000000.0


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:  # the descriptors, outputs and workspaces that a serving loop keeps
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inferno.jl_amd"))
        import inferno_hip as ih
        st["ih"] = ih
        if case["kind"] in ("rope", "append"):
            st["rope"] = ih.RopeParams(case["d"], case["rot"], interleaved=case["pairs"] == "interleaved", base=BASE, **_scaling(case))
        if case["kind"] in ("append", "attn"):
            st["cache"] = ih.KVCache(st["k"], st["v"])
        if case["kind"] == "rope":
            st["out"] = torch.empty_like(st["x"])
        elif case["kind"] == "append":
            st["out"] = torch.empty((case["s"] * case["m"], case["hq"] * case["d"]), device="cuda")
        elif case["kind"] == "attn":
            st["prefix"] = ih.KVCache(st["pk"], st["pv"])
            st["out"] = torch.empty_like(st["q"])
            st["ws"] = torch.empty(ih.attn_prefix_ws_bytes(case["hq"], case["m"], st["cache"], st["prefix"]), dtype=torch.uint8, device="cuda")
        else:
            st["out"] = torch.empty_like(st["v"])
            snap = (case["s"], case["t"], case["hv"], case["dk"], case["dv"])
            st["snap"] = torch.empty(snap, device="cuda") if case["snap"] else None
            st["new"] = None if case["snap"] else torch.empty_like(st["state"])
            n = ih.gated_delta_rule_ws_bytes(case["s"], case["t"], case["hk"], case["hv"], case["dk"], case["dv"], case["snap"])
            st["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    return st


def run(st):
    case = st["case"]
    if own:
        ih = st["ih"]
        if case["kind"] == "rope":
            return ih.rope(st["x"], st["pos"], case["h"], st["rope"], out=st["out"])
        if case["kind"] == "append":
            ih.rope_append(st["qkv"], case["hq"], st["cache"], st["len"], st["rope"], out=st["out"])
            return {"q": st["out"], "k": st["k"], "v": st["v"]}
        if case["kind"] == "attn":
            return ih.attn_prefix(st["q"], case["hq"], st["cache"], st["len"], prefix=st["prefix"], tree_mask=st["mask"],
                                  out=st["out"], ws=st["ws"])
        ih.gated_delta_rule(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"], new_state=st["new"],
                            snapshots=st["snap"], l2norm=True, out=st["out"], ws=st["ws"])
        return {"o": st["out"], "state": st["snap"] if case["snap"] else st["new"]}
    return {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn, "delta": _plain_delta}[case["kind"]](st)


# ---------------------------------------------------------------- plain forms

def _plain_angles(case, pos):
    """cos and sin [n, 1, rot / 2] of positions [n], the angles in 64 bits."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=pos.device)
    f = BASE ** (-2.0 * i / case["rot"])
    o = _scaling(case)
    if case["scaling"] == "linear":
        f = f / o["factor"]
    elif case["scaling"] == "by_parts":
        keep = ((o["orig_len"] * f / (2 * math.pi) - o["beta_slow"]) / (o["beta_fast"] - o["beta_slow"])).clamp(0, 1)
        f = (1 - keep) * f / o["factor"] + keep * f
    a = pos.double()[:, None, None] * f
    scale = o.get("attn_scale", 1.0)
    return (torch.cos(a) * scale).float(), (torch.sin(a) * scale).float()


def _plain_rotate(case, x, cos, sin):
    """x [n, h, d] fp32 with its leading entries rotated by pairs."""
    r = case["rot"]
    if case["pairs"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _plain_rope(st):
    case = st["case"]
    cos, sin = _plain_angles(case, st["pos"])
    return _plain_rotate(case, st["x"].view(case["n"], case["h"], case["d"]), cos, sin).view_as(st["x"])


def _plain_append(st):
    case = st["case"]
    s, m, hq, hkv, d = (case[x] for x in ("s", "m", "hq", "hkv", "d"))
    slot = st["len"].long()[:, None] + torch.arange(m, device="cuda")
    cos, sin = _plain_angles(case, slot.reshape(-1))
    x = st["qkv"].view(s * m, hq + 2 * hkv, d)
    qk = _plain_rotate(case, x[:, :hq + hkv], cos, sin)
    at = torch.arange(s, device="cuda")[:, None], slot
    st["k"][at] = qk[:, hq:].reshape(s, m, hkv, d).to(st["k"].dtype)
    st["v"][at] = x[:, hq + hkv:].reshape(s, m, hkv, d).to(st["v"].dtype)
    return {"q": qk[:, :hq].reshape(s * m, hq * d), "k": st["k"], "v": st["v"]}


def _plain_visible(st, keys):
    """[s, m, keys]: which of a sequence's cached and new entries each new token sees."""
    case = st["case"]
    j = torch.arange(keys, device="cuda") - st["len"].long()[:, None, None]  # [s, 1, keys]: 0.. are the new entries
    if st["mask"] is None:
        return j <= torch.arange(case["m"], device="cuda")[None, :, None]
    bit = (st["mask"][:, :, None] >> j.clamp(0, 63)) & 1
    return (j < 0) | ((j < case["m"]) & (bit == 1))


def _plain_attn(st):
    case = st["case"]
    s, m, hq, hkv, d = (case[x] for x in ("s", "m", "hq", "hkv", "d"))
    g = hq // hkv
    q = (st["q"] / math.sqrt(d)).view(s, m, hkv, g, d)
    # the prefix for all sequences at once: [hkv, s m g, d] with [hkv, d, p]
    qp = q.permute(2, 0, 1, 3, 4).reshape(hkv, s * m * g, d)
    zp = qp @ st["pk"][0].permute(1, 2, 0).float().contiguous()
    # each sequence's own entries: [s, hkv, m g, d] with [s, hkv, d, keys]
    qs = q.permute(0, 2, 1, 3, 4).reshape(s, hkv, m * g, d)
    zs = qs @ st["k"].permute(0, 2, 3, 1).float().contiguous()
    keys = zs.shape[-1]
    seen = _plain_visible(st, keys)[:, None, :, None, :]
    zs = zs.view(s, hkv, m, g, keys).masked_fill(~seen, -math.inf)
    zp = zp.view(hkv, s, m, g, -1).permute(1, 0, 2, 3, 4)
    top = torch.maximum(zp.amax(-1, keepdim=True), zs.amax(-1, keepdim=True))
    ep, es = torch.exp(zp - top), torch.exp(zs - top)
    total = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    op = ep.permute(1, 0, 2, 3, 4).reshape(hkv, s * m * g, -1) @ st["pv"][0].permute(1, 0, 2).float().contiguous()
    os_ = es.reshape(s, hkv, m * g, keys) @ st["v"].permute(0, 2, 1, 3).float().contiguous()
    o = op.view(hkv, s, m, g, d).permute(1, 0, 2, 3, 4) + os_.view(s, hkv, m, g, d)
    return (o / total).permute(0, 2, 1, 3, 4).reshape(s * m, hq * d)


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _plain_delta(st):
    """The recurrence written for chunks of tokens: inside a chunk a unit lower triangular system, inverted by blocks of
    twice the size each time; from chunk to chunk the state."""
    case = st["case"]
    s, t, hk, hv, dk, dv = (case[x] for x in ("s", "t", "hk", "hv", "dk", "dv"))
    c = 1 if case["snap"] else min(CHUNK, 1 << (t - 1).bit_length())
    n = -(-t // c)

    def chunks(x, heads):  # [s, t, h, ..] -> [s, hv, n, c, ..], zeros behind the end
        x = x.repeat_interleave(hv // heads, 2).transpose(1, 2)
        x = torch.nn.functional.pad(x, (0, 0) * (x.dim() - 3) + (0, n * c - t))
        return x.reshape(s, hv, n, c, *x.shape[3:])

    q, k, v = chunks(_unit(st["q"]) / math.sqrt(dk), hk), chunks(_unit(st["k"]), hk), chunks(st["v"], hv)
    beta, decay = chunks(st["beta"], hv), chunks(st["g"], hv).cumsum(-1)
    lower = torch.ones((c, c), dtype=torch.bool, device="cuda").tril()
    fade = torch.exp((decay[..., :, None] - decay[..., None, :]).masked_fill(~lower, -math.inf))
    a = (k @ k.transpose(-1, -2)) * fade * beta[..., None]
    inv = torch.eye(c, device="cuda").expand_as(a).contiguous()
    size = 1
    while size < c:  # (the blocks of `size` on the diagonal are inverted: those of 2 size from them)
        shape = (*a.shape[:3], c // (2 * size), 2, size, c // (2 * size), 2, size)
        left, full = inv.view(shape), a.view(shape)
        x = torch.diagonal(left[..., :, 1, :, :, 1, :], dim1=3, dim2=5).movedim(-1, 3)
        y = torch.diagonal(full[..., :, 1, :, :, 0, :], dim1=3, dim2=5).movedim(-1, 3)
        z = torch.diagonal(left[..., :, 0, :, :, 0, :], dim1=3, dim2=5).movedim(-1, 3)
        torch.diagonal(left[..., :, 1, :, :, 0, :], dim1=3, dim2=5).copy_((-(x @ y @ z)).movedim(3, -1))
        size *= 2
    grown = torch.exp(decay)[..., None]
    u, w = inv @ (v * beta[..., None]), inv @ (k * (beta[..., None] * grown))
    inner = (q @ k.transpose(-1, -2)) * fade
    last = torch.exp(decay[..., -1:] - decay)[..., None]
    state, out, kept = st["state"], [], []
    for i in range(n):
        x = u[:, :, i] - w[:, :, i] @ state
        out.append((q[:, :, i] * grown[:, :, i]) @ state + inner[:, :, i] @ x)
        state = state * grown[:, :, i, -1:] + (k[:, :, i] * last[:, :, i]).transpose(-1, -2) @ x
        if case["snap"]:
            kept.append(state)
    o = torch.stack(out, 2).view(s, hv, n * c, dv)[:, :, :t].transpose(1, 2).contiguous()
    return {"o": o, "state": torch.stack(kept, 1) if case["snap"] else state}


# ---------------------------------------------------------------- what a pass needs

def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["n"] * case["h"] * case["d"]
        return {"bytes": 8 * n + 4 * case["n"], "flops": 3 * n}
    if kind == "append":
        rows, d = case["s"] * case["m"], case["d"]
        return {"bytes": rows * d * (4 * (case["hq"] + 2 * case["hkv"]) + 4 * case["hq"] + 4 * case["hkv"]) + 4 * case["s"],
                "flops": 3 * rows * (case["hq"] + case["hkv"]) * case["rot"]}
    if kind == "attn":
        s, m, hq, hkv, d, p = (case[x] for x in ("s", "m", "hq", "hkv", "d", "p"))
        n = case["len"] if s == 1 else (case["len"] // 2 + case["len"]) / 2
        seen = p + n + (m + 1) / 2
        return {"bytes": 4 * hkv * d * (p + s * (n + m)) + 8 * s * m * hq * d, "flops": 4 * s * m * hq * d * seen}
    s, t, hk, hv, dk, dv = (case[x] for x in ("s", "t", "hk", "hv", "dk", "dv"))
    states = 1 + (t if case["snap"] else 1)
    return {"bytes": 4 * s * (t * (2 * hk * dk + 2 * hv * dv + 2 * hv) + states * hv * dk * dv), "flops": 7 * s * t * hv * dk * dv}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    st = _inputs(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attn": _exact_attn, "delta": _exact_delta}[case["kind"]](case, st)


def _exact_turn(case, x, pos):
    """x [n, h, d] as complex numbers times e^(i angle)."""
    r, o = case["rot"], _scaling(case)
    x = x.double()
    freq = []
    for i in range(r // 2):
        f = BASE ** (-2.0 * i / r)
        if case["scaling"] == "linear":
            f /= o["factor"]
        elif case["scaling"] == "by_parts":
            turns = o["orig_len"] * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - o["beta_slow"]) / (o["beta_fast"] - o["beta_slow"])))
            f *= keep + (1 - keep) / o["factor"]
        freq.append(f)
    angle = torch.outer(pos.double(), torch.tensor(freq, dtype=torch.float64, device=x.device))
    turn = torch.polar(torch.full_like(angle, o.get("attn_scale", 1.0)), angle)[:, None, :]
    half = case["pairs"] == "half"
    first, second = (x[..., :r // 2], x[..., r // 2:r]) if half else (x[..., 0:r:2], x[..., 1:r:2])
    z = torch.complex(first.contiguous(), second.contiguous()) * turn
    y = x.clone()
    if half:
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    else:
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    return y


def _exact_rope(case, st):
    return _exact_turn(case, st["x"].view(case["n"], case["h"], case["d"]), st["pos"]).view(case["n"], -1)


def _exact_append(case, st):
    s, m, hq, hkv, d = (case[x] for x in ("s", "m", "hq", "hkv", "d"))
    x = st["qkv"].view(s, m, hq + 2 * hkv, d)
    k, v, q = st["k"].double(), st["v"].double(), []
    for i in range(s):
        n = int(st["len"][i])
        y = _exact_turn(case, x[i, :, :hq + hkv], torch.arange(n, n + m, device="cuda"))
        q.append(y[:, :hq])
        k[i, n:n + m] = y[:, hq:]
        v[i, n:n + m] = x[i, :, hq + hkv:].double()
    return {"q": torch.cat(q).reshape(s * m, hq * d), "k": k, "v": v}


def _exact_attn(case, st):
    s, m, hq, hkv, d = (case[x] for x in ("s", "m", "hq", "hkv", "d"))
    out = torch.empty((s, m, hq, d), dtype=torch.float64, device="cuda")
    q = st["q"].double().view(s, m, hq, d)
    bits = st["mask"].cpu().tolist() if case["tree"] else None
    for h in range(hkv):
        of = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
        pk, pv = st["pk"][0, :, h].double(), st["pv"][0, :, h].double()
        for i in range(s):
            n = int(st["len"][i])
            k = torch.cat([pk, st["k"][i, :n + m, h].double()])
            v = torch.cat([pv, st["v"][i, :n + m, h].double()])
            new = torch.tensor([[bool(bits[i][r] >> j & 1) if bits else j <= r for j in range(m)] for r in range(m)], device="cuda")
            seen = torch.cat([torch.ones((m, case["p"] + n), dtype=torch.bool, device="cuda"), new], 1)
            z = q[i, :, of] @ k.T.contiguous() / math.sqrt(d)
            w = torch.softmax(z.masked_fill(~seen[:, None], -math.inf), -1)
            out[i, :, of] = w @ v
    return out.view(s * m, hq * d)


def _exact_delta(case, st):
    s, t, hk, hv, dk, dv = (case[x] for x in ("s", "t", "hk", "hv", "dk", "dv"))
    q, k, v, g, b = (st[x].double() for x in ("q", "k", "v", "g", "beta"))
    q = (q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) / math.sqrt(dk)).repeat_interleave(hv // hk, 2)
    k = (k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(hv // hk, 2)
    state = st["state"].double()
    o, kept = [], []
    for i in range(t):
        state = state * torch.exp(g[:, i])[..., None, None]
        miss = v[:, i] - (state * k[:, i, :, :, None]).sum(-2)
        state = state + k[:, i, :, :, None] * (b[:, i, :, None] * miss)[:, :, None, :]
        o.append((state * q[:, i, :, :, None]).sum(-2))
        if case["snap"]:
            kept.append(state)
    return {"o": torch.stack(o, 1), "state": torch.stack(kept, 1) if case["snap"] else state}
