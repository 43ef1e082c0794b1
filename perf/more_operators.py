"""Cases of the 8-bit projections, for timing and for comparing outputs.

A case is a dict of plain values whose "kind" says which operator it takes:

* norm  the residual's addition, the root-mean-square norm and its output as
        8-bit codes with a scale for each row: the input of a layer's
        projections;
* gate  silu(gate) * up of [gate | up] rows as 8-bit codes with scales: the
        input of the down projection;
* rows  rows as they are, as 8-bit codes with scales: the mixers' output
        before its projection, or a weight matrix whose rows are channels;
* gemm  the product of 8-bit rows with 8-bit weights, scales for each token
        and channel, fp32 out, or added to the residual.

Codes are returned as the values that they stand for.
Where `own` is false, run() computes them in plain torch operations.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6


def listed():
    return [
        # the next token of one conversation: the time is latency
        {"name": "norm_m1_k4096", "kind": "norm", "m": 1, "k": 4096, "add": True, "weight": True},
        # a verify step of 64 sequences (1 accepted + 4 drafted tokens), a small model's rows, nothing to add
        {"name": "norm_m320_k2048", "kind": "norm", "m": 320, "k": 2048, "add": False, "weight": True},
        # a prompt's rows
        {"name": "norm_m8190_k4096", "kind": "norm", "m": 8190, "k": 4096, "add": True, "weight": True},
        # a verify step of one sequence
        {"name": "gate_m5_k12288", "kind": "gate", "m": 5, "k": 12288},
        # a prompt of an odd length, a small model
        {"name": "gate_m4097_k6144", "kind": "gate", "m": 4097, "k": 6144},
        # the attention's output of 32 heads of 128 for a short prompt
        {"name": "rows_m515_k4096", "kind": "rows", "m": 515, "k": 4096},
        # a down projection's weights, dequantized, to codes with a scale a channel
        {"name": "rows_m4096_k12288", "kind": "rows", "m": 4096, "k": 12288},
        # the next token through [gate; up]: reading the weights is all there is
        {"name": "gemm_m1_24576x4096", "kind": "gemm", "m": 1, "n": 24576, "k": 4096, "accum": False},
        # a verify step through down, added to the residual
        {"name": "gemm_m5_4096x12288", "kind": "gemm", "m": 5, "n": 4096, "k": 12288, "accum": True},
        # a 64-node draft tree through a small model's [gate; up]
        {"name": "gemm_m64_12288x2048", "kind": "gemm", "m": 64, "n": 12288, "k": 2048, "accum": False},
        # a short prompt of an odd length through o, added to the residual
        {"name": "gemm_m515_4096x4096", "kind": "gemm", "m": 515, "n": 4096, "k": 4096, "accum": True},
        # the largest: a prompt through [gate; up]
        {"name": "gemm_m4096_24576x4096", "kind": "gemm", "m": 4096, "n": 24576, "k": 4096, "accum": False},
    ]


def _spread(rng, lo, hi, step=1):
    """A whole number in [lo, hi], spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + step)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    kind = rng.choice(["norm", "gate", "rows", "gemm", "gemm", "gemm"])
    if kind == "gemm":
        m, k = _spread(rng, 1, 4096), _spread(rng, 256, 12288, 32)
        n = _spread(rng, 100, min(25000, 400_000_000_000 // (m * k)))
        return {"kind": kind, "m": m, "n": n, "k": k, "accum": rng.random() < 0.5}
    k = _spread(rng, 256, 12288, 16)
    m = _spread(rng, 1, min(8192, 50_000_000 // k))
    if kind == "norm":
        return {"kind": kind, "m": m, "k": k, "add": rng.random() < 0.6, "weight": rng.random() < 0.8}
    return {"kind": kind, "m": m, "k": k}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 23)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rows(g, m, k):
    """Rows as a layer's activations are: channels of different sizes, a few of them much larger than the others."""
    size = torch.exp(0.5 * _randn(g, k))
    size[torch.randint(0, k, (max(1, k // 500),), generator=g, device="cuda")] *= 12.0
    return _randn(g, m, k) * size


def _codes(g, m, k):
    return (32.0 * _randn(g, m, k)).round_().clamp_(-127, 127).to(torch.int8)


def _inputs(case, seed):
    g = _gen(seed)
    m, k = case["m"], case["k"]
    if case["kind"] == "norm":
        return {"case": case, "x": _rows(g, m, k), "add": 0.3 * _randn(g, m, k) if case["add"] else None,
                "w": 1.0 + 0.2 * _randn(g, k) if case["weight"] else None}
    if case["kind"] == "gate":
        return {"case": case, "x": 2.0 * _randn(g, m, 2 * k)}
    if case["kind"] == "rows":
        return {"case": case, "x": _rows(g, m, k)}
    n = case["n"]
    return {"case": case, "q": _codes(g, m, k), "w": _codes(g, n, k),
            "qs": 0.02 * torch.rand(m, generator=g, device="cuda") + 0.01,
            "ws": 0.002 * torch.rand(n, generator=g, device="cuda") + 0.0002,
            "y": _randn(g, m, n) if case["accum"] else None}


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:  # the outputs and workspaces that a serving loop keeps
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inferno.jl_amd"))
        import inferno_hip as ih
        st["ih"] = ih
        m, k = case["m"], case["k"]
        if case["kind"] == "gemm":
            st["out"] = st["y"] if case["accum"] else torch.empty((m, case["n"]), device="cuda")
            st["space"] = torch.empty(ih.gemm_i8_ws_bytes(m, case["n"], k, case["accum"]), dtype=torch.uint8, device="cuda")
        else:
            st["out"] = torch.empty((m, k), dtype=torch.int8, device="cuda")
            st["scales"] = torch.empty(m, device="cuda")
    return st


def run(st):
    kind = st["case"]["kind"]
    if own:
        ih = st["ih"]
        if kind == "gemm":
            return ih.gemm_i8(st["q"], st["qs"], st["w"], st["ws"], accum=st["case"]["accum"], out=st["out"], ws=st["space"])
        if kind == "norm":
            q, s = ih.rmsnorm_i8(st["x"], st["w"], EPS, add=st["add"], out=st["out"], scales=st["scales"])
            return {"values": torch.mul(q, s[:, None]), "x": st["x"]} if st["case"]["add"] else {"values": torch.mul(q, s[:, None])}
        q, s = (ih.silu_mul_i8 if kind == "gate" else ih.quantize_i8)(st["x"], out=st["out"], scales=st["scales"])
        return {"values": torch.mul(q, s[:, None])}
    return {"norm": _plain_norm, "gate": _plain_gate, "rows": _plain_rows, "gemm": _plain_gemm}[kind](st)


# ---------------------------------------------------------------- plain forms

def _plain_values(t, factor=1.0):
    """Rows t times `factor` (one a row) as the values that their codes stand for, in 64 bits until the codes are there: a
    value half a step between two codes falls to either by the last bits of 32."""
    top = t.abs().amax(-1, keepdim=True)
    code = torch.round(t * 127.0 / torch.where(top > 0, top, torch.ones_like(top)))
    return code.float() * (top * factor / 127.0).float()


def _plain_norm(st):
    x = st["x"]
    if st["add"] is not None:
        x += st["add"]
    t = x.double()
    factor = 1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)
    values = _plain_values(t if st["w"] is None else t * st["w"].double(), factor)
    return {"values": values, "x": x} if st["add"] is not None else {"values": values}


def _plain_gate(st):
    k = st["case"]["k"]
    gate, up = st["x"][:, :k].double(), st["x"][:, k:].double()
    return {"values": _plain_values(gate / (1.0 + torch.exp(-gate)) * up)}


def _plain_rows(st):
    return {"values": _plain_values(st["x"].double())}


def _plain_gemm(st):
    y = (st["q"].float() @ st["w"].float().T) * st["qs"][:, None] * st["ws"]
    return y if st["y"] is None else st["y"].add_(y)


# ---------------------------------------------------------------- what a pass needs

def work(case):
    """Codes count one byte a value, as the operators hold them."""
    m, k = case["m"], case["k"]
    if case["kind"] == "norm":
        return {"bytes": m * k * (13 if case["add"] else 5) + 4 * m + (4 * k if case["weight"] else 0),
                "flops": m * k * (7 if case["add"] else 6)}
    if case["kind"] == "gate":
        return {"bytes": 9 * m * k + 4 * m, "flops": 8 * m * k}
    if case["kind"] == "rows":
        return {"bytes": 5 * m * k + 4 * m, "flops": 3 * m * k}
    n = case["n"]
    return {"bytes": m * k + n * k + m * n * (8 if case["accum"] else 4) + 4 * (m + n), "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    st = _inputs(case, seed)
    m, k = case["m"], case["k"]
    if case["kind"] == "gemm":
        out = torch.zeros((m, case["n"]), dtype=torch.float64, device="cuda") if st["y"] is None else st["y"].double()
        q = st["q"].double() * st["qs"].double()[:, None]
        for n in range(0, case["n"], 4096):
            w = (st["w"][n:n + 4096].double() * st["ws"][n:n + 4096].double()[:, None]).T.contiguous()
            out[:, n:n + 4096] += q @ w
        return out
    values = torch.empty((m, k), dtype=torch.float64, device="cuda")
    kept = torch.empty((m, k), dtype=torch.float64, device="cuda") if case["kind"] == "norm" and case["add"] else None
    for i in range(0, m, 1024):
        x = st["x"][i:i + 1024].double()
        if case["kind"] == "norm":
            if case["add"]:  # (the residual is held in 32 bits: the norm is that of the rounded sum)
                x = x + st["add"][i:i + 1024].double()
                kept[i:i + 1024] = x
                x = x.float().double()
            x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / k + EPS)
            if case["weight"]:
                x = x * st["w"].double()
        elif case["kind"] == "gate":
            x = torch.sigmoid(x[:, :k]) * x[:, :k] * x[:, k:]
        step = torch.linalg.vector_norm(x, math.inf, dim=-1, keepdim=True) / 127.0
        values[i:i + 1024] = torch.round(x / step) * step
    return {"values": values, "x": kept} if kept is not None else {"values": values}
