"""A verify step through one attention layer and one recurrent layer, as a serving loop runs it: quantized projections, rotary
positions into the KV cache, attention over a shared prefix, the gated delta rule with its snapshots, then the outcome
applied on the device (commit_state_, advance_len_), captured once and replayed with other tokens. Each replay is compared
with the definitions in 64 bits over the tokens that stand.

Tolerance: the projections are fp32-accurate (1e-5), so a key or value falls on the other side of a rounding to fp16 now and
then; were every one of them a whole step off (2^-10 of its size, twice half a step), the mixed rows would be off by about
that: 2^-10 in the 2-norm bounds it."""
import math

import numpy as np
import pytest

import _mixref as R
from _util import rel_l2

pytestmark = pytest.mark.gpu
H, HQ, HKV, D, S, M, P, CAP = 256, 4, 2, 64, 3, 5, 70, 64
HK, HV, DK, DV = 2, 4, 64, 32


@pytest.fixture(scope="module")
def ih():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import inferno_hip
    assert inferno_hip.quant_kernels_available(), inferno_hip._lib.last_error()
    return inferno_hip


def test_verify_steps(ih):
    import torch
    F, q8 = ih.formats, ih.formats.Q8_0
    st = ih.synth.stream_for
    n_qkv, n_mix = (HQ + 2 * HKV) * D, 2 * HK * DK + HV * DV + 2 * HV
    shapes = {"qkv": (n_qkv, H), "o": (H, HQ * D), "mix": (n_mix, H), "out": (H, HV * DV)}
    w, dense = {}, {}
    for name, (n, k) in shapes.items():
        w[name] = ih.quantized_kernels.synth_blocks(q8, st(7, name), n * k // F.BLOCK_ELEMS[q8])
        dense[name] = ih.dequant(q8, w[name], n * k).view(n, k).double().cpu().numpy()
    gen = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *a: torch.randn(a, generator=gen, device="cuda")  # noqa: E731
    pk, pv = (r(1, P, HKV, D).half() for _ in "kv")
    cache = ih.KVCache(*(torch.zeros(S, CAP, HKV, D, dtype=torch.float16, device="cuda") for _ in "kv"))
    prefix = ih.KVCache(pk, pv)
    rp = ih.RopeParams(D, D // 2, base=10000.0)
    x, h = r(S * M, H), torch.empty(S * M, H, device="cuda")
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    acc = torch.zeros(S, dtype=torch.int32, device="cuda")
    state, snap = torch.zeros(S, HV, DK, DV, device="cuda"), torch.empty(S, M, HV, DK, DV, device="cuda")
    ws1 = torch.empty(ih.attn_prefix_ws_bytes(HQ, M, cache, prefix), dtype=torch.uint8, device="cuda")
    ws2 = torch.empty(ih.gated_delta_rule_ws_bytes(S, M, HK, HV, DK, DV, True), dtype=torch.uint8, device="cuda")
    gain = 1.0 / 40  # (brings the synthetic weights' products to ordinary sizes)

    def step():
        h.copy_(x)
        qkv = ih.gemm_q_ex(q8, w["qkv"], h, n_qkv, H, act=ih.ACT_RMSNORM) * gain
        q = ih.rope_append(qkv, HQ, cache, lens, rp, pos0=P)
        a = ih.attn_prefix(q, HQ, cache, lens, prefix=prefix, ws=ws1)
        h.add_(ih.gemm_q(q8, w["o"], a, H, HQ * D), alpha=gain)
        p = (ih.gemm_q_ex(q8, w["mix"], h, n_mix, H, act=ih.ACT_RMSNORM) * gain).view(S, M, n_mix)
        k0, v0, g0 = HK * DK, 2 * HK * DK, 2 * HK * DK + HV * DV
        o = ih.gated_delta_rule(p[..., :k0].unflatten(-1, (HK, DK)), p[..., k0:v0].unflatten(-1, (HK, DK)),
                                p[..., v0:g0].unflatten(-1, (HV, DV)), -torch.nn.functional.softplus(p[..., g0:g0 + HV]),
                                torch.sigmoid(p[..., g0 + HV:]), state, snapshots=snap, l2norm=True, ws=ws2)
        h.add_(ih.gemm_q(q8, w["out"], o.view(S * M, HV * DV), H, HV * DV), alpha=gain)
        ih.commit_state_(state, snap, acc)
        ih.advance_len_(lens, acc)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        acc.fill_(-1)
        step()  # warm-up: no token stands
    torch.cuda.synchronize()
    assert int(lens.abs().sum()) == 0 and float(state.abs().max()) == 0.0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()

    def norm(v):
        return v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6)

    f16 = lambda v: v.astype(np.float32).astype(np.float16).astype(np.float64)  # noqa: E731
    th = R.theta(D // 2, 10000.0)

    def reference(rows, n_new):
        """h of the last n_new of a sequence's rows [t, H]."""
        t = len(rows)
        qkv = (norm(rows) @ dense["qkv"].T * gain).reshape(t, HQ + 2 * HKV, D)
        qk = R.rotate(qkv[:, : HQ + HKV], P + np.arange(t), th, False)
        a = R.attention(qk[None, :, :HQ], f16(qk[None, :, HQ:]), f16(qkv[None, :, HQ + HKV:]), pk[0].double().cpu().numpy(),
                        pv[0].double().cpu().numpy(), [0], D ** -0.5)[0].reshape(t, -1)
        hh = rows + a @ dense["o"].T * gain
        p = norm(hh) @ dense["mix"].T * gain
        k0, v0, g0 = HK * DK, 2 * HK * DK, 2 * HK * DK + HV * DV
        o = R.delta(p[None, :, :k0].reshape(1, t, HK, DK), p[None, :, k0:v0].reshape(1, t, HK, DK),
                    p[None, :, v0:g0].reshape(1, t, HV, DV), -np.logaddexp(0, p[None, :, g0:g0 + HV]),
                    1 / (1 + np.exp(-p[None, :, g0 + HV:])), None, l2norm=True)
        out = hh + o[0][0].numpy().reshape(t, -1) @ dense["out"].T * gain
        return out[t - n_new:], o[2][0].numpy()

    stand = [np.zeros((0, H)) for _ in range(S)]
    rng = np.random.default_rng(3)
    for i in range(6):
        n = rng.integers(-1, M, S).astype(np.int32)  # (-1: an invalid draft, nothing stands)
        x.copy_(r(S * M, H))
        acc.copy_(torch.from_numpy(n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, xs = h.double().cpu().numpy().reshape(S, M, H), x.double().cpu().numpy().reshape(S, M, H)
        for s in range(S):
            want, _ = reference(np.concatenate([stand[s], xs[s]]), M)
            assert math.isfinite(float(got[s].sum())) and rel_l2(got[s], want) <= 2.0 ** -10, (i, s, rel_l2(got[s], want))
            stand[s] = np.concatenate([stand[s], xs[s][: n[s] + 1]])
            if len(stand[s]):
                assert rel_l2(state[s].cpu().numpy(), reference(stand[s], 1)[1]) <= 2.0 ** -10, (i, s)
        assert lens.tolist() == [len(t) for t in stand]
        ih.attn_prefix(torch.randn(S * M, HQ * D, device="cuda"), HQ, cache, lens)  # eager work between the replays
