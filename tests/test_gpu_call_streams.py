"""Calls with stream= and without workspace or output, while the current stream allocates, writes and still reads."""
import pytest

import _mixref as R
from test_gpu_attn_prefix import Case
from test_gpu_delta import check, ih, make  # noqa: F401  (ih: the fixture)

pytestmark = pytest.mark.gpu
WAIT = 20_000_000  # clocks (some 10 ms): work that is still to come when a call returns


def crowd(like, n=6):
    """Allocations on the current stream of the sizes that a call made, written at once."""
    import torch
    return [torch.full(shape, 255, dtype=torch.uint8, device="cuda") for shape in like for _ in range(n)]


@pytest.mark.parametrize("handle", [False, True])
def test_attention_beside_the_current_stream(ih, handle):  # noqa: F811
    import torch
    c = Case(3, 5, 8, 2, 128, 700, [40, 3, 99], seed=5)
    cache, prefix = ih.KVCache(c.k, c.v), ih.KVCache(c.pk, c.pv)
    ln, _ = c.tensors()
    nb = ih.attn_prefix_ws_bytes(8, 5, cache, prefix)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        # memory of an output's and a workspace's size that the current stream frees while it still reads it
        old = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in (nb, 15 * 8 * 128 * 4)]
        torch.cuda._sleep(WAIT)
        kept = [t.clone() for t in old]
        del old
        with torch.cuda.stream(s):
            torch.cuda._sleep(WAIT // 4)
        out = ih.attn_prefix(c.q, 8, cache, ln, prefix=prefix, stream=s.cuda_stream if handle else s)
        others = crowd([(nb,), (15 * 8 * 128 * 4,)])
        torch.cuda.current_stream().wait_stream(s)
        c.check(out)
        assert all(bool((t == 7).all()) for t in kept) and all(bool((t == 255).all()) for t in others)
        del out, others, kept


def test_delta_beside_the_current_stream(ih):  # noqa: F811
    import torch
    q, k, v, g, b, st = make(2, 150, 2, 4, 64, 64, seed=5)
    o, _, last = R.delta(q, k, v, g, b, st)
    nb = ih.gated_delta_rule_ws_bytes(2, 150, 2, 4, 64, 64)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        new = torch.empty_like(st)
        with torch.cuda.stream(s):
            torch.cuda._sleep(WAIT)
        out = ih.gated_delta_rule(q, k, v, g, b, st, new_state=new, stream=s)
        others = crowd([(nb,), (out.numel() * 4,)])
        torch.cuda.current_stream().wait_stream(s)
        check(out, o, "o")
        check(new, last, "state")
        assert all(bool((t == 255).all()) for t in others)
        del out, others


def test_the_default_stream_from_another(ih):  # noqa: F811
    """stream=0 while another is current; the output, dropped while the current one still reads it, is not written again."""
    import torch
    q, k, v, g, b, st = make(2, 70, 2, 4, 64, 64, seed=9)
    want = ih.gated_delta_rule(q, k, v, g, b, st)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(4):
            out = ih.gated_delta_rule(q, k, v, g, b, st, stream=0)
            s.wait_stream(torch.cuda.default_stream())
            torch.cuda._sleep(WAIT)
            read = out.clone()
            del out
            ih.gated_delta_rule(k, q, v, g, b, st, stream=0)
            s.synchronize()
            assert torch.equal(read, want)
    torch.cuda.synchronize()


def test_accept_and_matmul_beside_the_current_stream(ih):  # noqa: F811
    """The other wrappers: a matmul and an accept step, and a count that is waited for on its own stream."""
    import torch
    F = ih.formats
    n, k = 512, 1024
    w = ih.quantized_kernels.synth_blocks(F.Q4_K, 11, n * k // F.BLOCK_ELEMS[F.Q4_K])
    x = torch.randn(5, k, device="cuda")
    logits = torch.randn(3, 5, 9000, device="cuda")
    tok = logits.argmax(-1).int()[:, :4].contiguous()
    tok[1, 2] = 5
    want, (count, am) = ih.gemm_q(F.Q4_K, w, x, n, k), ih.greedy_verify(logits, tok)
    assert count.tolist()[0] == 4 and count.tolist()[1] <= 2
    nb = ih.quantized_kernels.gemm_ws_bytes(F.Q4_K, 5, n, k)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(s):
            torch.cuda._sleep(WAIT)
        y = ih.gemm_q(F.Q4_K, w, x, n, k, stream=s)
        c, a = ih.greedy_verify(logits, tok, stream=s)
        others = crowd([(nb,), (5 * n * 4,), (12,), (60,)])
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, want) and torch.equal(c, count) and torch.equal(a, am)
        assert all(bool((t == 255).all()) for t in others)
        with torch.cuda.stream(s):
            torch.cuda._sleep(WAIT)
        assert ih.mtp_verify_step(logits, tok, stream=s)[0] == 4
        del y, c, a, others
