"""Contexts beside captures."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
def test_a_context_made_while_a_stream_captures(mode):
    """Making a context records nothing and does not end the capture; its first attention call may be part of it."""
    import makepad_b200 as m
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(500, h, 64, device="cuda", generator=gen).bfloat16() for h in (4, 2, 2))
    starts = torch.tensor([0, 200, 500], dtype=torch.int32, device="cuda")
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(), capture_error_mode=mode):
        x.add_(1)
        ctx = m.Context(0)
        got = m.prompt_attention(ctx, q, k, v, starts)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [2.0] * 4
    for a, b in ((0, 200), (200, 500)):
        s = torch.einsum("qhd,khd->hqk", q[a:b].double(), k[a:b].double().repeat_interleave(2, 1)) / 8
        s.masked_fill_(torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
        p, wide = torch.softmax(s, 2), v[a:b].double().repeat_interleave(2, 1)
        want, mass = torch.einsum("hqk,khd->qhd", p, wide), torch.einsum("hqk,khd->qhd", p, wide.abs())
        # weights and output rounded to bf16 (2^-8 each, of the magnitudes and of the value); fp32 sums of 64 products and 300 keys below 2^-12
        assert bool(((got[a:b].double() - want).abs() <= mass * (2 ** -8 + 2 ** -12) + want.abs() * 2 ** -8).all())
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))
    del graph
    ctx.close()
