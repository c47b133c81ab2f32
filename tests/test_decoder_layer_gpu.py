"""Whole decoder layers: norms, projections, rotary rows into the paged cache, attention, feed-forward, as a program runs them, against the same chain in
64 bits on the exported weights."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B = 2.0 ** -8          # half a step of bf16


def _t():
    import torch
    return torch


def _linear(ctx, kind, n, k, seed):
    import makepad_b200 as m
    from makepad_b200 import synth
    if kind == "q4":
        codes, scales = synth.q4_weight(n, k, seed=seed)
        # values of rms 1 / sqrt(K): the configured scales are |N(0,1)| * 0.02, the codes' rms is 4.6
        factor = np.float16(1 / (0.02 * 4.6 * math.sqrt(k)))
        return m.QuantLinear(m.Q4Weight(ctx, codes, (scales.view(np.float16) * factor).view(np.uint16)))
    codes, sf = synth.nvfp4_tensor(n, k, seed=seed, stream=1)
    return m.QuantLinear(m.Nvfp4Weight(ctx, codes, sf, 3.2 / math.sqrt(k)))


def _layers(ctx, kind, count, H, q_heads, kv_heads, D, F, post):
    import makepad_b200 as m
    torch = _t()
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    norm = lambda: 1 + 0.1 * torch.randn(H, device="cuda", generator=g)
    made = []
    for i in range(count):
        made.append(m.DecoderLayer(_linear(ctx, kind, (q_heads + 2 * kv_heads) * D, H, 10 * i), _linear(ctx, kind, H, q_heads * D, 10 * i + 1), _linear(ctx, kind, 2 * F, H, 10 * i + 2),
                                   _linear(ctx, kind, H, F, 10 * i + 3), norm(), norm(), q_heads=q_heads, kv_heads=kv_heads, alpha=0.5, attn_post=norm() if post else None,
                                   ffn_post=norm() if post else None))
    return made, 1 + 0.1 * torch.randn(H, device="cuda", generator=g)


def _reference(layers, last, embed, starts):
    """The chain in 64 bits; q, k and v rounded to bf16, as the cache holds them."""
    torch = _t()
    rms = lambda x, w, eps: x / (x.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
    r, x, post = torch.zeros_like(embed).double(), embed.double(), None
    for n, l in enumerate(layers):
        W = [p.w.dequantize().double() for p in (l.qkv, l.o, l.gate_up, l.down)]
        r = r + l.alpha * (x if post is None else rms(x, post, l.eps))
        qkv = (rms(r, l.attn_norm, l.eps) @ W[0].T).unflatten(1, (-1, l.head_dim))
        out = torch.zeros(r.shape[0], l.q_heads, l.head_dim, dtype=torch.float64, device="cuda")
        for a, b in zip(starts, starts[1:]):
            pos = torch.arange(b - a, device="cuda", dtype=torch.float64)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos[:, None] * l.frequencies)[:, None]
            half = l.head_dim // 2
            qk = qkv[a:b, :l.q_heads + l.kv_heads]
            z = torch.complex(qk[..., :half].contiguous(), qk[..., half:].contiguous()) * turn
            qk = torch.cat([z.real, z.imag], -1).bfloat16().double()
            v = qkv[a:b, l.q_heads + l.kv_heads:].bfloat16().double()
            hidden = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").triu(1)
            for h in range(l.q_heads):
                kh = h // (l.q_heads // l.kv_heads)
                s = (qk[:, h] @ qk[:, l.q_heads + kh].T / math.sqrt(l.head_dim)).masked_fill(hidden, -math.inf)
                out[a:b, h] = torch.softmax(s, 1) @ v[:, kh]
        x = out.flatten(1) @ W[1].T
        r = r + l.alpha * (x if l.attn_post is None else rms(x, l.attn_post, l.eps))
        gu = rms(r, l.ffn_norm, l.eps) @ W[2].T
        F = gu.shape[1] // 2
        x, post = (torch.nn.functional.silu(gu[:, :F]) * gu[:, F:]) @ W[3].T, l.ffn_post
    l = layers[-1]
    r = r + l.alpha * (x if post is None else rms(x, post, l.eps))
    return rms(r, last, l.eps)


def _finish(ctx, layers, last, r, x):
    import makepad_b200 as m
    l = layers[-1]
    return m.residual_norm(ctx, x, r, last, eps=l.eps, alpha=l.alpha, post_weight=l.ffn_post, out_dtype=_t().float32)[1]


def _prompts(ctx, layers, last, embed, starts):
    torch = _t()
    r, x, post = torch.zeros_like(embed), embed, None
    if layers[0].dtype is not torch.float32:
        x = embed.to(layers[0].dtype)
    at = torch.tensor(starts, dtype=torch.int32, device="cuda")
    positions = torch.cat([torch.arange(b - a) for a, b in zip(starts, starts[1:])]).int().cuda()
    for l in layers:
        r, x = l(r, x, starts=at, positions=positions, post=post)
        post = l.ffn_post
    return _finish(ctx, layers, last, r, x)


def _steps(ctx, layers, last, embed, starts, chunks, page_size):
    """The same prompts, each in chunks (then single tokens) through the paged cache -> rows in the order of `embed`."""
    import makepad_b200 as m
    torch = _t()
    n, lens = len(starts) - 1, [b - a for a, b in zip(starts, starts[1:])]
    l = layers[0]
    cache = m.PagedCache(ctx, len(layers), sum(-(-t // page_size) for t in lens), l.kv_heads, l.head_dim, n, -(-max(lens) // page_size), page_size)
    done, result, k = [0] * n, torch.empty_like(embed), 0
    while done != lens:
        new = [min(chunks[min(k, len(chunks) - 1)] + i, t - d) for i, (t, d) in enumerate(zip(lens, done))]
        rows = torch.cat([torch.arange(a + d, a + d + c) for a, d, c in zip(starts, done, new)]).cuda()
        step = cache.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), rows.numel())
        assert step.missing.item() == 0
        r, x, post = torch.zeros(rows.numel(), embed.shape[1], device="cuda"), embed[rows].to(l.dtype), None
        for i, layer in enumerate(layers):
            r, x = layer(r, x, step, cache, i, post=post, max_new=max(new))
            post = layer.ffn_post
        result[rows] = _finish(ctx, layers, last, r, x)
        done = [d + c for d, c in zip(done, new)]
        k += 1
    assert cache.free_count.item() == 0
    step = cache.plan(torch.full((n,), -1, dtype=torch.int32, device="cuda"), 0)
    assert sorted(cache.free.tolist()) == list(range(cache.free.numel())) and step.free_count.item() == cache.free.numel() and step.lens.tolist() == [0] * n
    return result


def _far(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("heads,post,page", [((4, 4, 64), False, 16), ((8, 2, 128), True, 64)])
def test_q4_layers_against_64_bits(ctx, heads, post, page):
    torch = _t()
    q_heads, kv_heads, D = heads
    layers, last = _layers(ctx, "q4", 2, 256, q_heads, kv_heads, D, 512, post)
    starts = [0, 40, 41, 170]
    embed = torch.randn(170, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    want = _reference(layers, last, embed, starts)
    # per layer the attention's weights are rounded to bf16 (B), and fp32 noise in front of the roundings of q, k and v moves a few of those by a step
    # (2 B each, on few elements: taken as B in the 2-norm); the blocks and norms behind pass a relative error on as it is, the residual sum
    # weakens it.  Two layers: 4 B, and as much again for the softmax, whose weights a relative error of the scores moves.
    tol = 8 * B
    whole = _prompts(ctx, layers, last, embed, starts)
    assert _far(whole, want) <= tol, _far(whole, want)
    for chunks in ([1000], [50, 7, 1], [1]):
        got = _steps(ctx, layers, last, embed, starts, chunks, page)
        assert _far(got, want) <= tol, (chunks, _far(got, want))
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))


def test_nvfp4_layers_through_cache_and_whole(ctx):
    """Four-bit activations turn an error of a bf16 step into another code now and then: a share of about 4 B of the codes by up to half of their value, which
    is 4 % of a row per quantisation in the 2-norm; eight of them in two layers, independent: 12 %, and twice that as the limit."""
    torch = _t()
    layers, last = _layers(ctx, "nvfp4", 2, 256, 8, 2, 64, 512, False)
    starts = [0, 100, 133]
    embed = torch.randn(133, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    whole = _prompts(ctx, layers, last, embed, starts)
    got = _steps(ctx, layers, last, embed, starts, [1000], 16)
    assert bool(torch.isfinite(whole).all()) and bool(torch.isfinite(got).all())
    assert _far(got, whole) <= 0.25, _far(got, whole)


def test_a_captured_decode_step(ctx):
    """A step of one token each, captured once and replayed while lengths, tables and cache grow, gives the bits of eager steps."""
    import makepad_b200 as m
    torch = _t()
    layers, last = _layers(ctx, "q4", 2, 256, 4, 2, 64, 512, False)
    n, T = 3, 3
    gen = torch.Generator(device="cuda").manual_seed(5)
    rows = torch.randn(20, T, 256, device="cuda", generator=gen)

    def make():
        return dict(cache=m.PagedCache(ctx, 2, 12, 2, 64, n, 4, 16), new=torch.ones(n, dtype=torch.int32, device="cuda"), x=torch.zeros(T, 256, device="cuda"))

    def step(s):
        plan = s["cache"].plan(s["new"], T)
        r, x = torch.zeros(T, 256, device="cuda"), s["x"]
        for i, l in enumerate(layers):
            r, x = l(r, x, plan, s["cache"], i, max_new=1)
        return _finish(ctx, layers, last, r, x)

    eager, graphed = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(make())                                     # (a warm-up: it reserves scratch)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(graphed)
    for i in range(20):
        graphed["x"].copy_(rows[i])
        eager["x"].copy_(rows[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(eager)), i
    assert torch.equal(graphed["cache"].lens, eager["cache"].lens) and graphed["cache"].lens.tolist() == [20] * n


@pytest.mark.parametrize("kind", ["q4", "nvfp4"])
@pytest.mark.parametrize("room", [12, 40, 150])
def test_rows_behind_the_last_token_touch_nothing(ctx, kind, room):
    """A step with room for more rows than it has tokens: whatever the others hold, the tokens' rows and the cache are the same."""
    import makepad_b200 as m
    torch = _t()
    layers, last = _layers(ctx, kind, 2, 256, 8, 2, 64, 512, True)
    new = torch.tensor([3, 0, 5, 1], dtype=torch.int32, device="cuda")
    rows = torch.randn(room, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    got = []
    for dead in (0.0, math.nan, 3e38):
        x = rows.clone()
        x[9:] = dead
        cache = m.PagedCache(ctx, 2, 8, 2, 64, 4, 2, 16)
        step = cache.plan(new, room)
        r = torch.zeros(room, 256, device="cuda")
        r[9:] = dead
        spoilt = [torch.full((room, w), math.nan, dtype=t, device="cuda") for w in (256, 512, 768, 1024) for t in (torch.float32, torch.bfloat16)]
        del spoilt                                       # (what is allocated next lies there)
        x, post = x.to(layers[0].dtype), None
        for i, l in enumerate(layers):
            r, x = l(r, x, step, cache, i, post=post)
            post = l.ffn_post
        got.append((_finish(ctx, layers, last, r, x)[:9], *cache.k, *cache.v))
    assert bool(torch.isfinite(got[0][0]).all())
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))


def test_layers_refuse_what_does_not_fit(ctx):
    import makepad_b200 as m
    torch = _t()
    w = torch.ones(256, device="cuda")
    q = lambda n, k, kind="q4": _linear(ctx, kind, n, k, 1)
    ok = dict(qkv=q(8 * 64, 256), o=q(256, 4 * 64), gate_up=q(1024, 256), down=q(256, 512))
    m.DecoderLayer(**ok, attn_norm=w, ffn_norm=w, q_heads=4, kv_heads=2)
    for bad in (dict(o=q(256, 192)), dict(o=q(192, 256)), dict(gate_up=q(1024, 192)), dict(down=q(256, 256)), dict(down=q(192, 512)), dict(down=q(256, 512, "nvfp4"))):
        with pytest.raises(m.MpqError):
            m.DecoderLayer(**{**ok, **bad}, attn_norm=w, ffn_norm=w, q_heads=4, kv_heads=2)
    with pytest.raises(m.MpqError):
        m.DecoderLayer(**ok, attn_norm=w, ffn_norm=w, q_heads=5, kv_heads=2)
