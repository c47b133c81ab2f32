"""Decoder layers of NVFP4 projections, stage by stage: what a layer gives each of its projections, and what they give back, is recorded; every stage is
compared with its definition in 64 bits on what the stage in front of it really gave, its activations quantised by the CPU restatement of the format.

B is half a step of bf16 (2^-8), U of fp32 (2^-24), both relative."""
import math
from types import SimpleNamespace

import numpy as np
import pytest

B, U = 2.0 ** -8, 2.0 ** -24
STAGES = ("qkv", "o", "gate_up", "down")


def _t():
    import torch
    return torch


def _recorder(weight):
    """A QuantLinear that keeps (codes, scales, tensor scale, output) of its calls."""
    import makepad_b200 as m

    class Recorder(m.QuantLinear):
        def forward(self, x, out=None):
            y = super().forward(x, out)
            self.calls.append((*x, y))
            return y
        __call__ = forward
    r = Recorder(weight)
    r.calls = []
    return r


def _layers(ctx, count, H, q_heads, kv_heads, D, F, post, scales, sizes=(1.0, 1.0, 1.0, 1.0), interleaved=False):
    """Layers whose projections give rows of rms `sizes` for rows of rms 1."""
    import makepad_b200 as m
    from makepad_b200 import synth
    torch = _t()
    g = torch.Generator(device="cuda").manual_seed(7)
    norm = lambda: 1 + 0.1 * torch.randn(H, device="cuda", generator=g)

    def linear(n, k, seed, size):
        codes, sf = synth.nvfp4_tensor(n, k, seed=seed, stream=1)
        return _recorder(m.Nvfp4Weight(ctx, codes, sf, size * 3.2 / math.sqrt(k)))
    shapes = (((q_heads + 2 * kv_heads) * D, H), (H, q_heads * D), (2 * F, H), (H, F))
    made = []
    for i in range(count):
        made.append(m.DecoderLayer(*(linear(n, k, 10 * i + j, sizes[j]) for j, (n, k) in enumerate(shapes)), norm(), norm(), q_heads=q_heads, kv_heads=kv_heads, alpha=0.5,
                                   interleaved=interleaved, attn_post=norm() if post else None, ffn_post=norm() if post else None, activation_scales=scales))
    return made


def _run(ctx, layers, embed, starts, chunks, page):
    """The prompts at `starts`, whole (chunks None) or in chunks through the cache -> (rows of each call in the order of `embed`, last residual, last x)."""
    import makepad_b200 as m
    torch = _t()
    n, lens, l = len(starts) - 1, [b - a for a, b in zip(starts, starts[1:])], layers[0]
    for layer in layers:
        for s in STAGES:
            getattr(layer, s).calls.clear()
    residual, last, calls = torch.empty(embed.shape, device="cuda"), torch.empty_like(embed), []
    if chunks is None:
        r, x, post = torch.zeros(embed.shape, device="cuda"), embed, None
        positions = torch.cat([torch.arange(t) for t in lens]).int().cuda()
        for layer in layers:
            r, x = layer(r, x, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), positions=positions, post=post)
            post = layer.ffn_post
        return [torch.arange(len(embed), device="cuda")], r, x
    cache = m.PagedCache(ctx, len(layers), sum(-(-t // page) for t in lens), l.kv_heads, l.head_dim, n, -(-max(lens) // page), page)
    done, k = [0] * n, 0
    while done != lens:
        new = [min(chunks[min(k, len(chunks) - 1)] + i, t - d) for i, (t, d) in enumerate(zip(lens, done))]
        rows = torch.cat([torch.arange(a + d, a + d + c) for a, d, c in zip(starts, done, new)]).cuda()
        step = cache.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), rows.numel())
        assert step.missing.item() == 0
        r, x, post = torch.zeros(rows.numel(), embed.shape[1], device="cuda"), embed[rows], None
        for i, layer in enumerate(layers):
            r, x = layer(r, x, step, cache, i, post=post, max_new=max(new))
            post = layer.ffn_post
        residual[rows], last[rows] = r, x
        calls.append(rows)
        done, k = [d + c for d, c in zip(done, new)], k + 1
    return calls, residual, last


def _recorded(linear, calls, rows):
    """-> (quantised input as fp64 values, output as fp64, tensor scale) in the order of the rows."""
    from oracle import oracle
    torch = _t()
    assert len(linear.calls) == len(calls)
    x, y = torch.empty(rows, linear.w.K, dtype=torch.float64, device="cuda"), torch.empty(rows, linear.w.N, dtype=torch.float64, device="cuda")
    for at, (codes, sf, ts, out) in zip(calls, linear.calls):
        x[at] = torch.from_numpy(oracle.nvfp4_dequantize(codes.cpu().numpy(), sf.cpu().numpy(), ts)).cuda().double()
        y[at] = out.double()
    return x, y, linear.calls[0][2]


def _quantised(x, ts):
    """(values after quantisation, the blocks' scales per element) of fp32 rows, by the CPU restatement."""
    from oracle import oracle
    torch = _t()
    codes, sf = oracle.nvfp4_quantize(x.float().cpu().numpy(), ts)
    scale = oracle.e4m3_to_f32(sf).astype(np.float64) * np.float32(ts)
    return torch.from_numpy(oracle.nvfp4_dequantize(codes, sf, ts)).cuda().double(), torch.from_numpy(np.repeat(scale, 16, axis=1)).cuda()


def _rms(x, w, eps):
    return x / (x.square().mean(1, keepdim=True) + eps).sqrt() * w.double()


def _same_codes(got, x, ts, where):
    """The quantised rows are those of x, but for a few: fp32 is within 32 U of x, so that at most one bf16 in 2^10 rounds the other way, each of which can turn its own
    code, or with the block's largest one value in sixteen the block's scale, which turns up to sixteen: 2^-9 of the values at most (and five, for small arrays)."""
    want, _ = _quantised(x, ts)
    flips = int((got != want).sum())
    assert flips <= 5 + got.numel() * 2 ** -9, (where, flips, got.numel())


def _projected(y, x, w, where):
    """fp32 sums of K products, each addition cut to 2 u of the magnitudes; then bf16."""
    want, mass = x @ w.T, x.abs() @ w.abs().T
    assert bool(((y - want).abs() <= B * want.abs() + 4 * x.shape[1] * U * mass + 2.0 ** -126).all()), where


def _turned(x, positions, freq, interleaved):
    torch = _t()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] * freq)[:, None]
    half, y = x.shape[2] // 2, torch.empty_like(x)
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    z = torch.complex(a.contiguous(), b.contiguous()) * turn
    (y[..., 0::2] if interleaved else y[..., :half]).copy_(z.real)
    (y[..., 1::2] if interleaved else y[..., half:]).copy_(z.imag)
    return y


def _attention(l, qkv, starts):
    """(out, what the weights' rounding can move it by) of bf16 QKV rows, q and k rounded to bf16 behind their rotation."""
    torch = _t()
    rows = qkv.unflatten(1, (-1, l.head_dim))
    out = torch.zeros(rows.shape[0], l.q_heads, l.head_dim, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(out)
    for a, b in zip(starts, starts[1:]):
        qk = _turned(rows[a:b, :l.q_heads + l.kv_heads].contiguous(), torch.arange(b - a, device="cuda"), l.frequencies, l.interleaved).bfloat16().double()
        v, hidden = rows[a:b, l.q_heads + l.kv_heads:], torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").triu(1)
        for h in range(l.q_heads):
            kh = h // (l.q_heads // l.kv_heads)
            p = torch.softmax((qk[:, h] @ qk[:, l.q_heads + kh].T / math.sqrt(l.head_dim)).masked_fill(hidden, -math.inf), 1)
            out[a:b, h], mass[a:b, h] = p @ v[:, kh], p @ v[:, kh].abs()
    return out.flatten(1), mass.flatten(1)


def _check(layers, embed, starts, calls, residual, last):
    torch = _t()
    T = embed.shape[0]
    r, x, post = torch.zeros(embed.shape, dtype=torch.float64, device="cuda"), embed.double(), None
    for n, l in enumerate(layers):
        W = [getattr(l, s).w.dequantize().double() for s in STAGES]
        (ax, ay, at), (ox, oy, ot), (gx, gy, gt), (dx, dy, dt) = (_recorded(getattr(l, s), calls, T) for s in STAGES)
        assert (at, ot, gt, dt) == tuple(l.activation_scales)
        r = r + l.alpha * (x if post is None else _rms(x, post, l.eps))
        _same_codes(ax, _rms(r, l.attn_norm, l.eps).bfloat16(), at, (n, "qkv"))
        _projected(ay, ax, W[0], (n, "qkv"))
        # Attention is off by up to e = B of its weights' mass (their rounding, and 2^-12 for fp32) and B of itself.  A value e away from what is quantised here goes to the
        # neighbouring code, a step (at most two scales s) away, with the probability e / step: e * 2 s in the sum of squares.  Where the block's
        # largest moves its scale (probability 16 e / largest), sixteen values are rounded on another grid (step^2 / 6 each): as much again.
        out, mass = _attention(l, ay, starts)
        want, s = _quantised(out.bfloat16(), ot)
        e = (B + 2 ** -12) * mass + B * out.abs()
        # (values that are all 2^-10 steps of the smallest block scale or less have s = 0: a step is then that scale's)
        step = 2 * s.clamp(min=2.0 ** -9 * ot)
        assert float((ox - want).square().sum()) <= 2 * float((e * step).sum()), (n, "o", float((ox - want).norm() / want.norm()))
        _projected(oy, ox, W[1], (n, "o"))
        r = r + l.alpha * (oy if l.attn_post is None else _rms(oy, l.attn_post, l.eps))
        _same_codes(gx, _rms(r, l.ffn_norm, l.eps).bfloat16(), gt, (n, "gate_up"))
        _projected(gy, gx, W[2], (n, "gate_up"))
        F = gy.shape[1] // 2
        _same_codes(dx, (torch.nn.functional.silu(gy[:, :F]) * gy[:, F:]).float(), dt, (n, "down"))      # (fp32 within 4 units: far fewer)
        _projected(dy, dx, W[3], (n, "down"))
        x, post = dy, l.ffn_post
    assert torch.equal(last.double(), x)
    # (fp32 sums of four terms, each within 32 U)
    assert bool(((residual.double() - r).abs() <= 4 * 32 * U * (r.abs() + 8)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,post,interleaved,scales", [((8, 2, 64), False, False, None), ((4, 4, 128), True, True, (1.0, 0.25, 2.0 ** -5, 1 / 3)), ((4, 1, 64), True, False, (0.01,) * 4)])
def test_nvfp4_layers_stage_by_stage(ctx, heads, post, interleaved, scales):
    torch = _t()
    layers = _layers(ctx, 2, 256, *heads, 512, post, scales, interleaved=interleaved)
    starts = [0, 40, 41, 110]
    embed = torch.randn(110, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    for chunks in (None, [1000], [50, 7, 1], [1]):
        calls, residual, last = _run(ctx, layers, embed, starts, chunks, 16)
        _check(layers, embed, starts, calls, residual, last)
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))


@pytest.mark.gpu
def test_nvfp4_layers_of_small_activations(ctx):
    """Attention and SwiGLU that give a thousandth: with tensor scales of their own they keep what four bits can hold, with a scale of 1 whole blocks become zeros."""
    torch = _t()
    starts = [0, 300]
    embed = torch.randn(300, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).bfloat16()
    lost = {}
    for scales in ((1.0, 2.0 ** -16, 1.0, 2.0 ** -16), None):
        layers = _layers(ctx, 1, 256, 8, 2, 64, 512, True, scales, sizes=(2.0 ** -8, 1.0, 2.0 ** -5, 1.0))
        for chunks in (None, [100]):
            calls, residual, last = _run(ctx, layers, embed, starts, chunks, 32)
            _check(layers, embed, starts, calls, residual, last)
        l = layers[0]
        (ax, ay, _), (ox, _, ot), (gx, gy, _), (dx, _, dt) = (_recorded(getattr(l, s), calls, 300) for s in STAGES)
        out, mass = _attention(l, ay, starts)
        F = gy.shape[1] // 2
        for name, got, want, e in (("o", ox, out, 2 * B * mass + B * out.abs()), ("down", dx, torch.nn.functional.silu(gy[:, :F]) * gy[:, F:], 0.0)):
            top = want.abs().unflatten(1, (-1, 16)).amax(2).repeat_interleave(16, 1)
            assert 2.0 ** -12 < float(want.square().mean().sqrt()) < 2.0 ** -8, name
            # half of the largest step is the block's scale, a sixth of its largest value rounded to e4m3 (2^-4): 17/96
            lost[name, scales is None] = float(((got - want).abs() > top * 17 / 96 + e).double().mean())
    assert lost["o", False] == 0 and lost["down", False] == 0
    assert lost["o", True] > 0.1 and lost["down", True] > 0.1


def _shapes(fmt, q_heads=4, kv_heads=2, D=64, H=256, F=512):
    """Stands in for four projections where nothing is launched."""
    made = [SimpleNamespace(ctx=None, w=SimpleNamespace(fmt=fmt, N=n, K=k)) for n, k in (((q_heads + 2 * kv_heads) * D, H), (H, q_heads * D), (2 * F, H), (H, F))]
    return dict(zip(STAGES, made), attn_norm=None, ffn_norm=None, q_heads=q_heads, kv_heads=kv_heads, frequencies=())


def test_activation_scales_that_are_refused():
    import makepad_b200 as m
    assert m.DecoderLayer(**_shapes(m._lib.FMT_NVFP4)).activation_scales == (1.0,) * 4
    assert m.DecoderLayer(**_shapes(m._lib.FMT_NVFP4), activation_scales=[1, 2, 3, 0.5]).activation_scales == (1.0, 2.0, 3.0, 0.5)
    for bad in ((1.0,) * 3, (1.0,) * 5, (1.0, 0.0, 1.0, 1.0), (-1.0, 1.0, 1.0, 1.0), (1.0, 1.0, math.nan, 1.0), (1.0, 1.0, math.inf, 1.0), (1e-45, 1.0, 1.0, 1.0), (1.0, 1e39, 1.0, 1.0)):
        with pytest.raises(m.MpqError):
            m.DecoderLayer(**_shapes(m._lib.FMT_NVFP4), activation_scales=bad)
    with pytest.raises(m.MpqError):
        m.DecoderLayer(**_shapes(m._lib.FMT_Q4), activation_scales=(1.0,) * 4)
