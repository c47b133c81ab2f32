"""A decoder layer whose projections are quantised: norms, QKV, rotary rows into a paged cache, attention, feed-forward.

  x -> [norm] -> QKV -> kv_append -> attention -> O -> [norm + residual] -> gate+up -> SwiGLU -> down -> [norm + residual of the next layer]

The residual stream is fp32; a layer hands its last projection's output on to the next layer's norm, which adds it (alpha, a gate and a norm behind
the block are that norm's).  Q4 projections take and give fp32 rows, NVFP4 ones bf16 rows (quantised on the way in).  Everything
runs in libmpq and follows lengths that lie on the GPU: a step of fixed shape can be captured as a CUDA graph after one warm-up call.
"""
from __future__ import annotations

from . import _lib
from .decoder_ops import KvStep, _bad, kv_append, kv_plan, paged_attention, prompt_attention, residual_norm, rotary_frequencies
from .quant_linear import Context, QuantLinear, _torch, nvfp4_quantize


class PagedCache:
    """Pages of keys and values for several layers, and who has them: up to `requests` requests of up to max_blocks pages."""

    def __init__(self, ctx: Context, layers: int, pages: int, kv_heads: int, head_dim: int, requests: int, max_blocks: int, page_size: int = 16):
        torch = _torch()
        dev = f"cuda:{ctx.device}"
        self.ctx, self.page_size = ctx, page_size
        self.k = [torch.zeros((pages, kv_heads, page_size, head_dim), dtype=torch.bfloat16, device=dev) for _ in range(layers)]
        self.v = [torch.zeros_like(k) for k in self.k]
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.block_table = torch.zeros((requests, max_blocks), dtype=torch.int32, device=dev)
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=dev)

    def plan(self, new_lens, tokens: int) -> KvStep:
        """The next step: new_lens int32 [requests] on the GPU (negative: the request has ended), `tokens` rows of activations."""
        return kv_plan(self.ctx, new_lens, self.lens, self.block_table, self.free, self.free_count, page_size=self.page_size, tokens=tokens, inplace=True)


class DecoderLayer:
    """Projections qkv [(q_heads + 2 kv_heads) D][H], o [H][q_heads D], gate_up [2F][H], down [H][F], all Q4 or all NVFP4 (QuantLinear), and the
    weights of the norms in front of the two blocks (fp32 [H]); attn_post, ffn_post: of norms behind them.

    activation_scales (NVFP4 only): the tensor scales with which the rows in front of qkv, o, gate_up and down are quantised, 1 each if None.  A block of 16
    values keeps all that NVFP4 has to give where its largest magnitude is between 0.094 and 2688 times the scale.  Below that its own scale loses bits, at 0.0059 times
    and less the block becomes zeros; above, it saturates.  So what a model's attention averages, or its SwiGLU gives, to a few thousandths wants
    a scale of its own: the largest magnitude seen in calibration / 2688 leaves the most room below."""

    def __init__(self, qkv: QuantLinear, o: QuantLinear, gate_up: QuantLinear, down: QuantLinear, attn_norm, ffn_norm, *, q_heads: int, kv_heads: int,
                 frequencies=None, interleaved: bool = False, eps: float = 1e-6, alpha: float = 1.0, attn_post=None, ffn_post=None, activation_scales=None):
        self.qkv, self.o, self.gate_up, self.down = qkv, o, gate_up, down
        self.ctx, self.fmt = qkv.ctx, qkv.w.fmt
        if any(p.w.fmt != self.fmt for p in (o, gate_up, down)):
            _bad("the projections of a layer have one format")
        if activation_scales is not None and self.fmt == _lib.FMT_Q4:
            _bad("activation_scales are for NVFP4 projections")
        self.activation_scales = tuple(float(a) for a in (activation_scales if activation_scales is not None else (1.0,) * 4))
        if len(self.activation_scales) != 4 or not all(2.0 ** -126 <= a <= 2.0 ** 126 for a in self.activation_scales):
            _bad("activation_scales are four positive fp32 numbers: of the rows in front of qkv, o, gate_up and down")
        if q_heads <= 0 or kv_heads <= 0:
            _bad("q_heads and kv_heads must be positive", _lib.ERR_SHAPE)
        H, heads = qkv.w.K, q_heads + 2 * kv_heads
        if qkv.w.N % heads or o.w.K * heads != qkv.w.N * q_heads or o.w.N != H or gate_up.w.K != H or down.w.N != H or gate_up.w.N != 2 * down.w.K:
            _bad("the projections' shapes do not fit together", _lib.ERR_SHAPE)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, qkv.w.N // heads
        if self.head_dim not in (64, 128) or q_heads % kv_heads:
            _bad(f"the attention has heads of 64 or 128, query heads a multiple of kv_heads ({q_heads} and {kv_heads} heads of {self.head_dim})", _lib.ERR_SHAPE)
        self.attn_norm, self.ffn_norm, self.attn_post, self.ffn_post = attn_norm, ffn_norm, attn_post, ffn_post
        self.frequencies = rotary_frequencies(self.ctx, self.head_dim) if frequencies is None else frequencies
        self.interleaved, self.eps, self.alpha = interleaved, eps, alpha
        torch = _torch()
        self.dtype = torch.float32 if self.fmt == _lib.FMT_Q4 else torch.bfloat16      # of rows between the projections

    def _project(self, linear, x, scale):
        if self.fmt == _lib.FMT_Q4:
            return linear(x)
        codes, sf = nvfp4_quantize(self.ctx, x, scale)
        return linear((codes, sf, scale))

    def forward(self, residual, x, step: KvStep = None, cache: PagedCache = None, layer: int = 0, *, starts=None, positions=None, post=None, max_new: int = 0):
        """-> (residual, x) for the next layer, residual updated in place.

        residual fp32 [T][H]; x [T][H]: the last layer's output (the embedding, with a residual of zeros), which this layer's first norm adds, behind
        a norm with the weights `post` (the last layer's ffn_post) if given.  With `step` and `cache` the tokens attend to their
        requests' pages (max_new: the most new tokens of a request, 1 for a step of single tokens, 0 if not known; see paged_attention); else the T rows are whole prompts, packed at `starts` with their `positions`."""
        ctx, T, (qkv_scale, o_scale, gate_up_scale, down_scale) = self.ctx, residual.shape[0], self.activation_scales
        residual, y = residual_norm(ctx, x, residual, self.attn_norm, eps=self.eps, alpha=self.alpha, post_weight=post, out_dtype=self.dtype, inplace=True)
        qkv = self._project(self.qkv, y, qkv_scale)
        if step is not None:
            k, v = cache.k[layer], cache.v[layer]
            q, _, _ = kv_append(ctx, qkv, self.q_heads, self.kv_heads, positions=step.positions, frequencies=self.frequencies, interleaved=self.interleaved,
                                k_cache=k, v_cache=v, slots=step.slots)
            a = paged_attention(ctx, q, k, v, step.starts, step.lens, cache.block_table, max_new=max_new, out_dtype=self.dtype)
        else:
            q, k, v = kv_append(ctx, qkv, self.q_heads, self.kv_heads, positions=positions, frequencies=self.frequencies, interleaved=self.interleaved, rows=True)
            a = prompt_attention(ctx, q, k, v, starts, out_dtype=self.dtype)
        x = self._project(self.o, a.view(T, -1), o_scale)
        residual, y = residual_norm(ctx, x, residual, self.ffn_norm, eps=self.eps, alpha=self.alpha, post_weight=self.attn_post, out_dtype=self.dtype, inplace=True)
        gate_up = self._project(self.gate_up, y, gate_up_scale)
        if self.fmt == _lib.FMT_Q4:
            return residual, self.down.forward_swiglu(gate_up)
        codes, sf = nvfp4_quantize(ctx, gate_up, down_scale, swiglu_fused=True)
        return residual, self.down((codes, sf, down_scale))

    __call__ = forward
