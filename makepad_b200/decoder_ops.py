"""What runs between a decoder layer's projections, on top of the C ABI: norms, the paged cache, attention.

Tensors are torch CUDA tensors on the context's device; every call enqueues on that device's current stream.  Packed rows: the
new tokens of request i are rows starts[i] .. starts[i + 1] - 1, and rows behind starts[n] are left as they are.  There is no
gradient: outputs do not require one, whatever the inputs say.
"""
from __future__ import annotations

from typing import NamedTuple

from . import _lib
from .quant_linear import Context, MpqError, _raw, _stream, _torch


class KvStep(NamedTuple):
    """A step's plan: what kv_append and the attention read."""
    starts: object        # int32 [n + 1]
    lens: object          # int32 [n]: tokens in the cache, the step's own with them
    positions: object     # int32 [tokens]
    slots: object         # int64 [tokens], -1 behind the last token
    free_count: object    # int32 [1]
    missing: object       # int32 [1]: 0, or why nothing grew


def _bad(text: str, status: int = _lib.ERR_INVALID_ARG):
    raise MpqError(status, text)


def _need(ctx: Context, name: str, t, dtype, shape=None):
    """The address of a contiguous tensor of that type (and shape) on the context's device."""
    if t.dtype is dtype and t.get_device() == ctx.device and t.is_contiguous() and (shape is None or t.shape == shape):
        return t.data_ptr()
    if t.dtype is dtype and t.get_device() == ctx.device and t.is_contiguous():
        _bad(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}", _lib.ERR_SHAPE)
    _bad(f"{name} must be a contiguous {dtype} tensor on cuda:{ctx.device}")


def rotary_frequencies(ctx: Context, rot_dim: int, base: float = 10000.0):
    """base^(-2i / rot_dim) for i < rot_dim / 2, fp64: the angle of pair i is its position times this."""
    torch = _torch()
    return base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=f"cuda:{ctx.device}") / rot_dim)


def residual_norm(ctx: Context, x, residual=None, weight=None, *, eps: float = 1e-6, alpha: float = 1.0, post_weight=None, gate=None,
                  out_dtype=None, inplace: bool = False, norm: bool = True):
    """-> (residual', y): residual' = residual + alpha * gate * t with t = x, or its RMS norm times post_weight; y = the RMS norm of
    residual' times weight.

    x fp32 or bf16 [M][H]; residual fp32 [M][H] or None (zeros); gate fp32 [H] or [M][H]; weights fp32 [H].  y has out_dtype (fp32 or
    bf16; x's if None), and is None with norm=False.  inplace: residual itself is updated."""
    torch = _torch()
    if x.dim() != 2 or x.dtype not in (torch.float32, torch.bfloat16):
        _bad("x must be fp32 or bf16 [M][H]")
    M, H = x.shape
    out_dtype = out_dtype or x.dtype
    if out_dtype not in (torch.float32, torch.bfloat16):
        _bad("out_dtype must be fp32 or bf16")
    if inplace and residual is None:
        _bad("inplace needs a residual")
    f32 = torch.float32
    xp = _need(ctx, "x", x, x.dtype)
    rp = None if residual is None else _need(ctx, "residual", residual, f32, (M, H))
    wp = None if weight is None else _need(ctx, "weight", weight, f32, (H,))
    pp = None if post_weight is None else _need(ctx, "post_weight", post_weight, f32, (H,))
    gp = None if gate is None else _need(ctx, "gate", gate, f32, (H,) if gate.dim() == 1 else (M, H))
    stride = H if gate is not None and gate.dim() == 2 else 0
    r = residual if inplace else x.new_empty(M, H, dtype=f32)
    y = x.new_empty(M, H, dtype=out_dtype) if norm else None
    ctx.check(ctx.lib.mpq_residual_norm(_raw(ctx.h), xp, x.dtype is torch.bfloat16, M, H, rp, r.data_ptr(), pp, gp, stride, alpha, wp, eps,
                                        None if y is None else y.data_ptr(), out_dtype is torch.bfloat16, _stream(ctx)))
    return r, y


def kv_plan(ctx: Context, new_lens, lens, block_table, free, free_count, *, page_size: int, tokens: int, inplace: bool = False) -> KvStep:
    """The step of n requests, from their lengths on the device: pages of those that ended go back on the stack `free`, pages for the new
    tokens are taken from it into `block_table` (both updated in place); see mpq_kv_plan.

    new_lens, lens int32 [n]; block_table int32 [n][max_blocks]; free int32 [pages] with free_count int32 [1]; tokens: rows that the
    step has room for.  inplace: lens and free_count are updated themselves."""
    torch = _torch()
    i32, n = torch.int32, lens.shape[0]
    if block_table.dim() != 2:
        _bad("block_table must be [n][max_blocks]", _lib.ERR_SHAPE)
    blocks = block_table.shape[1]
    np_, lp = _need(ctx, "new_lens", new_lens, i32, (n,)), _need(ctx, "lens", lens, i32, (n,))
    tp, fp, cp = _need(ctx, "block_table", block_table, i32, (n, blocks)), _need(ctx, "free", free, i32), _need(ctx, "free_count", free_count, i32, (1,))
    if tokens < 0:
        _bad("tokens must not be negative", _lib.ERR_SHAPE)
    # one allocation for all outputs, cut without bookkeeping of views (an allocation each is 7 of a call's 18 us)
    slots, positions, starts, missing, lens_out, count_out = lens.new_empty(3 * tokens + 2 * n + 3).unsafe_split_with_sizes([2 * tokens, tokens, n + 1, 1, n, 1])
    slots = slots.view(torch.int64)
    if inplace:
        lens_out, count_out = lens, free_count
    ctx.check(ctx.lib.mpq_kv_plan(_raw(ctx.h), n, np_, lp, lens_out.data_ptr(), tp, blocks, fp, free.numel(), cp, count_out.data_ptr(), page_size, tokens,
                                  starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), missing.data_ptr(), _stream(ctx)))
    return KvStep(starts, lens_out, positions, slots, count_out, missing)


def _cache(ctx: Context, k_cache, v_cache):
    """(addresses, pages, kv heads, page size, head dim) of a cache."""
    bf16 = _torch().bfloat16
    if k_cache.dim() != 4:
        _bad("a cache is [pages][kv_heads][page_size][head_dim]", _lib.ERR_SHAPE)
    shape = k_cache.shape
    return (_need(ctx, "k_cache", k_cache, bf16), _need(ctx, "v_cache", v_cache, bf16, shape), *shape)


def kv_append(ctx: Context, qkv, q_heads: int, kv_heads: int, *, positions=None, frequencies=None, interleaved: bool = False, k_cache=None, v_cache=None,
              slots=None, rows: bool = False):
    """Rows of a QKV projection -> (q, k, v) bf16: rotary positions on q and k, q [T][q_heads][D] out, k and v into the cache at `slots`, and
    as rows [T][kv_heads][D] with rows=True (else None).

    qkv fp32 or bf16 [T][(q_heads + 2 kv_heads) * D]; positions int32 [T] and frequencies fp64 [rot_dim / 2] (None: no rotation); slots
    int64 [T] with k_cache and v_cache (None: no cache)."""
    torch = _torch()
    if qkv.dim() != 2 or qkv.dtype not in (torch.float32, torch.bfloat16) or qkv.get_device() != ctx.device or qkv.stride(1) != 1:
        _bad(f"qkv must be fp32 or bf16 rows on cuda:{ctx.device}")
    T, wide = qkv.shape
    if q_heads <= 0 or kv_heads <= 0 or wide % (q_heads + 2 * kv_heads):
        _bad(f"{wide} columns do not hold {q_heads} + 2 x {kv_heads} heads", _lib.ERR_SHAPE)
    D = wide // (q_heads + 2 * kv_heads)
    fp = pp = sp = kp = vp = None
    rot = pages = size = 0
    if frequencies is not None:
        if positions is None:
            _bad("frequencies need positions")
        rot = 2 * frequencies.numel()
        fp, pp = _need(ctx, "frequencies", frequencies, torch.float64), _need(ctx, "positions", positions, torch.int32, (T,))
    if slots is not None:
        if k_cache is None or v_cache is None:
            _bad("slots need a cache")
        sp = _need(ctx, "slots", slots, torch.int64, (T,))
        kp, vp, pages, heads, size, dim = _cache(ctx, k_cache, v_cache)
        if heads != kv_heads or dim != D:
            _bad(f"the cache has {heads} heads of {dim}, the rows {kv_heads} of {D}", _lib.ERR_SHAPE)
    bf16 = torch.bfloat16
    q = qkv.new_empty(T, q_heads, D, dtype=bf16)
    k, v = (qkv.new_empty(T, kv_heads, D, dtype=bf16), qkv.new_empty(T, kv_heads, D, dtype=bf16)) if rows else (None, None)
    ctx.check(ctx.lib.mpq_kv_append(_raw(ctx.h), qkv.data_ptr(), qkv.dtype is bf16, qkv.stride(0) if T > 1 else wide, T, q_heads, kv_heads, D, pp, fp, rot, interleaved,
                                    q.data_ptr(), None if k is None else k.data_ptr(), None if v is None else v.data_ptr(), sp, kp, vp, pages, size, _stream(ctx)))
    return q, k, v


def _head_rows(ctx: Context, name: str, t):
    """Address and row stride of bf16 [T][heads][D] whose heads lie beside each other (rows may be further apart)."""
    if t.dim() != 3 or t.dtype is not _torch().bfloat16 or t.get_device() != ctx.device:
        _bad(f"{name} must be bf16 [tokens][heads][head_dim] on cuda:{ctx.device}")
    T, heads, D = t.shape
    stride = t.stride()
    if (D > 1 and stride[2] != 1) or (heads > 1 and stride[1] != D):
        _bad(f"the heads of {name} must lie beside each other")
    return t.data_ptr(), stride[0] if T > 1 else heads * D


def _out(ctx, q, out_dtype, out):
    torch = _torch()
    if out is not None:
        if out.dtype not in (torch.float32, torch.bfloat16) or (out_dtype or out.dtype) is not out.dtype:
            _bad("out must be fp32 or bf16, and of out_dtype")
        _need(ctx, "out", out, out.dtype, q.shape)
        return out
    dtype = out_dtype or torch.bfloat16
    if dtype not in (torch.float32, torch.bfloat16):
        _bad("out_dtype must be fp32 or bf16")
    return torch.empty_like(q, dtype=dtype, memory_format=torch.contiguous_format)


def paged_attention(ctx: Context, q, k_cache, v_cache, starts, lens, block_table, *, scale: float = None, max_new: int = 0, out_dtype=None, out=None):
    """Attention of the new tokens q bf16 [T][q_heads][D] (D 64 or 128) over their requests' pages -> [T][q_heads][D], bf16 or fp32.

    starts int32 [n + 1], lens int32 [n] (with the new tokens, whose k and v are in the cache), block_table int32 [n][max_blocks]; scale:
    D^-1/2 if None; max_new: the most new tokens of a request, 0 if not known.  It chooses the kernel: 1 for a step of single tokens (left out, such a step
    takes a third longer), max(new) or 0 where requests have more (said too small, every 8 or 16 rows read the cache again: up to 15 times the time).  k and v of new
    tokens must be finite, also for the rows that do not see them; what lies behind lens[i] may be anything.  out must not overlap an input."""
    torch = _torch()
    qp, stride = _head_rows(ctx, "q", q)
    T, heads, D = q.shape
    kp, vp, pages, kv_heads, size, dim = _cache(ctx, k_cache, v_cache)
    if dim != D:
        _bad(f"the cache has heads of {dim}, q of {D}", _lib.ERR_SHAPE)
    n = lens.shape[0]
    if block_table.dim() != 2:
        _bad("block_table must be [n][max_blocks]", _lib.ERR_SHAPE)
    i32, blocks = torch.int32, block_table.shape[1]
    sp, lp, tp = _need(ctx, "starts", starts, i32, (n + 1,)), _need(ctx, "lens", lens, i32, (n,)), _need(ctx, "block_table", block_table, i32, (n, blocks))
    out = _out(ctx, q, out_dtype, out)
    ctx.check(ctx.lib.mpq_paged_attention(_raw(ctx.h), qp, stride, T, heads, kp, vp, pages, size, kv_heads, D, n, sp, lp, tp, blocks, max_new,
                                          D ** -0.5 if scale is None else scale, out.data_ptr(), out.dtype is torch.float32, _stream(ctx)))
    return out


def prompt_attention(ctx: Context, q, k, v, starts, *, scale: float = None, out_dtype=None, out=None):
    """Causal attention of whole prompts, packed: q bf16 [T][q_heads][D], k and v bf16 [T][kv_heads][D] (D 64 or 128; rows may be parts of
    wider ones) -> [T][q_heads][D], bf16 or fp32.  starts int32 [n + 1].  v must be finite throughout a prompt.  out must not overlap an
    input."""
    torch = _torch()
    (qp, qs), (kp, ks), (vp, vs) = _head_rows(ctx, "q", q), _head_rows(ctx, "k", k), _head_rows(ctx, "v", v)
    T, heads, D = q.shape
    if k.shape != v.shape or k.shape[0] != T or k.shape[2] != D:
        _bad(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together", _lib.ERR_SHAPE)
    n = starts.shape[0] - 1
    sp = _need(ctx, "starts", starts, torch.int32, (n + 1,))
    out = _out(ctx, q, out_dtype, out)
    ctx.check(ctx.lib.mpq_prompt_attention(_raw(ctx.h), qp, qs, kp, ks, vp, vs, T, heads, k.shape[1], D, n, sp, D ** -0.5 if scale is None else scale,
                                           out.data_ptr(), out.dtype is torch.float32, _stream(ctx)))
    return out
