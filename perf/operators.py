"""The operators between a decoder layer's projections, as timed cases: their plain form in torch, and the library's calls.

A case is a dict of plain values with a "kind":

  plan     kv_plan           pages, block tables, slot maps and positions of a step, from the requests' lengths
  append   kv_append         rotary positions on the rows of a QKV projection; q out, k and v rows into the paged cache
  paged    paged_attention   attention of each request's new tokens over its pages
  prompt   prompt_attention  causal attention over whole prompts, packed one behind the other
  norm     residual_norm     norm of a block's output, gate, residual sum, norm in front of the next block

Head counts and widths are those of the 7B and 70B projections of the benchmark (32 heads of 128 on 4096; 64 on 8192, there with 8
heads of keys and values) and generic smaller ones.  Lengths go by the case alone ("mix" is their seed), values by the seed.
"""
import math
import random

import torch

own = False

_context = []


def _library():
    """The package and one context per process, as a program keeps it."""
    import makepad_b200 as mpq
    if not _context:
        _context.append(mpq.Context(0))
    return mpq, _context[0]


def listed():
    return [
        # 64 requests decoded together, a token each: the smallest call, where latency counts
        {"name": "plan decode 64", "kind": "plan", "n": 64, "new": 1, "kv": 4096, "P": 16, "ended": 0.0, "mix": 1},
        # a step of a busy server: a thousand requests, some with a chunk of a prompt, some that have ended
        {"name": "plan mixed 1000", "kind": "plan", "n": 1000, "new": 64, "kv": 8192, "P": 16, "ended": 0.1, "mix": 2},
        # the QKV rows of 64 sequences of the 7B shape behind a Q4 projection (fp32 rows)
        {"name": "append 64 rows 7B", "kind": "append", "T": 64, "Hq": 32, "Hkv": 32, "D": 128, "P": 16, "dtype": "fp32", "rot": 128, "interleaved": False, "far": 4096, "mix": 3},
        # a prompt of the 70B shape behind an NVFP4 projection (bf16 rows), at far positions
        {"name": "append 8000 rows 70B", "kind": "append", "T": 8000, "Hq": 64, "Hkv": 8, "D": 128, "P": 64, "dtype": "bf16", "rot": 128, "interleaved": True, "far": 131072, "mix": 4},
        # one request of the 7B shape, one token: latency
        {"name": "decode 1 request 7B", "kind": "paged", "n": 1, "new": 1, "kv": 4001, "Hq": 32, "Hkv": 32, "D": 128, "P": 16, "mix": 5},
        # 64 requests of unlike lengths, a token each, grouped heads: the cache is read once
        {"name": "decode 64 requests 70B", "kind": "paged", "n": 64, "new": 1, "kv": 8000, "Hq": 64, "Hkv": 8, "D": 128, "P": 16, "mix": 6},
        # two requests' chunks of a long prompt over what they have in the cache
        {"name": "chunk 1024 over 16000", "kind": "paged", "n": 2, "new": 1024, "kv": 16000, "Hq": 64, "Hkv": 8, "D": 128, "P": 64, "mix": 7},
        # one prompt of no round length, 7B shape
        {"name": "prompt 1000 7B", "kind": "prompt", "n": 1, "least": 1000, "most": 1000, "Hq": 32, "Hkv": 32, "D": 128, "mix": 8},
        # prompts of 17 to 1500 tokens packed, narrow heads in groups
        {"name": "prompts packed 16", "kind": "prompt", "n": 16, "least": 17, "most": 1500, "Hq": 32, "Hkv": 8, "D": 64, "mix": 9},
        # a long prompt, grouped heads: the tensor cores' rate
        {"name": "prompt 8192", "kind": "prompt", "n": 1, "least": 8192, "most": 8192, "Hq": 32, "Hkv": 8, "D": 128, "mix": 10},
        # one token of the 7B shape in front of a Q4 projection
        {"name": "norm 1 row 7B", "kind": "norm", "M": 1, "H": 4096, "x": "fp32", "out": "fp32", "post": False, "gate": "none"},
        # a prompt's rows: norm behind the block too, a gate of one value per column, bf16 for an NVFP4 projection
        {"name": "norm 8192 rows 70B", "kind": "norm", "M": 8192, "H": 8192, "x": "bf16", "out": "bf16", "post": True, "gate": "row"},
    ]


#: query heads, key and value heads, width of a head
_HEADS = [(32, 32, 128), (64, 8, 128), (32, 8, 128), (40, 8, 128), (28, 4, 128), (32, 8, 64), (12, 12, 64), (15, 5, 64)]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform over lo..hi."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind, mix = rng.choice(["plan", "append", "paged", "paged", "prompt", "prompt", "norm"]), rng.randrange(1 << 30)
    q, kv, d = rng.choice(_HEADS)
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        n = _log(rng, 1, 1000)
        return {"kind": kind, "n": n, "new": rng.choice([1, _log(rng, 2, 64)]), "kv": _log(rng, 100, 8192), "P": page, "ended": rng.choice([0.0, 0.2]), "mix": mix}
    if kind == "append":
        rot = rng.choice([d, d, d // 2])
        return {"kind": kind, "T": _log(rng, 1, 8000), "Hq": q, "Hkv": kv, "D": d, "P": page, "dtype": rng.choice(["fp32", "bf16"]), "rot": rot,
                "interleaved": rng.choice([False, True]), "far": _log(rng, 1000, 131072), "mix": mix}
    if kind == "paged":
        new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 1024)])
        # what a pass holds: 56 requests of 8000 tokens at most, and 2^31 scores in the plain form
        length = _log(rng, max(new, 64), 16000)
        n = _log(rng, 1, max(1, min(64, 56 * 8000 * 8 // (length * kv), (1 << 31) // (q * new * length))))
        return {"kind": kind, "n": n, "new": new, "kv": length, "Hq": q, "Hkv": kv, "D": d, "P": page, "mix": mix}
    if kind == "prompt":
        most = _log(rng, 16, 6000)
        n = _log(rng, 1, max(1, min(32, (1 << 31) // (q * most * most))))
        return {"kind": kind, "n": n, "least": _log(rng, 1, most), "most": most, "Hq": q, "Hkv": kv, "D": d, "mix": mix}
    h = _log(rng, 32, 1024) * 8
    return {"kind": kind, "M": _log(rng, 1, 8192), "H": h, "x": rng.choice(["fp32", "bf16"]), "out": rng.choice(["fp32", "bf16"]),
            "post": rng.choice([False, True]), "gate": rng.choice(["none", "row", "all"])}


def _lengths(case):
    """The requests' lengths, of the case alone: (new tokens, tokens in the cache with them) of each; the first has the most."""
    r, n = random.Random(case["mix"]), case["n"]
    if case["kind"] == "prompt":
        new = [case["most"]] + [_log(r, case["least"], case["most"]) for _ in range(n - 1)]
        return new, list(new)
    new = [case["new"]] + [r.randint(1, case["new"]) for _ in range(n - 1)]
    kv = [case["kv"]] + [r.randint(max(k, case["kv"] // 8), max(k, case["kv"])) for k in new[1:]]
    if case["kind"] == "plan":
        new = [-1 if i and r.random() < case["ended"] else k for i, k in enumerate(new)]
    return new, [max(k, t) for k, t in zip(new, kv)]


def _ceil(a, b):
    return -(-a // b)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(new):
    return _ints([sum(new[:i]) for i in range(len(new) + 1)])


def _tables(g, lens, page, width, pages):
    """Block tables over pages in random order, and the pages left over."""
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    blocks = _ints([_ceil(t, page) for t in lens], torch.int64)
    first = blocks.cumsum(0) - blocks
    j = torch.arange(width, device="cuda")
    at = first[:, None] + j
    table = torch.where(j < blocks[:, None], order[at.clamp(max=pages - 1)], torch.zeros_like(order[:1]))
    return table.to(torch.int32).contiguous(), order[sum(_ceil(t, page) for t in lens):]


def prepare(case, seed):
    g, kind, s = _gen(seed), case["kind"], dict(case)
    if kind in ("plan", "paged", "prompt"):
        new, lens = _lengths(case)
    if kind == "plan":
        page = case["P"]
        before = [max(0, t - max(k, 0)) for k, t in zip(new, lens)]
        width = max(_ceil(t, page) for t in lens)
        pages = sum(_ceil(t, page) for t in lens) + 64
        table, left = _tables(g, before, page, width, pages)
        s.update(new_lens=_ints(new), lens=_ints(before), table=table, tokens=sum(max(k, 0) for k in new))
        s["free"] = torch.cat([left, left.new_zeros(pages - left.numel())])
        s["count"] = _ints([left.numel()])
    elif kind == "append":
        t, d, page = case["T"], case["D"], case["P"]
        pages = _ceil(t, page) + 3
        s["qkv"] = _randn(g, t, (case["Hq"] + 2 * case["Hkv"]) * d, dtype=torch.float32 if case["dtype"] == "fp32" else torch.bfloat16)
        s["positions"] = torch.randint(0, case["far"], (t,), device="cuda", generator=g, dtype=torch.int32)
        s["slots"] = torch.randperm(pages * page, device="cuda", generator=g)[:t].contiguous()
        s["freq"] = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        s["k"], s["v"] = _randn(g, pages, case["Hkv"], page, d), _randn(g, pages, case["Hkv"], page, d)
    elif kind == "paged":
        page = case["P"]
        pages = sum(_ceil(t, page) for t in lens) + 5
        s["k"], s["v"] = (_randn(g, pages, case["Hkv"], page, case["D"]) for _ in range(2))
        s["table"], _ = _tables(g, lens, page, _ceil(max(lens), page), pages)
        s.update(q=_randn(g, sum(new), case["Hq"], case["D"]), starts=_starts(new), lens=_ints(lens), most_new=max(new), most_kv=max(lens))
    elif kind == "prompt":
        # rows of a projection: q, k and v of a token beside each other
        rows = _randn(g, sum(new), case["Hq"] + 2 * case["Hkv"], case["D"])
        s["q"], s["k"], s["v"] = rows.split([case["Hq"], case["Hkv"], case["Hkv"]], dim=1)
        s.update(starts=_starts(new), most=max(new))
    else:
        m, h = case["M"], case["H"]
        s["x"] = _randn(g, m, h, dtype=torch.float32 if case["x"] == "fp32" else torch.bfloat16)
        s["residual"] = _randn(g, m, h, dtype=torch.float32) * 4
        s["weight"] = 1 + 0.1 * _randn(g, h, dtype=torch.float32)
        s["post_weight"] = 1 + 0.1 * _randn(g, h, dtype=torch.float32) if case["post"] else None
        s["gate_values"] = {"none": None, "row": _randn(g, h, dtype=torch.float32), "all": _randn(g, m, h, dtype=torch.float32)}[case["gate"]]
    return s


EPS, ALPHA = 1e-6, 0.5


# ---- the plain forms -----------------------------------------------------------------------------------------------------


def _plain_plan(s):
    page, table, free, tokens = s["P"], s["table"], s["free"], s["tokens"]
    new, old, count = s["new_lens"].long(), s["lens"].long(), s["count"].long()
    (n, width), pages = table.shape, free.numel()
    j = torch.arange(width, device="cuda")
    ended, grow = new < 0, new.clamp(min=0)
    before = torch.where(ended, 0, old)
    after, had = before + grow, (old + page - 1) // page
    given, kept = torch.where(ended, had, 0), torch.where(ended, 0, had)
    # the pages of ended requests go on top of the free ones
    at = count + (given.cumsum(0) - given)[:, None] + j
    spot = torch.where(j < given[:, None], at, pages)
    free.copy_(torch.cat([free, free[:1]]).scatter(0, spot.reshape(-1), table.reshape(-1))[:pages])
    total = count + given.sum()
    # all requests grow, or none
    need = (after + page - 1) // page - kept
    missing = (need.sum() - total).clamp(min=0)
    missing = torch.where(grow.sum() > tokens, -2, missing)
    missing = torch.where((after > width * page).any(), -1, missing)
    fits = missing == 0
    fresh = (j >= kept[:, None]) & (j < (kept + need)[:, None]) & fits
    top = total - 1 - ((need.cumsum(0) - need - kept)[:, None] + j)
    table.copy_(torch.where(fresh, free[top.clamp(0, pages - 1)], table))
    grow = torch.where(fits, grow, 0)
    starts = torch.cat([grow.new_zeros(1), grow.cumsum(0)])
    t = torch.arange(tokens, device="cuda")
    who = torch.searchsorted(starts[1:], t, right=True).clamp(max=n - 1)
    pos = before[who] + t - starts[who]
    live = t < starts[-1]
    slot = table[who, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    return {"starts": starts.int(), "lens": (before + grow).int(), "positions": torch.where(live, pos, 0).int(), "slots": torch.where(live, slot, -1),
            "count": (total - torch.where(fits, need.sum(), 0)).int(), "missing": missing.int(), "table": table, "free": free}


def _plain_rotate(x, cos, sin, rot, interleaved):
    """x [T][H][D]: the first `rot` elements of each head turned by pairs, (i, i + rot/2) or (2i, 2i + 1)."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _plain_append(s):
    t, d, page = s["T"], s["D"], s["P"]
    x = s["qkv"].float().view(t, -1, d)
    q, k, v = x.split([s["Hq"], s["Hkv"], s["Hkv"]], dim=1)
    angle = s["positions"].double()[:, None] * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    where, off = s["slots"] // page, s["slots"] % page
    s["k"][where, :, off] = _plain_rotate(k, cos, sin, s["rot"], s["interleaved"]).bfloat16()
    s["v"][where, :, off] = v.bfloat16()
    return _plain_rotate(q, cos, sin, s["rot"], s["interleaved"]).bfloat16(), s["k"], s["v"]


def _plain_attention(q, k, v, new, lens):
    """q [n][Hkv][G][Q][D], k and v [n][Hkv][L][D] in 32 bits; request i has new[i] rows of q and lens[i] keys."""
    n, heads, group, rows, d = q.shape
    keys = k.shape[2]
    s = torch.matmul(q.reshape(n, heads, group * rows, d), k.transpose(2, 3)).mul_(d ** -0.5).view(n, heads, group, rows, keys)
    last = (lens - new)[:, None] + torch.arange(rows, device="cuda")
    seen = torch.arange(keys, device="cuda") <= last[..., None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p.view(n, heads, group * rows, keys), v).view(n, heads, group, rows, d) / total


def _padded(starts, new, most, tokens):
    """Rows of request i and place j among packed tokens, and whether there is one."""
    j = torch.arange(most, device="cuda")
    there = j < new[:, None]
    return torch.where(there, starts[:-1, None].long() + j, tokens), there


def _plain_unpad(o, at, tokens):
    n, heads, group, rows, d = o.shape
    out = torch.zeros(tokens + 1, heads * group, d, dtype=torch.bfloat16, device="cuda")
    out[at] = o.permute(0, 3, 1, 2, 4).reshape(n, rows, heads * group, d).bfloat16()
    return out[:tokens]


def _plain_paged(s):
    tokens, heads, d, page = s["q"].shape[0], s["Hkv"], s["D"], s["P"]
    new = s["starts"].diff()
    at, _ = _padded(s["starts"], new, s["most_new"], tokens)
    q = s["q"][at.clamp(max=tokens - 1)].float().view(s["n"], s["most_new"], heads, -1, d).permute(0, 2, 3, 1, 4)
    table = s["table"].long()
    keys = table.shape[1] * page
    k = s["k"][table].permute(0, 2, 1, 3, 4).reshape(s["n"], heads, keys, d).float()
    v = s["v"][table].permute(0, 2, 1, 3, 4).reshape(s["n"], heads, keys, d).float()
    return _plain_unpad(_plain_attention(q, k, v, new, s["lens"]), at, tokens)


def _plain_prompt(s):
    tokens, heads, d, most = s["q"].shape[0], s["Hkv"], s["D"], s["most"]
    new = s["starts"].diff()
    at, _ = _padded(s["starts"], new, most, tokens)
    rows = at.clamp(max=tokens - 1)
    q = s["q"][rows].float().view(s["n"], most, heads, -1, d).permute(0, 2, 3, 1, 4)
    k, v = (s[x][rows].float().permute(0, 2, 1, 3) for x in ("k", "v"))
    # (the rows behind a prompt's end are copies of another's: they see keys, and are left out)
    return _plain_unpad(_plain_attention(q, k, v, new.clamp(max=most), new), at, tokens)


def _plain_rms(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _plain_norm(s):
    x = s["x"].float()
    if s["post_weight"] is not None:
        x = _plain_rms(x, s["post_weight"])
    if s["gate_values"] is not None:
        x = x * s["gate_values"]
    r = s["residual"] + ALPHA * x
    return r, _plain_rms(r, s["weight"]).to(torch.float32 if s["out"] == "fp32" else torch.bfloat16)


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "paged": _plain_paged, "prompt": _plain_prompt, "norm": _plain_norm}


# ---- the library's calls ---------------------------------------------------------------------------------------------------


def _own(s):
    (mpq, ctx), kind = _library(), s["kind"]
    if kind == "plan":
        step = mpq.kv_plan(ctx, s["new_lens"], s["lens"], s["table"], s["free"], s["count"], page_size=s["P"], tokens=s["tokens"])
        return {"starts": step.starts, "lens": step.lens, "positions": step.positions, "slots": step.slots, "count": step.free_count,
                "missing": step.missing, "table": s["table"], "free": s["free"]}
    if kind == "append":
        q, _, _ = mpq.kv_append(ctx, s["qkv"], s["Hq"], s["Hkv"], positions=s["positions"], frequencies=s["freq"], interleaved=s["interleaved"],
                                k_cache=s["k"], v_cache=s["v"], slots=s["slots"])
        return q, s["k"], s["v"]
    if kind == "paged":
        return mpq.paged_attention(ctx, s["q"], s["k"], s["v"], s["starts"], s["lens"], s["table"], max_new=s["most_new"])
    if kind == "prompt":
        return mpq.prompt_attention(ctx, s["q"], s["k"], s["v"], s["starts"])
    return mpq.residual_norm(ctx, s["x"], s["residual"], s["weight"], eps=EPS, alpha=ALPHA, post_weight=s["post_weight"], gate=s["gate_values"],
                             out_dtype=torch.float32 if s["out"] == "fp32" else torch.bfloat16)


def run(s):
    return _own(s) if own else _PLAIN[s["kind"]](s)


def _pairs(new, kv):
    """Pairs of a query token and a key that it sees."""
    return sum(k * t - k * (k - 1) // 2 for k, t in zip(new, kv))


def work(case):
    kind = case["kind"]
    if kind == "norm":
        m, h = case["M"], case["H"]
        size = {"fp32": 4, "bf16": 2}
        gate = {"none": 0, "row": h, "all": m * h}[case["gate"]]
        return {"bytes": m * h * (size[case["x"]] + 8 + size[case["out"]]) + 4 * (h + gate + (h if case["post"] else 0)), "flops": 8 * m * h}
    if kind == "append":
        wide = (case["Hq"] + 2 * case["Hkv"]) * case["D"]
        return {"bytes": case["T"] * (wide * (6 if case["dtype"] == "fp32" else 4) + 12) + 4 * case["rot"], "flops": 3 * case["T"] * wide}
    new, kv = _lengths(case)
    if kind == "plan":
        page, tokens = case["P"], sum(max(k, 0) for k in new)
        moved = sum(_ceil(t, page) if k < 0 else _ceil(t, page) - _ceil(t - k, page) for k, t in zip(new, kv))
        return {"bytes": 16 * case["n"] + 8 * moved + 12 * tokens + 16, "flops": 0}
    tokens, q, heads, d = sum(new), case["Hq"], case["Hkv"], case["D"]
    tables = sum(_ceil(t, case["P"]) for t in kv) * 4 if kind == "paged" else 0
    return {"bytes": 4 * sum(kv) * heads * d + 4 * tokens * q * d + tables + 8 * case["n"], "flops": 4 * d * q * _pairs(new, kv)}


# ---- 64 bits, from the definitions ---------------------------------------------------------------------------------------------


def _exact_rows(q, k, v):
    """q [a][Hq][D], k and v [b][Hkv][D], the a rows the last of the b keys' tokens."""
    a, heads, d = q.shape
    b, group = k.shape[0], heads // k.shape[1]
    future = torch.ones(a, b, dtype=torch.bool, device="cuda").triu(b - a + 1)
    out = torch.empty(a, heads, d, dtype=torch.float64, device="cuda")
    for h in range(heads):
        scores = (q[:, h].double() @ k[:, h // group].double().T) / math.sqrt(d)
        out[:, h] = torch.softmax(scores.masked_fill(future, -math.inf), dim=1) @ v[:, h // group].double()
    return out


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "plan":
        return None
    if kind == "norm":
        x = s["x"].double()
        if s["post_weight"] is not None:
            x = x / ((x * x).sum(1, keepdim=True) / case["H"] + EPS).sqrt() * s["post_weight"].double()
        r = s["residual"].double() + ALPHA * x * (1.0 if s["gate_values"] is None else s["gate_values"].double())
        return r, r / ((r * r).sum(1, keepdim=True) / case["H"] + EPS).sqrt() * s["weight"].double()
    if kind == "append":
        t, rot, d, page = case["T"], case["rot"], case["D"], case["P"]
        x = s["qkv"].double().reshape(t, -1, d)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["freq"])[:, None]
        first = x[..., :rot].unflatten(-1, (rot // 2, 2) if case["interleaved"] else (2, rot // 2))
        pair = torch.view_as_complex((first if case["interleaved"] else first.transpose(-1, -2)).contiguous()) * turn
        back = torch.view_as_real(pair)
        turned = torch.cat([(back if case["interleaved"] else back.transpose(-1, -2)).flatten(-2), x[..., rot:]], dim=-1)
        caches = []
        for cache, rows in ((s["k"], turned[:, case["Hq"]:case["Hq"] + case["Hkv"]]), (s["v"], x[:, case["Hq"] + case["Hkv"]:])):
            flat = cache.double().transpose(1, 2).reshape(-1, case["Hkv"], d)
            flat[s["slots"]] = rows
            caches.append(flat.view(-1, page, case["Hkv"], d).transpose(1, 2).contiguous())
        return turned[:, :case["Hq"]].contiguous(), caches[0], caches[1]
    if kind == "prompt":
        at = s["starts"].tolist()
        return torch.cat([_exact_rows(s["q"][a:b], s["k"][a:b], s["v"][a:b]) for a, b in zip(at, at[1:])])
    at, parts = s["starts"].tolist(), []
    for i, length in enumerate(s["lens"].tolist()):
        pages = s["table"][i, :_ceil(length, case["P"])].long()
        k, v = (s[c][pages].transpose(1, 2).reshape(-1, case["Hkv"], case["D"])[:length] for c in ("k", "v"))
        parts.append(_exact_rows(s["q"][at[i]:at[i + 1]], k, v))
    return torch.cat(parts)
