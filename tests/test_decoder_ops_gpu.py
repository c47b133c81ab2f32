"""Norms, the paged cache and attention against plain forms in 64 bits, at the sizes and masks where they can go wrong.

u is half a step of fp32 (2^-24), B half a step of bf16 (2^-8), both relative; each tolerance counts them."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

U, B = 2.0 ** -24, 2.0 ** -8


def _t():
    import torch
    return torch


def _m():
    import makepad_b200
    return makepad_b200


def _randn(seed, *shape, dtype=None):
    torch = _t()
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g)
    return x if dtype is None else x.to(dtype)


def _ints(values, dtype=None):
    torch = _t()
    return torch.tensor(values, dtype=dtype or torch.int32, device="cuda")


# ---- norms ---------------------------------------------------------------------------------------------------------------


def _norm_reference(x, residual, weight, post, gate, alpha, eps):
    """(residual', y) in 64 bits and how far fp32 may be from them."""
    torch = _t()
    H = x.shape[1]
    # a sum of H squares: at most 32 in a row in a thread, ten levels of shuffles and warps; half of it after the root, the division,
    # the root and two products: 21 + 5 roundings, taken as 32
    n = 32 * U
    t = x.double()
    if post is not None:
        t = t / (t.square().mean(1, keepdim=True) + eps).sqrt() * post.double()
    if gate is not None:
        t = t * gate.double()
    r = alpha * t + (0 if residual is None else residual.double())
    r_off = U * r.abs() + n * (alpha * t).abs() + 2.0 ** -149
    inv = 1 / (r.square().mean(1, keepdim=True) + eps).sqrt()
    w = torch.ones(H, dtype=torch.float64, device="cuda") if weight is None else weight.double()
    y = r * inv * w
    # the row's scale moves with the error of the whole row
    y_off = n * y.abs() + (inv * w).abs() * r_off + y.abs() * r_off.norm(dim=1, keepdim=True) / r.norm(dim=1, keepdim=True).clamp(min=1e-30)
    return r, r_off, y, y_off


@pytest.mark.parametrize("M,H", [(1, 8), (1, 4096), (3, 264), (7, 11008), (200, 4096), (300, 2056), (150, 8192), (2, 32768), (160, 16384)])
@pytest.mark.parametrize("kinds", [("fp32", "fp32"), ("bf16", "bf16"), ("fp32", "bf16"), ("bf16", "fp32")])
def test_residual_norm(ctx, M, H, kinds):
    torch, m = _t(), _m()
    types = {"fp32": torch.float32, "bf16": torch.bfloat16}
    x = _randn(1, M, H, dtype=types[kinds[0]])
    residual, weight, post = _randn(2, M, H) * 3, 1 + _randn(3, H) * 0.2, 1 + _randn(4, H) * 0.2
    for k, (res, w, po, gate) in enumerate([(residual, weight, None, None), (None, weight, None, None), (residual, weight, post, _randn(5, H)),
                                            (residual, None, post, _randn(6, M, H)), (residual, weight, None, _randn(7, M, H))]):
        alpha, eps = (1.0, 1e-6) if k == 0 else (0.25, 1e-5)
        before = None if res is None else res.clone()
        r, y = m.residual_norm(ctx, x, res, w, eps=eps, alpha=alpha, post_weight=po, gate=gate, out_dtype=types[kinds[1]])
        want_r, r_off, want_y, y_off = _norm_reference(x, res, w, po, gate, alpha, eps)
        assert y.dtype is types[kinds[1]] and r.dtype is torch.float32
        assert bool(((r.double() - want_r).abs() <= r_off).all())
        y_off = y_off + (B * want_y.abs() + 2.0 ** -134 if kinds[1] == "bf16" else 0)
        assert bool(((y.double() - want_y).abs() <= y_off * (1 + 2 ** -7)).all()), float(((y.double() - want_y).abs() / y_off).max())
        if res is not None:
            assert torch.equal(res, before)
            r2, y2 = m.residual_norm(ctx, x, res, w, eps=eps, alpha=alpha, post_weight=po, gate=gate, out_dtype=types[kinds[1]], inplace=True)
            assert r2 is res and torch.equal(res, r) and torch.equal(y2, y)
            res.copy_(before)
    r, none = m.residual_norm(ctx, x, residual, norm=False)
    assert none is None and bool(((r.double() - (residual.double() + x.double())).abs() <= U * r.double().abs()).all())


def test_residual_norm_keeps_infinities_and_nan_in_their_rows(ctx):
    torch, m = _t(), _m()
    x = _randn(1, 6, 512)
    x[1, 3], x[3, 5], x[5] = math.inf, math.nan, 0.0
    r, y = m.residual_norm(ctx, x, None, None, eps=1e-6)
    fine = torch.isfinite(y).all(1).tolist()
    assert fine == [True, False, True, False, True, True] and bool((y[5] == 0).all())


def test_residual_norm_refuses(ctx):
    torch, m = _t(), _m()
    x = _randn(1, 4, 64)
    for bad in (lambda: m.residual_norm(ctx, x[:, :60].contiguous()), lambda: m.residual_norm(ctx, x.half()), lambda: m.residual_norm(ctx, x, x.bfloat16()),
                lambda: m.residual_norm(ctx, x, x[:2].contiguous()), lambda: m.residual_norm(ctx, x, weight=x[0, :32].contiguous()), lambda: m.residual_norm(ctx, x.cpu()),
                lambda: m.residual_norm(ctx, x.T), lambda: m.residual_norm(ctx, x[:0]), lambda: m.residual_norm(ctx, x, eps=-1.0), lambda: m.residual_norm(ctx, x, eps=math.nan),
                lambda: m.residual_norm(ctx, x, out_dtype=torch.float16), lambda: m.residual_norm(ctx, x, inplace=True), lambda: m.residual_norm(ctx, _randn(1, 1, 32776)),
                lambda: m.residual_norm(ctx, _randn(1, 257)[1:].view(4, 64))):
        with pytest.raises(m.MpqError):
            bad()


# ---- the plan of a step -----------------------------------------------------------------------------------------------------


def _plan_reference(new, lens, table, free, count, page, tokens):
    lens, table, free = list(lens), [list(r) for r in table], list(free)
    width = len(table[0])
    for i, k in enumerate(new):
        if k < 0:
            for b in range(-(-lens[i] // page)):
                free[count] = table[i][b]
                count += 1
            lens[i] = 0
    need = [-(-(t + max(k, 0)) // page) - -(-t // page) for k, t in zip(new, lens)]
    missing = max(0, sum(need) - count)
    if sum(max(k, 0) for k in new) > tokens:
        missing = -2
    if any(t + max(k, 0) > width * page for k, t in zip(new, lens)):
        missing = -1
    starts, positions, slots = [0], [], []
    for i, k in enumerate(new):
        k = max(k, 0) if missing == 0 else 0
        for pos in range(lens[i], lens[i] + k):
            if pos % page == 0:
                count -= 1
                table[i][pos // page] = free[count]
            positions.append(pos)
            slots.append(table[i][pos // page] * page + pos % page)
        lens[i] += k
        starts.append(starts[-1] + k)
    rest = tokens - len(slots)
    return starts, lens, positions + [0] * rest, slots + [-1] * rest, count, missing, table, free


def _plan_state(seed, n, page, most, new_most, spare, ended, width=None):
    r = random.Random(seed)
    lens = [r.randint(0, most) for _ in range(n)]
    new = [-1 if r.random() < ended else r.randint(0, new_most) for _ in range(n)]
    width = width or max(1, -(-(most + new_most) // page))
    used = sum(-(-t // page) for t in lens)
    order = list(range(used + spare))
    r.shuffle(order)
    table = [[-7] * width for _ in range(n)]
    for i, t in enumerate(lens):
        for b in range(-(-t // page)):
            table[i][b] = order.pop()
    return new, lens, table, order + [-9] * used, len(order)


def _plan_check(ctx, new, lens, table, free, count, page, tokens, inplace=False):
    torch, m = _t(), _m()
    want = _plan_reference(new, lens, table, free, count, page, tokens)
    lens_d, table_d, free_d, count_d = _ints(lens), _ints(table), _ints(free), _ints([count])
    step = m.kv_plan(ctx, _ints(new), lens_d, table_d, free_d, count_d, page_size=page, tokens=tokens, inplace=inplace)
    if inplace:
        assert step.lens is lens_d and step.free_count is count_d
    else:
        assert lens_d.tolist() == lens and count_d.tolist() == [count]
    got = [x.tolist() for x in (step.starts, step.lens, step.positions, step.slots, step.free_count, step.missing, table_d)]
    assert got[:4] == [want[0], want[1], want[2], want[3]]
    assert got[4] == [want[4]] and got[5] == [want[5]] and got[6] == want[6]
    assert free_d.tolist()[:count] == free[:count]                       # pages in use are taken off the count only
    assert free_d.tolist()[:want[4]] == want[7][:want[4]]
    return step


@pytest.mark.parametrize("n,page,most,new_most,ended", [(1, 16, 0, 1, 0.0), (1, 16, 100, 5000, 0.0), (5, 16, 40, 33, 0.4), (64, 16, 900, 1, 0.0), (64, 64, 700, 1, 0.5),
                                                        (300, 32, 300, 70, 0.2), (513, 16, 50, 3, 0.1), (1025, 256, 2000, 40, 0.3), (8192, 16, 60, 3, 0.2), (33, 16, 64, 0, 0.3)])
def test_kv_plan(ctx, n, page, most, new_most, ended):
    for seed, inplace in ((1, False), (2, True)):
        new, lens, table, free, count = _plan_state(seed, n, page, most, new_most, n * (new_most // page + 1) + 3, ended)
        tokens = sum(max(k, 0) for k in new)
        _plan_check(ctx, new, lens, table, free, count, page, tokens + (0 if seed == 1 else 77), inplace)


@pytest.mark.parametrize("n", [9, 900])
def test_kv_plan_grows_all_or_nothing(ctx, n):
    # too few pages, also where this step's returns are just enough, and one short of it
    new, lens, table, free, count = _plan_state(3, n, 16, 100, 60, 5 * n, 0.1)
    want = _plan_reference(new, lens, table, free, count, 16, 10 ** 6)
    assert want[5] == 0 and 0 < want[4] < count
    short = want[4]                                                      # pages left over: without them it fits exactly
    tokens = sum(max(k, 0) for k in new) + 5
    step = _plan_check(ctx, new, lens, table, free[short:] + [-9] * short, count - short, 16, tokens)
    assert step.missing.item() == 0 and step.free_count.item() == 0
    step = _plan_check(ctx, new, lens, table, free[short + 1:] + [-9] * (short + 1), count - short - 1, 16, tokens)
    assert step.missing.item() == 1 and step.starts.tolist() == [0] * (n + 1) and set(step.slots.tolist()) == {-1}
    # a request that is longer than its row of the table, and more tokens than there are rows
    new2 = list(new)
    new2[n // 2] = 16 * len(table[0]) + 1
    assert _plan_check(ctx, new2, lens, table, free, count, 16, 10 ** 4).missing.item() == -1
    assert _plan_check(ctx, new, lens, table, free, count, 16, tokens - 6).missing.item() == -2


def test_kv_plan_steps_of_a_server(ctx):
    """Fifty steps in place: what the tables say stays a division of the pages among the requests."""
    torch, m = _t(), _m()
    r, n, page, pages, width = random.Random(5), 40, 16, 600, 20
    lens, table, free, count = _ints([0] * n), _ints([[0] * width] * n), _ints(list(range(pages))), _ints([pages])
    host = [0] * n
    for _ in range(50):
        new = [-1 if host[i] and r.random() < 0.1 else r.choice([0, 1, 1, 1, r.randint(2, 50)]) for i in range(n)]
        new = [k if host[i] + k <= page * width else -1 for i, k in enumerate(new)]
        step = m.kv_plan(ctx, _ints(new), lens, table, free, count, page_size=page, tokens=sum(max(k, 0) for k in new), inplace=True)
        if step.missing.item() == 0:
            host = [0 if k < 0 else t + k for k, t in zip(new, host)]
        else:
            host = [0 if k < 0 else t for k, t in zip(new, host)]
        assert lens.tolist() == host
        rows = table.tolist()
        held = [p for t, row in zip(host, rows) for p in row[:-(-t // page)]]
        assert sorted(held + free.tolist()[:count.item()]) == list(range(pages))


def test_kv_plan_refuses(ctx):
    torch, m = _t(), _m()
    ok = dict(new=_ints([1]), lens=_ints([0]), table=_ints([[0]]), free=_ints([0]), count=_ints([1]), page=16, tokens=1)

    def call(**k):
        a = {**ok, **k}
        m.kv_plan(ctx, a["new"], a["lens"], a["table"], a["free"], a["count"], page_size=a["page"], tokens=a["tokens"])
    call()
    for bad in (dict(page=8), dict(page=48), dict(page=512), dict(tokens=-1), dict(new=_ints([1, 1])), dict(lens=_ints([0], torch.int64)), dict(table=_ints([0])),
                dict(table=_ints([[0], [0]])), dict(count=_ints([1, 1])), dict(free=_ints([])), dict(new=torch.tensor([1], dtype=torch.int32))):
        with pytest.raises((m.MpqError, RuntimeError)):
            call(**bad)
    with pytest.raises(m.MpqError):
        call(new=_ints([1] * 8193), lens=_ints([0] * 8193), table=_ints([[0]] * 8193))


# ---- rotary rows into the cache -----------------------------------------------------------------------------------------------


def _rotated(x, positions, freq, interleaved):
    torch = _t()
    rot = 2 * freq.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] * freq)[:, None]
    y = x.double().clone()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    z = torch.complex(a.contiguous(), b.contiguous()) * turn
    a.copy_(z.real)
    b.copy_(z.imag)
    return y


@pytest.mark.parametrize("T,q_heads,kv_heads,D,rot,page", [(1, 32, 32, 128, 128, 16), (5, 8, 1, 64, 32, 64), (130, 15, 5, 64, 64, 256), (3, 6, 2, 80, 48, 32), (9, 4, 4, 256, 256, 16),
                                                           (17, 12, 3, 16, 16, 16), (40, 64, 8, 128, 0, 128)])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_kv_append(ctx, T, q_heads, kv_heads, D, rot, page, kind, interleaved):
    torch, m = _t(), _m()
    wide = (q_heads + 2 * kv_heads) * D
    whole = _randn(1, T, wide + 40, dtype=torch.float32 if kind == "fp32" else torch.bfloat16)
    qkv = whole[:, 8:8 + wide] if kind == "bf16" else whole[:, 4:4 + wide]                 # rows 16-byte aligned, not contiguous
    pages = T // page + 3
    k_cache, v_cache = _randn(2, pages, kv_heads, page, D, dtype=torch.bfloat16), _randn(3, pages, kv_heads, page, D, dtype=torch.bfloat16)
    slots = torch.randperm(pages * page, device="cuda")[:T].contiguous()
    far = torch.randint(0, 1 << 20, (T,), device="cuda", dtype=torch.int32)
    far[0] = 2 ** 31 - 1 if T > 1 else 1048575
    freq = m.rotary_frequencies(ctx, rot) if rot else None
    skipped = T > 2
    if skipped:
        slots[T // 2] = -1
        slots[T - 1] = pages * page                                                        # behind the cache: q and rows only
    before = k_cache.clone(), v_cache.clone()
    q, k, v = m.kv_append(ctx, qkv, q_heads, kv_heads, positions=far if rot else None, frequencies=freq, interleaved=interleaved, k_cache=k_cache, v_cache=v_cache, slots=slots, rows=True)
    x = qkv.view(T, -1, D)
    turned = _rotated(x, far, freq, interleaved) if rot else x.double()
    wants = turned[:, :q_heads], turned[:, q_heads:q_heads + kv_heads], x[:, q_heads + kv_heads:].double()
    live = slots >= 0
    # the product position * frequency: 2^-53 of up to 2^31 turns; sine and cosine 2 u, their argument u pi; two products and a sum: 8 u of
    # |a| + |b|, which is at most 2 |(a, b)|; then bf16
    size = torch.sqrt(x.double().square().amax(2, keepdim=True) * 2)
    for got, want in zip((q, k, v), wants):
        off = (got.double() - want).abs() - B * want.abs() - (16 * U + 2 ** -20) * size[:, :1].amax(1, keepdim=True).clamp(min=size.max())
        assert bool((off[live] <= 0).all()), float(off[live].max())
    assert torch.equal(v[live], x[:, q_heads + kv_heads:].bfloat16()[live])
    flat = [c.transpose(1, 2).reshape(-1, kv_heads, D) for c in (k_cache, v_cache)]
    old = [c.transpose(1, 2).reshape(-1, kv_heads, D).clone() for c in before]
    inside = live & (slots < pages * page)
    for f, o, rows in zip(flat, old, (k, v)):
        o[slots[inside]] = rows[inside]
        assert torch.equal(f, o)
    q2, none, _ = m.kv_append(ctx, qkv, q_heads, kv_heads, positions=far if rot else None, frequencies=freq, interleaved=interleaved)
    assert none is None and torch.equal(q2[live], q[live])


def test_kv_append_leaves_skipped_rows(ctx):
    import ctypes as C
    torch, m = _t(), _m()
    x = _randn(1, 4, 3 * 64)
    q = torch.full((4, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros(2, 2, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    slots = _ints([3, -1, 5, -1], torch.int64)
    ctx.check(ctx.lib.mpq_kv_append(ctx.h, x.data_ptr(), 0, 192, 4, 1, 1, 64, None, None, 0, 0, q.data_ptr(), None, None, slots.data_ptr(), cache[0].data_ptr(), cache[1].data_ptr(), 2, 16,
                                    C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert bool((q[1] == 7).all()) and bool((q[3] == 7).all()) and torch.equal(q[0, 0], x[0, :64].bfloat16()) and torch.equal(q[2, 0], x[2, :64].bfloat16())
    assert int((cache != 0).any(-1).sum()) == 4


def test_kv_append_refuses(ctx):
    torch, m = _t(), _m()
    x, f, pos, slots = _randn(1, 4, 6 * 64), m.rotary_frequencies(ctx, 64), _ints([0, 1, 2, 3]), _ints([0, 1, 2, 3], torch.int64)
    cache = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    ok = dict(positions=pos, frequencies=f, k_cache=cache, v_cache=cache.clone(), slots=slots)
    m.kv_append(ctx, x, 4, 1, **ok)
    for heads, bad in (((4, 1), dict(frequencies=f.float())), ((4, 1), dict(positions=None)), ((4, 1), dict(k_cache=None)), ((4, 1), dict(slots=slots.int())), ((4, 1), dict(positions=pos[:3])),
                       ((2, 2), {}), ((5, 1), {}), ((0, 3), {}), ((4, 1), dict(k_cache=cache[:, :, :8].contiguous(), v_cache=cache[:, :, :8].contiguous())),
                       ((4, 1), dict(v_cache=cache[:1].contiguous())), ((4, 1), dict(frequencies=m.rotary_frequencies(ctx, 80))), ((4, 1), dict(frequencies=m.rotary_frequencies(ctx, 24))),
                       ((4, 1), dict(k_cache=cache.float(), v_cache=cache.float()))):
        with pytest.raises(m.MpqError):
            m.kv_append(ctx, x, *heads, **{**ok, **bad})
    for rows in (x.half(), x.cpu(), x.T, x[:0], _randn(1, 4, 386)[:, 1:385], _randn(1, 4, 387)[:, :384]):
        with pytest.raises(m.MpqError):
            m.kv_append(ctx, rows, 4, 1)


# ---- attention -----------------------------------------------------------------------------------------------------------------


def _attention_reference(q, k, v, scale):
    """q [a][Hq][D] the last a tokens of k, v [b][Hkv][D] -> (out in 64 bits, what the weights' rounding can move it by)."""
    torch = _t()
    a, heads, D = q.shape
    b, kv_heads = k.shape[0], k.shape[1]
    out = torch.zeros(a, heads, D, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(out)
    if a == 0 or b == 0:
        return out, mass
    i, j = torch.arange(a, device="cuda")[:, None], torch.arange(b, device="cuda")[None]
    seen = j <= b - a + i
    rows = seen.any(1)
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv_heads)].double(), v[:, h // (heads // kv_heads)].double()
        s = (scale * (q[:, h].double() @ kh.T)).masked_fill(~seen, -math.inf)
        p = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300))
        p = torch.where(rows[:, None], p / p.sum(1, keepdim=True).clamp(min=1e-300), 0.0)
        out[:, h], mass[:, h] = p @ vh, p @ vh.abs()
    return out, mass


def _off(got, out, mass, D, scores):
    """got - out over what it may be: a weight of v is rounded to bf16 (B of its share); a score is a sum of D products in fp32, each rounded or cut
    to 2 u of the sum of magnitudes (`scores`), which moves the weights by that relatively, twice (their sum moves too); a sum over the keys in fp32
    2^-12 of the magnitudes (a thousand additions, each cut to 2 u); then the output's own rounding."""
    allowed = mass * (B + 2 ** -12 + 4 * D * U * scores) + (B * out.abs() if got.dtype is _t().bfloat16 else 0) + 2.0 ** -126
    return float(((got.double() - out).abs() / allowed).max()) if got.numel() else 0.0


def _paged_case(seed, new, lens, kv_heads, D, page, extra=2, poison=True):
    """Caches whose unused places hold NaN, and tables whose unused entries lie outside the cache."""
    torch = _t()
    r = random.Random(seed)
    blocks = [-(-t // page) for t in lens]
    pages = sum(blocks) + extra
    order = list(range(pages))
    r.shuffle(order)
    width = max(max(blocks), 1) + 1
    table = [[order.pop() if b < blocks[i] else r.choice([-1, 2 ** 31 - 1, pages]) for b in range(width)] for i in range(len(lens))]
    k, v = _randn(seed + 1, pages, kv_heads, page, D, dtype=torch.bfloat16), _randn(seed + 2, pages, kv_heads, page, D, dtype=torch.bfloat16)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for i, t in enumerate(lens):
        for b in range(blocks[i]):
            used[table[i][b], :min(page, t - b * page)] = True
    if poison:
        hole = ~used.cuda()[:, None, :, None].expand_as(k)
        k[hole], v[hole] = math.nan, math.inf
    return k, v, table


def _gathered(cache, row, t, page):
    torch = _t()
    pages = torch.tensor(row[:-(-t // page)], dtype=torch.int64, device="cuda")
    return cache[pages].transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:t]


def _check_paged(ctx, new, lens, q_heads, kv_heads, D, page, seed=0, max_new=None, out_dtype=None, stride=0, scale=None):
    torch, m = _t(), _m()
    k, v, table = _paged_case(seed, new, lens, kv_heads, D, page)
    T = sum(new)
    q = _randn(seed + 3, max(T, 1), q_heads * D + stride, dtype=torch.bfloat16)[:, :q_heads * D].unflatten(1, (q_heads, D))
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    got = m.paged_attention(ctx, q, k, v, _ints(starts), _ints(lens), _ints(table), max_new=max(new) if max_new is None else max_new, out_dtype=out_dtype, scale=scale)
    again = m.paged_attention(ctx, q, k, v, _ints(starts), _ints(lens), _ints(table), max_new=max(new) if max_new is None else max_new, out_dtype=out_dtype, scale=scale)
    assert torch.equal(got[:T], again[:T])
    scale = D ** -0.5 if scale is None else scale
    for i, (a, t) in enumerate(zip(new, lens)):
        kk, vv = (_gathered(c, table[i], t, page) for c in (k, v))
        mine = got[starts[i]:starts[i + 1]]
        qq = q[starts[i]:starts[i + 1]]
        out, mass = _attention_reference(qq, kk, vv, scale)
        size = scale * float(qq.double().norm(dim=2).max() * kk.double().norm(dim=2).max()) if a and t else 0.0
        assert _off(mine, out, mass, D, size) <= 1, (i, a, t, _off(mine, out, mass, D, size))
        assert bool((mine[:max(0, a - t)] == 0).all())                 # rows without a key


HEADS = [(4, 4, 128), (8, 1, 128), (6, 2, 64), (5, 1, 64), (16, 1, 128), (20, 1, 64)]


@pytest.mark.parametrize("q_heads,kv_heads,D", HEADS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_paged_attention_single_tokens(ctx, q_heads, kv_heads, D, page):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 3001]
    _check_paged(ctx, [1] * len(lens), lens, q_heads, kv_heads, D, page)


@pytest.mark.parametrize("q_heads,kv_heads,D", HEADS)
@pytest.mark.parametrize("page", [16, 128])
def test_paged_attention_chunks(ctx, q_heads, kv_heads, D, page):
    new = [3, 1, 8, 0, 17, 40, 130, 2, 300, 0]
    lens = [3, 700, 9, 50, 500, 41, 130, 2000, 777, 0]
    _check_paged(ctx, new, lens, q_heads, kv_heads, D, page)
    _check_paged(ctx, new, lens, q_heads, kv_heads, D, page, max_new=0, out_dtype=_t().float32, stride=64, scale=0.3)


@pytest.mark.parametrize("max_new", [0, 1, 300])
def test_paged_attention_rows_without_keys(ctx, max_new):
    """More new tokens than the cache holds: the first rows see nothing and are zero; whatever max_new says."""
    _check_paged(ctx, [5, 300, 7, 1, 2], [2, 100, 0, 0, 900], 8, 2, 128, 16, max_new=max_new)


@pytest.mark.parametrize("new,length,heads", [([1], 40001, (8, 1, 128)), ([1], 20000, (2, 2, 64)), ([5, 1], 9000, (4, 2, 128)), ([600], 5000, (8, 2, 128)), ([200, 1, 64], 12000, (4, 1, 64))])
def test_paged_attention_long(ctx, new, length, heads):
    lens = [length] + [max(k, length // 3) for k in new[1:]]
    _check_paged(ctx, new, lens, *heads, 32)


@pytest.mark.parametrize("new,lens,heads", [([40] * 16, [700] * 16, (32, 8, 64)), ([40] * 19, [700] * 19, (32, 8, 64)), ([40, 0, 33] + [40] * 10, [700, 900, 33] + [1400] * 10, (16, 8, 128)),
                                            ([40] * 3, [5000, 40, 41], (8, 2, 128)), ([64, 20], [900, 2000], (8, 8, 128))])
def test_paged_attention_about_a_unit_for_each_cta(ctx, new, lens, heads):
    """Fewer units than SMs, and a few more; of like lengths, and not."""
    _check_paged(ctx, new, lens, *heads, 64)


@pytest.mark.parametrize("length", [41, 600, 5000])
def test_paged_attention_of_a_few_among_many_requests(ctx, length):
    """Several requests to an entry of the sums, most of them without new tokens."""
    new = [40 if i in (0, 77, 399) else 0 for i in range(400)]
    _check_paged(ctx, new, [length if k else 30 for k in new], 8, 2, 128, 16)


def test_paged_attention_many_requests(ctx):
    r = random.Random(1)
    lens = [r.randint(1, 300) for _ in range(700)]
    _check_paged(ctx, [1] * 700, lens, 8, 2, 64, 16)
    _check_paged(ctx, [r.randint(0, min(t, 20)) for t in lens], lens, 4, 4, 64, 16)


def test_paged_attention_large_scores(ctx):
    """Scores of several hundred, of both signs, and keys of one direction: the running maximum moves late and by much."""
    torch, m = _t(), _m()
    D, page, t = 128, 16, 2000
    k, v, table = _paged_case(1, [1], [t], 1, D, page)
    ramp = torch.linspace(-40, 40, t, device="cuda")
    q = torch.ones(300, 1, D, dtype=torch.bfloat16, device="cuda")
    flat = torch.zeros(t, 1, D, dtype=torch.bfloat16, device="cuda")
    flat[:, 0, :] = ramp[:, None].bfloat16()
    for i, b in enumerate(table[0][:-(-t // page)]):
        piece = flat[i * page:(i + 1) * page, 0]
        k[b, 0, :piece.shape[0]] = piece
    for order in (1, -1):
        for new in (1, 300):
            qq = (q[:new] * order).contiguous()
            got = m.paged_attention(ctx, qq, k, v, _ints([0, new]), _ints([t]), _ints(table), max_new=new)
            out, mass = _attention_reference(qq, _gathered(k, table[0], t, page), _gathered(v, table[0], t, page), D ** -0.5)
            assert _off(got, out, mass, D, 40 * D ** 0.5) <= 1


def test_paged_attention_entries_outside_the_cache_read_as_zeros(ctx):
    torch, m = _t(), _m()
    for D, new in ((128, 1), (64, 40), (128, 300)):
        k, v, table = _paged_case(4, [new], [600], 2, D, 16)
        zeroed = [list(table[0])]
        kk, vv = k.clone(), v.clone()
        for b, wrong in ((3, -1), (20, 2 ** 31 - 1), (30, k.shape[0])):
            kk[table[0][b]] = 0
            vv[table[0][b]] = 0
            zeroed[0][b] = wrong
        q = _randn(5, new, 6, D, dtype=torch.bfloat16)
        a = m.paged_attention(ctx, q, k, v, _ints([0, new]), _ints([600]), _ints(zeroed), max_new=new)
        b = m.paged_attention(ctx, q, kk, vv, _ints([0, new]), _ints([600]), _ints(table), max_new=new)
        assert torch.equal(a, b)


def test_paged_attention_bounds_its_lengths(ctx):
    """Lengths beyond the table and starts beyond the rows are cut, nothing else is read or written."""
    torch, m = _t(), _m()
    k, v, table = _paged_case(4, [1], [64], 1, 64, 16, poison=False)
    table = [table[0][:4]]
    q = _randn(5, 3, 2, 64, dtype=torch.bfloat16)
    out = torch.full((3, 2, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    m.paged_attention(ctx, q, k, v, _ints([0, 1]), _ints([10 ** 9]), _ints(table), max_new=1, out=out)
    want = m.paged_attention(ctx, q[:1], k, v, _ints([0, 1]), _ints([64]), _ints(table), max_new=1)
    assert torch.equal(out[:1], want) and bool((out[1:] == 9).all())
    for max_new in (1, 0):
        out.fill_(9)
        m.paged_attention(ctx, q, k, v, _ints([1, 2 ** 31 - 1]), _ints([64]), _ints(table), max_new=max_new, out=out)
        assert bool((out[0] == 9).all()) and bool(torch.isfinite(out).all()) and not bool((out[1:] == 9).any())


@pytest.mark.parametrize("q_heads,kv_heads,D", HEADS)
@pytest.mark.parametrize("lens", [[1], [2, 1, 0, 3], [127, 128, 129, 1, 0, 255, 256, 257], [1000], [5] * 60, [64, 700, 1, 300]])
def test_prompt_attention(ctx, q_heads, kv_heads, D, lens):
    torch, m = _t(), _m()
    T = sum(lens)
    rows = _randn(len(lens), T + 3, (q_heads + 2 * kv_heads) * D + 8, dtype=torch.bfloat16)[:, :-8].unflatten(1, (-1, D))
    q, k, v = rows.split([q_heads, kv_heads, kv_heads], dim=1)
    k[T:], v[T:] = math.nan, math.nan                                 # rows of nobody
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((T + 3, q_heads, D), 5.0, dtype=dtype, device="cuda")
        got = m.prompt_attention(ctx, q, k, v, _ints(starts), out=out)
        assert got is out and bool((out[T:] == 5).all())
        for i, t in enumerate(lens):
            at = slice(starts[i], starts[i + 1])
            want, mass = _attention_reference(q[at], k[at], v[at], D ** -0.5)
            size = D ** -0.5 * float(q[at].double().norm(dim=2).max() * k[at].double().norm(dim=2).max()) if t else 0.0
            assert _off(got[at], want, mass, D, size) <= 1, (i, t)


def test_prompt_attention_keeps_to_its_prompt(ctx):
    """NaN and infinities in one prompt do not reach its neighbours."""
    torch, m = _t(), _m()
    lens = [100, 77, 300, 130]
    starts = [0, 100, 177, 477, 607]
    q, k, v = (_randn(s, 607, 4, 128, dtype=torch.bfloat16) for s in (1, 2, 3))
    clean = m.prompt_attention(ctx, q, k, v, _ints(starts))
    k2, v2 = k.clone(), v.clone()
    k2[100:177], v2[100:177] = math.nan, math.inf
    k2[477:], v2[477:] = math.inf, math.nan
    got = m.prompt_attention(ctx, q, k2, v2, _ints(starts))
    assert torch.equal(got[:100], clean[:100]) and torch.equal(got[177:477], clean[177:477])
    assert not bool(torch.isfinite(got[100:177].float()).any())


def test_prompt_attention_long(ctx):
    torch, m = _t(), _m()
    T = 5003
    q, k, v = _randn(1, T, 4, 128, dtype=torch.bfloat16), _randn(2, T, 2, 128, dtype=torch.bfloat16), _randn(3, T, 2, 128, dtype=torch.bfloat16)
    got = m.prompt_attention(ctx, q, k, v, _ints([0, T]))
    want, mass = _attention_reference(q, k, v, 128 ** -0.5)
    assert _off(got, want, mass, 128, 128 ** -0.5 * 16 ** 2) <= 1
    assert torch.equal(got, m.prompt_attention(ctx, q, k, v, _ints([0, T])))


def test_attention_refuses(ctx):
    torch, m = _t(), _m()
    k, v, table = _paged_case(4, [1], [64], 2, 64, 16, poison=False)
    q, s, t, tb = _randn(5, 3, 4, 64, dtype=torch.bfloat16), _ints([0, 3]), _ints([64]), _ints(table)
    m.paged_attention(ctx, q, k, v, s, t, tb)
    wide = _randn(5, 3, 4, 96, dtype=torch.bfloat16)
    for a in ((q.float(), k, v, s, t, tb), (q, k.float(), v, s, t, tb), (q[:, :3], k, v, s, t, tb), (_randn(5, 3, 3, 64, dtype=torch.bfloat16), k, v, s, t, tb), (q, k, v, s[:1], t, tb),
              (q, k, v, s, t.long(), tb), (q, k, v, s, t, tb[0]), (q[:0], k, v, s, t, tb), (q.cpu(), k, v, s, t, tb), (q, k[:, :, :8].contiguous(), v[:, :, :8].contiguous(), s, t, tb),
              (q.transpose(0, 1), k, v, s, t, tb), (wide, wide.new_zeros(4, 2, 16, 96), wide.new_zeros(4, 2, 16, 96), s, t, tb)):
        with pytest.raises(m.MpqError):
            m.paged_attention(ctx, *a)
    for kw in (dict(scale=math.inf), dict(scale=math.nan), dict(max_new=-1), dict(out_dtype=torch.float16), dict(out=q[:2])):
        with pytest.raises(m.MpqError):
            m.paged_attention(ctx, q, k, v, s, t, tb, **kw)
    kk = _randn(6, 3, 2, 64, dtype=torch.bfloat16)
    m.prompt_attention(ctx, q, kk, kk, s)
    for a in ((q, kk[:2], kk, s), (q, kk, kk.float(), s), (wide, kk, kk, s), (q, kk, kk, s[:1]), (q, kk[:, :, :32], kk[:, :, :32], s), (q, kk, kk, s.long())):
        with pytest.raises(m.MpqError):
            m.prompt_attention(ctx, *a)


# ---- streams, graphs ---------------------------------------------------------------------------------------------------------------


def test_a_captured_step_follows_its_lengths(ctx):
    """plan -> append -> attention captured once and replayed while the requests grow, against eager calls on copies of the state."""
    torch, m = _t(), _m()
    n, heads, kv_heads, D, page, pages, width = 6, 8, 2, 128, 16, 64, 8
    freq = m.rotary_frequencies(ctx, D)

    def state():
        return dict(lens=_ints([0] * n), table=_ints([[0] * width] * n), free=_ints(list(range(pages))), count=_ints([pages]), new=_ints([0] * n),
                    k=torch.zeros(pages, kv_heads, page, D, dtype=torch.bfloat16, device="cuda"), v=torch.zeros(pages, kv_heads, page, D, dtype=torch.bfloat16, device="cuda"),
                    qkv=torch.zeros(64, (heads + 2 * kv_heads) * D, device="cuda"), out=torch.zeros(64, heads, D, dtype=torch.bfloat16, device="cuda"))

    def step(s):
        plan = m.kv_plan(ctx, s["new"], s["lens"], s["table"], s["free"], s["count"], page_size=page, tokens=64, inplace=True)
        q, _, _ = m.kv_append(ctx, s["qkv"], heads, kv_heads, positions=plan.positions, frequencies=freq, k_cache=s["k"], v_cache=s["v"], slots=plan.slots)
        m.paged_attention(ctx, q, s["k"], s["v"], plan.starts, plan.lens, s["table"], max_new=s.get("max_new", 0), out=s["out"])
        return plan

    for max_new in (0, 2):
        a, b = state(), state()
        a["max_new"] = b["max_new"] = max_new
        step(a)                                                       # (a warm-up: it reserves scratch)
        a.update(state(), max_new=max_new)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(a)
        r = random.Random(2)
        for i in range(12):
            new = [-1 if i > 5 and r.random() < 0.2 else r.randint(0, 10) for _ in range(n)]
            for s in (a, b):
                s["new"].copy_(_ints(new))
                s["qkv"].copy_(_randn(i, 64, (heads + 2 * kv_heads) * D))
            graph.replay()
            plan = step(b)
            live = plan.starts[-1].item()
            torch.cuda.synchronize()
            for x in ("lens", "count"):
                assert torch.equal(a[x], b[x])
            assert torch.equal(a["k"], b["k"]) and torch.equal(a["out"][:live], b["out"][:live])


def test_calls_on_another_stream(ctx):
    torch, m = _t(), _m()
    q, k, v = _randn(1, 900, 8, 128, dtype=torch.bfloat16), _randn(2, 900, 2, 128, dtype=torch.bfloat16), _randn(3, 900, 2, 128, dtype=torch.bfloat16)
    starts = _ints([0, 400, 900])
    want = m.prompt_attention(ctx, q, k, v, starts)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        q2 = q * 1.0
        got = m.prompt_attention(ctx, q2, k, v, starts)
    s.synchronize()
    assert torch.equal(got, want)
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))


@pytest.mark.parametrize("new,max_new", [([1, 1], 1), ([70, 3], 0)])
def test_a_cache_behind_32_bits(ctx, new, max_new):
    """Pages whose elements lie beyond 2^32 of a cache, and rows of q that lie 2^32 elements apart, give what a small cache and packed rows give."""
    torch, m = _t(), _m()
    q_heads, kv_heads, D, page, T = 8, 2, 128, 64, sum(new)
    lens, pages = [130, 75], (1 << 32) // (2 * 64 * 128) + 8
    starts, lens_dev, table = _ints([0, new[0], T]), _ints(lens), [[0, 1, 2], [3, 4, 0]]
    qkv = _randn(5, T, (q_heads + 2 * kv_heads) * D)
    places = [(i, lens[i] - n + j) for i, n in enumerate(new) for j in range(n)]
    freq, positions = m.rotary_frequencies(ctx, D), _ints([t for _, t in places])
    small = [_randn(6 + i, 5, kv_heads, page, D, dtype=torch.bfloat16) for i in (0, 1)]
    outs, kept = [], []
    for base in (0, pages - 5):
        k, v = (torch.empty(pages, kv_heads, page, D, dtype=torch.bfloat16, device="cuda") for _ in (0, 1)) if base else (s.clone() for s in small)
        if base:
            k[base:] = small[0]
            v[base:] = small[1]
        slots = torch.tensor([(table[i][t // page] + base) * page + t % page for i, t in places], dtype=torch.int64, device="cuda")
        q, _, _ = m.kv_append(ctx, qkv, q_heads, kv_heads, positions=positions, frequencies=freq, k_cache=k, v_cache=v, slots=slots)
        if base and T < 5:
            far = torch.empty(5 << 30, dtype=torch.bfloat16, device="cuda").as_strided((T, q_heads, D), (4 << 30, D, 1))
            far.copy_(q)
            q = far
        outs.append(m.paged_attention(ctx, q, k, v, starts, lens_dev, _ints(table) + base, max_new=max_new))
        kept.append((k[base:base + 5].clone(), v[base:base + 5].clone()))
        del k, v, q
    assert torch.equal(outs[0], outs[1]) and all(torch.equal(a, b) for a, b in zip(*kept))
    assert not torch.equal(kept[0][0], small[0])
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))


def test_more_work_than_a_call_may_have():
    """2^24 tokens of one prompt are 2^32 + 2^17 tiles with the units' ends: not 2^17.  Nothing is begun, and the status says why."""
    torch, m = _t(), _m()
    own = m.Context(0)
    rows = torch.zeros((1 << 24, 1, 64), dtype=torch.bfloat16, device="cuda")
    out = torch.ones_like(rows)
    m.prompt_attention(own, rows, rows, rows, _ints([0, 1 << 24]), out=out)
    with pytest.raises(m.MpqError) as e:
        own.check(own.lib.mpq_context_poll_status(own.h))
    assert e.value.status == m._lib.ERR_UNSUPPORTED and bool((out == 1).all())
    own.check(own.lib.mpq_context_poll_status(own.h))
    m.prompt_attention(own, rows[:300], rows[:300], rows[:300], _ints([0, 300]), out=out[:300])       # the context goes on
    own.check(own.lib.mpq_context_poll_status(own.h))
    assert bool((out[:300] == 0).all()) and bool((out[300:] == 1).all())


def test_two_contexts_at_once():
    """Calls of two contexts on two streams, beside each other: each has its own pieces and counters."""
    torch, m = _t(), _m()
    contexts = [m.Context(0), m.Context(0)]
    data, want = [], []
    for i, c in enumerate(contexts):
        k, v, table = _paged_case(10 * i, [1, 300], [5000, 4000], 2, 128, 16)
        q = _randn(20 + i, 301, 8, 128, dtype=torch.bfloat16)
        rows = [_randn(30 + i + j, 2000, h, 64, dtype=torch.bfloat16) for j, h in enumerate((8, 2, 2))]
        data.append((q, k, v, _ints([0, 1, 301]), _ints([5000, 4000]), _ints(table), rows, _ints([0, 700, 2000])))

    def run(c, d):
        return [m.paged_attention(c, d[0], *d[1:6]), m.paged_attention(c, d[0][:1].contiguous(), d[1], d[2], _ints([0, 1]), d[4][:1].contiguous(), d[5][:1].contiguous(), max_new=1),
                m.prompt_attention(c, *d[6], d[7])]
    for c, d in zip(contexts, data):
        want.append(run(c, d))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(contexts[i], data[i]))
    torch.cuda.synchronize()
    for i, c in enumerate(contexts):
        for g in got[i]:
            for a, b in zip(g, want[i]):
                assert torch.equal(a, b)
        c.check(c.lib.mpq_context_poll_status(c.h))


@pytest.mark.parametrize("kind", ["few", "many", "prompt"])
def test_a_first_call_inside_a_capture(kind):
    """Without room for pieces (none can be had in a capture) units stay whole: other last bits, the same attention."""
    torch, m = _t(), _m()
    ctx = m.Context(0)
    new, lens, D = ([1, 1, 1], [5000, 40, 0], 128) if kind == "few" else ([200, 1, 30], [3000, 700, 30], 128)
    k, v, table = _paged_case(1, new, lens, 2, D, 16)
    starts = [0, new[0], new[0] + new[1], sum(new)]
    q = _randn(2, sum(new), 8, D, dtype=torch.bfloat16)
    rows = [_randn(3 + j, 1500, h, D, dtype=torch.bfloat16) for j, h in enumerate((8, 2, 2))]
    args = (_ints(starts), _ints(lens), _ints(table))
    at = _ints([0, 1000, 1500])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = m.prompt_attention(ctx, *rows, at) if kind == "prompt" else m.paged_attention(ctx, q, k, v, *args, max_new=max(new))
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    if kind == "prompt":
        for a, b in ((0, 1000), (1000, 1500)):
            want, mass = _attention_reference(rows[0][a:b], rows[1][a:b], rows[2][a:b], D ** -0.5)
            assert _off(out[a:b], want, mass, D, D ** -0.5 * 16 ** 2) <= 1
    else:
        for i, (a, t) in enumerate(zip(new, lens)):
            want, mass = _attention_reference(q[starts[i]:starts[i + 1]], _gathered(k, table[i], t, 16), _gathered(v, table[i], t, 16), D ** -0.5)
            assert _off(out[starts[i]:starts[i + 1]], want, mass, D, D ** -0.5 * 16 ** 2) <= 1, i
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))
    ctx.close()


def test_scale_zero_and_wide_groups(ctx):
    """Equal weights; more query heads per head of keys than a tile has rows."""
    torch, m = _t(), _m()
    _check_paged(ctx, [1, 3, 200], [100, 700, 300], 4, 2, 64, 16, scale=0.0)
    _check_paged(ctx, [1, 5], [333, 40], 300, 1, 64, 16)
    _check_paged(ctx, [40], [400], 130, 1, 128, 32)
    q, k, v = _randn(1, 70, 272, 64, dtype=torch.bfloat16), _randn(2, 70, 1, 64, dtype=torch.bfloat16), _randn(3, 70, 1, 64, dtype=torch.bfloat16)
    got = m.prompt_attention(ctx, q, k, v, _ints([0, 3, 70]))
    for a, b in ((0, 3), (3, 70)):
        want, mass = _attention_reference(q[a:b], k[a:b], v[a:b], 0.125)
        assert _off(got[a:b], want, mass, 64, 0.125 * 13 ** 2) <= 1
