"""Outputs that lie over inputs are refused."""
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "overlap.h"
#include <cstdio>
#include <random>
#include <vector>
using namespace mpq;
int main()
{
    std::mt19937 rng(1);
    auto pick = [&](int a, int b) { return a + (int)(rng() % (unsigned)(b - a + 1)); };
    long bad = 0, yes = 0;
    auto at = [](long x) { return reinterpret_cast<const void*>((uintptr_t)x); };
    for (int trial = 0; trial < 200000; ++trial) {
        const int a = pick(1, 300), n = pick(0, 60), b = pick(1, 300), rows = pick(0, 6), w = pick(1, 20), s = w + pick(0, 40);
        bool want = false;
        for (int i = 0; i < rows; ++i) want |= n > 0 && a < b + i * s + w && b + i * s < a + n;
        yes += want;
        bad += overlaps(at(a), n, at(b), rows, w, s) != want;
        if (rows == 1) bad += overlaps(at(a), n, at(b), w) != want;
    }
    // far strides, and more rows than an address space holds
    bad += overlaps(at(1l << 40), 4096, at(1l << 39), 1l << 30, 512, (__int128)1 << 63);
    bad += !overlaps(at((1l << 39) + 3 * (1l << 33) + 511), 4096, at(1l << 39), 4, 512, (__int128)1 << 33);
    bad += overlaps(at((1l << 39) + 3 * (1l << 33) + 512), 4096, at(1l << 39), 4, 512, (__int128)1 << 33);
    bad += overlaps(nullptr, 4096, at(16), 4096) || overlaps(at(16), 4096, nullptr, 4096);
    std::printf("%ld\n", bad);
    return bad != 0 || yes < 1000;
}
"""


def test_overlaps():
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "t.cpp"), os.path.join(tmp, "t")
        open(src, "w").write(PROGRAM)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "makepad_b200", "csrc"), src, "-o", exe])
        out = subprocess.run([exe], capture_output=True, text=True)
        assert out.returncode == 0 and out.stdout.strip() == "0", out.stdout + out.stderr


def _bf16(*shape):
    import torch
    return torch.randn(shape, device="cuda").bfloat16()


def _refused(ctx, call):
    import makepad_b200 as m
    launches = ctx.launches
    with pytest.raises(m.MpqError) as e:
        call()
    assert e.value.status == m._lib.ERR_INVALID_ARG and ctx.launches == launches


@pytest.mark.gpu
def test_attention_does_not_write_over_what_it_reads(ctx):
    import makepad_b200 as m
    import torch
    T, D = 40, 64
    # rows of a projection, and out in memory behind, over and between them
    room = _bf16(4 * T * 8 * D)
    rows = room[:T * 8 * D].view(T, 8, D)
    q, k, v = rows.split([4, 2, 2], dim=1)
    starts = torch.tensor([0, 17, T], dtype=torch.int32, device="cuda")
    want = m.prompt_attention(ctx, q.clone(), k.clone(), v.clone(), starts)
    out = room[T * 8 * D:T * 12 * D].view(T, 4, D)
    assert torch.equal(m.prompt_attention(ctx, q, k, v, starts, out=out), want)
    packed = q.contiguous()
    for over in (packed, room[:T * 4 * D].view(T, 4, D), room[T * 8 * D - 8:T * 12 * D - 8].view(T, 4, D), room[4 * D:T * 4 * D + 4 * D].view(T, 4, D)):
        _refused(ctx, lambda: m.prompt_attention(ctx, packed if over is packed else q, k, v, starts, out=over))
    both = _bf16(2 * T * 4 * D)
    half = both[:T * 4 * D].view(T, 4, D)
    _refused(ctx, lambda: m.prompt_attention(ctx, half, k, v, starts, out=both.view(torch.float32).view(T, 4, D)))
    _refused(ctx, lambda: m.prompt_attention(ctx, packed, half[:, :2], v, starts, out=half))
    _refused(ctx, lambda: m.prompt_attention(ctx, packed, k, half[:, 2:], starts, out=half))
    # a row of out in the room between rows of q is none of them
    wide = _bf16(3, 4096)
    wq = wide[:, :256].unflatten(1, (4, D))
    one = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    kk = _bf16(3, 2, D)
    gap = wide.view(-1)[1024:1024 + 3 * 256].view(3, 4, D)
    assert torch.equal(m.prompt_attention(ctx, wq, kk, kk, one, out=gap), m.prompt_attention(ctx, wq.clone(), kk, kk, one))


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
def test_paged_attention_does_not_write_over_what_it_reads(ctx, max_new):
    import makepad_b200 as m
    import torch
    n, D, page = 6, 64, 16
    k, v, q = _bf16(8, 2, page, D), _bf16(8, 2, page, D), _bf16(n, 4, D)
    table = torch.arange(8, dtype=torch.int32, device="cuda")[:n].view(n, 1).repeat(1, 600).contiguous()
    starts, lens = torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.full((n,), 9, dtype=torch.int32, device="cuda")
    m.paged_attention(ctx, q, k, v, starts, lens, table, max_new=max_new)
    for over in (q, k.view(-1)[:n * 4 * D].view(n, 4, D), v.view(-1)[-n * 4 * D:].view(n, 4, D), table.view(-1)[-n * 2 * D:].view(torch.bfloat16).view(n, 4, D)):
        _refused(ctx, lambda: m.paged_attention(ctx, q, k, v, starts, lens, table, max_new=max_new, out=over))
    # lengths and starts inside of out
    words = torch.zeros(n * 4 * D // 2, dtype=torch.int32, device="cuda")
    words[100:100 + n] = 9
    words[200:200 + n + 1] = starts
    out = words.view(torch.bfloat16).view(n, 4, D)
    _refused(ctx, lambda: m.paged_attention(ctx, q, k, v, starts, words[100:100 + n], table, max_new=max_new, out=out))
    _refused(ctx, lambda: m.paged_attention(ctx, q, k, v, words[200:200 + n + 1], lens, table, max_new=max_new, out=out))


@pytest.mark.gpu
def test_norms_do_not_write_over_what_others_read(ctx):
    import makepad_b200 as m
    import torch
    M, H = 6, 64
    f32 = torch.float32

    def call(x, residual=None, residual_out=None, post=None, gate=None, stride=0, weight=None, y=None):
        p = lambda t: None if t is None else t.data_ptr()
        ctx.check(ctx.lib.mpq_residual_norm(ctx.h, p(x), x.dtype is torch.bfloat16, M, H, p(residual), p(residual_out), p(post), p(gate), stride, 0.5, p(weight), 1e-6,
                                            p(y), y is not None and y.dtype is torch.bfloat16, torch.cuda.current_stream().cuda_stream))
    x, r, w, gate = torch.randn(M, H, device="cuda"), torch.randn(M, H, device="cuda"), torch.randn(H, device="cuda"), torch.randn(M, 80, device="cuda")
    y = torch.empty(M, H, device="cuda")
    want_r, want_y = m.residual_norm(ctx, x, r, w, alpha=0.5, gate=gate[:, :H].contiguous())
    for out in (r.clone(), x.clone(), torch.empty_like(r)):                   # in place of the residual, or of x, or neither
        args = (out if torch.equal(out, x) else x, out if torch.equal(out, r) else r, out)
        call(*args, gate=gate, stride=80, weight=w, y=y)
        assert torch.equal(out, want_r) and torch.equal(y, want_y)
    both = torch.randn(8192, device="cuda")                                 # (a gate of six rows 1000 apart lies in it)
    at = lambda n, rows=M, wide=H: both[n:n + rows * wide].view(rows, wide)
    half = lambda n: both[n:].view(torch.bfloat16)[:M * H].view(M, H)
    for bad in (dict(x=at(0), y=at(0)), dict(x=at(0), y=at(M * H - 4)), dict(x=x, residual=at(0), y=at(64)), dict(x=x, residual_out=at(0), y=at(0)), dict(x=x, residual_out=at(0), y=half(M * H - 4)),
                dict(x=at(64), residual_out=at(0)), dict(x=x, residual=at(64), residual_out=at(0)), dict(x=half(0), residual_out=at(0)), dict(x=x, residual_out=at(0), post=both[M * H - 4:M * H + 60]),
                dict(x=x, residual_out=at(0), weight=both[:64]), dict(x=x, y=at(0), weight=both[M * H - 64:M * H]), dict(x=x, y=at(0), gate=both[60:], stride=0),
                dict(x=x, y=at(80), gate=both, stride=400), dict(x=x, residual_out=at(80, 1), y=at(8 * 80), gate=at(0), stride=80)):
        _refused(ctx, lambda: call(**bad))
    call(x, y=at(80), gate=both, stride=1000)                                 # rows of the gate on either side: 0..63 and 1000..1063, y 80..463
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_append_does_not_write_over_what_others_read(ctx):
    import torch
    T, D, pages, page = 5, 64, 2, 16
    room = torch.zeros(1 << 16, dtype=torch.bfloat16, device="cuda")
    at = lambda n: room[n:].data_ptr()
    positions, slots = torch.arange(T, dtype=torch.int32, device="cuda"), torch.arange(T, dtype=torch.int64, device="cuda")
    freq = torch.ones(D // 2, dtype=torch.float64, device="cuda")

    def call(qkv=0, bf16=1, stride=256, pos=positions.data_ptr(), f=freq.data_ptr(), q=8192, k=None, v=None, s=slots.data_ptr(), kc=16384, vc=24576):
        ctx.check(ctx.lib.mpq_kv_append(ctx.h, at(qkv), bf16, stride, T, 2, 1, D, pos, f, D, 0, at(q), None if k is None else at(k), None if v is None else at(v), s, at(kc), at(vc), pages, page,
                                        torch.cuda.current_stream().cuda_stream))
    call()
    call(k=32768, v=40960)
    call(stride=2048, q=256, k=2048 + 256, v=4096 + 256)                      # between the rows
    for bad in (dict(q=0), dict(q=1272), dict(bf16=0, q=2552), dict(stride=2048, q=8192), dict(k=8192 + 632), dict(k=9000, v=9312), dict(kc=8192), dict(vc=16384), dict(vc=16384 + 2040), dict(kc=1000),
                dict(pos=at(8192)), dict(f=at(16384)), dict(s=at(24576)), dict(s=at(8192 + 632)), dict(k=16384 + 2000), dict(v=24576 - 296)):
        _refused(ctx, lambda: call(**bad))
    torch.cuda.synchronize()
