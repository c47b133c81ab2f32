"""The number of requests of an attention call: arithmetic on the host, and the calls at the limit."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "attention_plan.h"
#include <cstdio>
#include <initializer_list>
using namespace mpq;
int main()
{
    // every accepted number of requests lies in the entries, each of which has some of them; no int overflows on the way
    long bad = 0;
    static_assert(ATTN_MOST_REQUESTS + ATTN_ENTRIES < (1ll << 31), "attn_per adds them");
    for (int64_t n : {int64_t(1), int64_t(ATTN_ENTRIES), int64_t(ATTN_ENTRIES + 1), int64_t(99999), int64_t(ATTN_MOST_REQUESTS - 1), int64_t(ATTN_MOST_REQUESTS)}) {
        const int64_t per = attn_per((int)n);
        if (per < 1 || per * ATTN_ENTRIES < n || (per - 1) * ATTN_ENTRIES >= n) ++bad;
    }
    std::printf("%ld\n", bad);
    return bad != 0;
}
"""


def test_requests_fit_their_entries():
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "t.cpp"), os.path.join(tmp, "t")
        open(src, "w").write(PROGRAM)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-I",
                               os.path.join(ROOT, "makepad_b200", "csrc"), src, "-o", exe])
        out = subprocess.run([exe], capture_output=True, text=True)
        assert out.returncode == 0 and out.stdout.strip() == "0", out.stdout + out.stderr


def _rows(seed, *shape):
    import torch
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).bfloat16()


MOST = 1 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31 - 200, 2 ** 31 - 1, 2 ** 40])
def test_more_requests_than_a_call_may_have_are_refused(ctx, n):
    """On the host: arrays of that length need not be there."""
    import makepad_b200 as m
    import torch
    q, starts = _rows(1, 4, 2, 64), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    cache, out = _rows(2, 2, 2, 16, 64), torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    launches = ctx.launches
    with pytest.raises(m.MpqError) as e:
        ctx.check(ctx.lib.mpq_prompt_attention(ctx.h, q.data_ptr(), 128, q.data_ptr(), 128, q.data_ptr(), 128, 4, 2, 2, 64, n, starts.data_ptr(), 0.125, out.data_ptr(), 0, stream))
    assert e.value.status == m._lib.ERR_UNSUPPORTED
    with pytest.raises(m.MpqError) as e:
        ctx.check(ctx.lib.mpq_paged_attention(ctx.h, q.data_ptr(), 128, 4, 2, cache.data_ptr(), cache.data_ptr(), 2, 16, 2, 64, n, starts.data_ptr(), starts.data_ptr(), starts.data_ptr(), 1, 1,
                                              0.125, out.data_ptr(), 0, stream))
    assert e.value.status == m._lib.ERR_UNSUPPORTED
    assert ctx.launches == launches and bool((out == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("with_rows", [{0: 300, MOST - 1: 40}, {0: 1, 31: 2, 32: 5, 64: 1, 777777: 200, 777778: 1, MOST - 2: 3}])
def test_as_many_requests_as_a_call_may_have(ctx, with_rows):
    """Nearly all of them without tokens: what the others get is what they get alone."""
    import makepad_b200 as m
    import torch
    new = torch.zeros(MOST + 1, dtype=torch.int64)
    for i, k in with_rows.items():
        new[i + 1] = k
    starts, T = new.cumsum(0).int().cuda(), sum(with_rows.values())
    few = torch.tensor([0] + list(with_rows.values())).cumsum(0).int().cuda()
    q, k, v = _rows(1, T, 4, 64), _rows(2, T, 2, 64), _rows(3, T, 2, 64)
    f32 = torch.float32
    got, want = m.prompt_attention(ctx, q, k, v, starts, out_dtype=f32), m.prompt_attention(ctx, q, k, v, few, out_dtype=f32)
    # units may be cut elsewhere, and weights that stand against another maximum are rounded to bf16 anew: 2^-8 on either side, of values that are at most 5;
    # sums of 300 keys in fp32, in another order, stay far below that
    near = lambda a, b: bool(((a - b).abs() <= 2 * 2 ** -8 * 5).all())
    assert near(got, want)
    # a cache in which each of them has a page, or for the long ones enough
    lens = torch.zeros(MOST, dtype=torch.int32)
    for i, count in with_rows.items():
        lens[i] = max(1, min(count, 32))
    table = torch.zeros(MOST, 2, dtype=torch.int32)
    for j, i in enumerate(with_rows):
        table[i, 0], table[i, 1] = 2 * j, 2 * j + 1
    cache = [_rows(4 + j, 2 * len(with_rows), 2, 16, 64) for j in (0, 1)]
    ids = list(with_rows)
    for max_new in (0, 1):
        got = m.paged_attention(ctx, q, *cache, starts, lens.cuda(), table.cuda(), max_new=max_new, out_dtype=f32)
        want = m.paged_attention(ctx, q, *cache, few, lens[ids].cuda(), table[ids].contiguous().cuda(), max_new=max_new, out_dtype=f32)
        assert near(got, want)
    ctx.check(ctx.lib.mpq_context_poll_status(ctx.h))
