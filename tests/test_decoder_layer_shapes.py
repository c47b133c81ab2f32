"""What a decoder layer refuses before anything is launched."""
from types import SimpleNamespace

import pytest


def _layer(q_heads, kv_heads, D, fmt=None):
    import makepad_b200 as m
    H, F = 256, 512
    shapes = (((q_heads + 2 * kv_heads) * D, H), (H, q_heads * D), (2 * F, H), (H, F))
    return m.DecoderLayer(*(SimpleNamespace(ctx=None, w=SimpleNamespace(fmt=fmt or m._lib.FMT_Q4, N=n, K=k)) for n, k in shapes), None, None, q_heads=q_heads, kv_heads=kv_heads, frequencies=())


@pytest.mark.parametrize("heads", [(4, 4, 64), (4, 1, 128), (6, 2, 64)])
def test_heads_that_the_attention_has(heads):
    l = _layer(*heads)
    assert (l.q_heads, l.kv_heads, l.head_dim) == heads


@pytest.mark.parametrize("heads", [(4, 4, 32), (4, 2, 96), (2, 1, 80), (2, 2, 256), (3, 2, 64), (2, 4, 64), (4, 0, 64), (4, -1, 64)])
def test_heads_that_it_has_not_are_refused_by_the_constructor(heads):
    import makepad_b200 as m
    with pytest.raises(m.MpqError) as e:
        _layer(*heads)
    assert e.value.status == m._lib.ERR_SHAPE
