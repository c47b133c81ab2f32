"""Norms at the borders between the kernels' variants: columns per thread and rows on an SM."""
import pytest

from test_decoder_ops_gpu import B, _norm_reference, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 148, 149, 296, 297, 400, 2368, 2369])
@pytest.mark.parametrize("H", [4096, 4104, 5120, 5128, 8192, 8200])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_rows_and_columns_at_the_borders(ctx, M, H, kind):
    import makepad_b200 as m
    import torch
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    x, residual, weight, post, gate = _randn(1, M, H, dtype=dtype), _randn(2, M, H) * 3, 1 + _randn(3, H) * 0.2, 1 + _randn(4, H) * 0.2, _randn(5, H)
    r, y = m.residual_norm(ctx, x, residual, weight, eps=1e-5, alpha=0.25, post_weight=post, gate=gate, out_dtype=dtype)
    want_r, r_off, want_y, y_off = _norm_reference(x, residual, weight, post, gate, 0.25, 1e-5)
    assert bool(((r.double() - want_r).abs() <= r_off).all())
    y_off = y_off + (B * want_y.abs() + 2.0 ** -134 if kind == "bf16" else 0)
    assert bool(((y.double() - want_y).abs() <= y_off * (1 + 2 ** -7)).all())
    again = m.residual_norm(ctx, x, residual, weight, eps=1e-5, alpha=0.25, post_weight=post, gate=gate, out_dtype=dtype)
    assert torch.equal(again[0], r) and torch.equal(again[1], y)
