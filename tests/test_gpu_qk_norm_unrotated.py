"""Columns that are not rotated (past R, or of a token at a negative position) do not depend on each other: an infinity
or NaN that a weight or a gradient has in one of them stays there."""

import math

import pytest
import torch

import kv_reference as ref
from conftest import cpu_randn

pytestmark = pytest.mark.gpu


def inputs(dev, dtype, d):
    from low_bit_fake_quant import rotary_table
    q, k = cpu_randn(6, 3, d, seed=1, dtype=dtype).to(dev), cpu_randn(6, 2, d, seed=2, dtype=dtype).to(dev)
    w = (1 + 0.3 * cpu_randn(2, d, seed=3, dtype=torch.float32)).to(dev)
    cos, sin = rotary_table(6, d // 2, device=dev)
    pos = torch.tensor([0, 3, -1, 5, -7, 2], device=dev)
    return q, k, w[0], w[1], cos, sin, pos


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float32), (128, torch.float16)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_weight_that_is_not_finite(gpu, bad, d, dtype, pairs):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, wk, cos, sin, pos = inputs(gpu, dtype, d)
    clean = qk_norm_rope(q, k, wq, wk, cos, sin, pos, pairs=pairs)
    for col in (d // 2 + 5, d - 1, 2):  # two that are never rotated, one only of padding
        wb = wq.clone()
        wb[col] = bad
        y, _ = qk_norm_rope(q, k, wb, wk, cos, sin, pos, pairs=pairs)
        rows = pos < 0 if col == 2 else torch.ones_like(pos, dtype=torch.bool)
        other = torch.arange(d, device=gpu) != col
        assert torch.equal(y[rows][..., other], clean[0][rows][..., other]), col
        got = y[rows][..., col].double()
        # (no value of q is 0)
        assert torch.isnan(got).all() if math.isnan(bad) else torch.equal(got, torch.sign(q[rows][..., col].double()) * bad)


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float32)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_gradient_that_is_not_finite_reaches_its_own_column_of_the_weights(gpu, bad, d, dtype, pairs):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, wk, cos, sin, pos = inputs(gpu, dtype, d)
    for token, col in ((1, d // 2 + 5), (2, d // 2 + 4), (2, 3)):  # (token 2 is padding)
        leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
        y = qk_norm_rope(*leaves, cos, sin, pos, pairs=pairs)
        dy = [torch.ones_like(t) for t in y]
        plain = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        dy[0][token, 1, col] = bad
        got = torch.autograd.grad(y, leaves, dy)
        other = torch.arange(d, device=gpu) != col
        assert torch.equal(got[2][other], plain[2][other]) and not torch.isfinite(got[2][col]), (token, col)
        assert torch.equal(got[1], plain[1]) and torch.equal(got[3], plain[3])
        rest = torch.ones(q.shape[:2], dtype=torch.bool, device=gpu)
        rest[token, 1] = False
        assert torch.equal(got[0][rest], plain[0][rest])
        assert not torch.isfinite(got[0][token, 1, col])


def test_unrotated_columns_are_the_norm(gpu):
    q, k, wq, wk, cos, sin, pos = inputs(gpu, torch.float32, 128)
    from low_bit_fake_quant import qk_norm_rope
    y, _ = qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    r = 1 / (q.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    want = q.double() * r * wq.double()
    for got, w in ((y[..., 64:], want[..., 64:]), (y[pos < 0], want[pos < 0])):
        # 16 additions halved by the root, the reciprocal root, two products and the rounding: under 32 * 2^-24
        ref.check(got, w, 32 * 2.0 ** -24 * w.abs(), "unrotated")
