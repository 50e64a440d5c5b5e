"""Q/K norm where mean(x^2) + eps lies below fp32's normal numbers: rows of zeros or of tiny values with an eps of
next to nothing, or none.

Bounds: those of test_gpu_qk_norm, and what sums below the normal numbers lose: each of D squares and additions is off by
up to 2^-150, and the mean by as much, together 2 * 2^-150 of v = mean + eps; the root halves that relative to v."""

import pytest
import torch

import kv_reference as ref
from conftest import cpu_randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size,eps", [(1e-19, 0.0), (1e-20, 0.0), (3e-21, 0.0), (1e-20, 1e-40), (1e-25, 1e-40), (1e-25, 1e-38),
                                      (1e-19, 1e-38), (1e-17, 1e-38)])
def test_tiny_rows(gpu, size, eps, d, dtype, pairs):
    from low_bit_fake_quant import qk_norm_rope, rotary_table
    S = 7
    cos, sin = rotary_table(S, d, device=gpu)
    x = [(cpu_randn(S, h, d, seed=h, dtype=torch.float32) * size).to(dtype).to(gpu).requires_grad_() for h in (3, 1)]
    w = (1 + 0.3 * cpu_randn(d, seed=9, dtype=torch.float32)).to(gpu).requires_grad_()
    y = qk_norm_rope(x[0], x[1], w, None, cos, sin, eps=eps, pairs=pairs)
    dy = [cpu_randn(*t.shape, seed=5 + i, dtype=torch.float32).to(dtype).to(gpu) for i, t in enumerate(y)]
    got = torch.autograd.grad(y, [*x, w], dy)
    e = float(torch.tensor(eps, dtype=torch.float32))
    c, s = cos.double(), sin.double()
    one = torch.ones_like(c)
    for i, ww in ((0, w.detach().double()), (1, None)):
        t = x[i].detach().double()
        v = t.square().mean(-1, keepdim=True) + e
        lost = 2.0 ** -150 / v
        want = ref.norm_rope(t, ww, c, s, pairs, e)
        sizes = [ref.norm_rope(t.abs(), ww, one, o, pairs, e).abs() for o in (one, -one)]
        ref.check(y[i].detach(), want, ref.U[dtype] * want.abs() + (32 * 2.0 ** -24 + lost) * (sizes[0] + sizes[1]), "forward")
        dx, dw, mag = ref.norm_rope_grad(t, ww, dy[i].double(), c, s, pairs, e)
        r = 1 / v.sqrt()
        g = sum(ref.rotate(dy[i].double().abs(), one[:, None], o[:, None], pairs) .abs() for o in (one, -one))
        g = g if ww is None else g * ww.abs()
        # (three factors r)
        bound = (64 * 2.0 ** -24 + 3 * lost) * r * (g + t.abs() * r * (g * t.abs() * r).mean(-1, keepdim=True))
        ref.check(got[i], dx, ref.U[dtype] * dx.abs() + bound, "dx")
        if i == 0:
            terms = (g / ww.abs() * t.abs() * r).flatten(0, -2)
            ref.check(got[2], dw, 2.0 ** -24 * dw.abs() + (528 * 2.0 ** -24 + lost.max()) * terms.sum(0), "dw")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("eps", [1e-45, 1e-40, 1e-38, 1e-6])
def test_zeros_stay_zeros(gpu, eps, dtype):
    from low_bit_fake_quant import qk_norm_rope, rotary_table
    cos, sin = rotary_table(3, 64, device=gpu)
    x = torch.zeros(3, 2, 64, dtype=dtype, device=gpu)
    q, k = qk_norm_rope(x, x, None, None, cos, sin, eps=eps)
    assert not q.any() and not k.any()
