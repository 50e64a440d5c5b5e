"""Q/K norm with rotation, forward and backward, against the formulas in 64 bits.

Bounds.  Forward: the output's rounding u |y|, and fp32 arithmetic before it: the
sum of squares (up to 16 additions deep: 2^-24 each, halved by the root), the
reciprocal root (2^-23), two products and two of the rotation: under 32 * 2^-24
of |n_a| + |n_b|.  Backward dx: the same for dy's rotation, times the two sums of
up to 16 deep: under 64 * 2^-24 of r (|g w| + |xhat| mean |g w xhat|).  Weights: every
term is off by under 16 * 2^-24 of itself, and the sums by up to 512 * 2^-24 of the sum
of magnitudes (fp32 over the rows of a wave, then 64 bits), then one rounding."""

import math

import pytest
import torch

import kv_reference as ref
from conftest import cpu_randn

pytestmark = pytest.mark.gpu

EPS = 1e-6


def case(dev, B, S, hq, hk, d, dtype, wdtype=torch.float32, rot=None, seed=0, far=1000):
    from low_bit_fake_quant import rotary_table
    q, k = cpu_randn(B, S, hq, d, seed=seed, dtype=dtype).to(dev), cpu_randn(B, S, hk, d, seed=seed + 1, dtype=dtype).to(dev)
    wq, wk = ((1 + 0.3 * cpu_randn(d, seed=seed + s, dtype=torch.float32)).to(wdtype).to(dev) for s in (2, 3))
    cos, sin = rotary_table(S + far, rot or d, device=dev)
    pos = torch.randint(0, S + far, (B, S), generator=torch.Generator().manual_seed(seed + 4)).to(dev)
    return q, k, wq, wk, cos, sin, pos


def check_forward(x, w, y, cos, sin, pos, pairs):
    c, s = cos.double()[pos], sin.double()[pos]
    x64, w64 = x.detach().double(), None if w is None else w.detach().double()
    want = ref.norm_rope(x64, w64, c, s, pairs, EPS)
    one = torch.ones_like(c)
    size = ref.norm_rope(x64.abs(), None if w is None else w64.abs(), one, -one, pairs, EPS).abs() \
        + ref.norm_rope(x64.abs(), None if w is None else w64.abs(), one, one, pairs, EPS).abs()
    tiny = 2.0 ** -24 if y.dtype == torch.float16 else 0.0
    ref.check(y.detach(), want, ref.U[y.dtype] * want.abs() + 32 * 2.0 ** -24 * size + tiny, "forward")


SHAPES = [(1, 1, 1, 1, 64), (3, 5, 7, 2, 128), (1, 130, 12, 12, 128), (2, 33, 5, 1, 64), (24, 1, 32, 8, 128),
          (1, 8200, 3, 2, 64)]


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(gpu, shape, dtype, pairs):
    from low_bit_fake_quant import qk_norm_rope
    B, S, hq, hk, d = shape
    for rot in (d, d // 2, 16):
        q, k, wq, wk, cos, sin, pos = case(gpu, B, S, hq, hk, d, dtype, rot=rot)
        yq, yk = qk_norm_rope(q, k, wq, wk, cos, sin, pos, pairs=pairs)
        assert yq.shape == q.shape and yk.dtype == dtype and yq.is_contiguous()
        check_forward(q, wq, yq, cos, sin, pos, pairs)
        check_forward(k, wk, yk, cos, sin, pos, pairs)


def gradients(args, dyq, dyk, **kw):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, wk = (t.detach().requires_grad_() for t in args[:4])
    yq, yk = qk_norm_rope(q, k, wq, wk, *args[4:], **kw)
    return torch.autograd.grad((yq, yk), (q, k, wq, wk), (dyq, dyk))


def check_gradient(x, w, dy, dx, dw, cos, sin, pos, pairs):
    c, s = cos.double()[pos], sin.double()[pos]
    x, w, dy = x.detach().double(), w.detach().double(), dy.double()
    want, wdw, mag = ref.norm_rope_grad(x, w, dy, c, s, pairs, EPS)
    r = 1.0 / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    one = torch.ones_like(c)
    turned = (ref.rotate(dy.abs(), one[..., None, :], one[..., None, :], pairs).abs()
              + ref.rotate(dy.abs(), one[..., None, :], one[..., None, :], pairs, back=True).abs()) * w.abs()
    size = r * (turned + (x * r).abs() * (turned * (x * r).abs()).mean(-1, keepdim=True))
    tiny = 2.0 ** -24 if dx.dtype == torch.float16 else 0.0
    ref.check(dx, want, ref.U[dx.dtype] * want.abs() + 64 * 2.0 ** -24 * size + tiny, "dx")
    mag2 = (turned / w.abs().clamp_min(1e-30) * (x * r).abs()).flatten(0, -2).sum(0)
    ref.check(dw, wdw, ref.U[dw.dtype] * wdw.abs() + 528 * 2.0 ** -24 * mag2, "dw")


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float32, torch.bfloat16)], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(gpu, shape, dtype, wdtype, pairs):
    B, S, hq, hk, d = shape
    for rot in (d, 32):
        args = case(gpu, B, S, hq, hk, d, dtype, wdtype, rot=rot, seed=5)
        dyq, dyk = (cpu_randn(*t.shape, seed=s, dtype=dtype).to(gpu) for t, s in ((args[0], 8), (args[1], 9)))
        dq, dk, dwq, dwk = gradients(args, dyq, dyk, pairs=pairs)
        q, k, wq, wk, cos, sin, pos = args
        check_gradient(q, wq, dyq, dq, dwq, cos, sin, pos, pairs)
        check_gradient(k, wk, dyk, dk, dwk, cos, sin, pos, pairs)
        again = gradients(args, dyq, dyk, pairs=pairs)
        assert all(torch.equal(a, b) for a, b in zip(again, (dq, dk, dwq, dwk)))  # a fixed order


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_gradient_against_differences(gpu, pairs):
    """Central differences of the 64-bit forward along random directions, h = 1e-4: their
    own error is h^2 / 6 of a third derivative of order 10 (2e-8) and 1e-12 of rounding;
    the fp32 gradient's 64 * 2^-24 = 4e-6 of the sum of |dx d| bounds the rest."""
    args = case(gpu, 1, 4, 3, 2, 64, torch.float32)
    q, k, wq, wk, cos, sin, pos = args
    dyq, dyk = (cpu_randn(*t.shape, seed=s, dtype=torch.float32).to(gpu) for t, s in ((q, 8), (k, 9)))
    grads = gradients(args, dyq, dyk, pairs=pairs)
    c, s = cos.double()[pos], sin.double()[pos]

    def loss(v):
        return ((ref.norm_rope(v[0], v[2], c, s, pairs, EPS) * dyq).sum()
                + (ref.norm_rope(v[1], v[3], c, s, pairs, EPS) * dyk).sum())

    base = [t.double() for t in (q, k, wq, wk)]
    for which in range(4):
        for seed in range(3):
            dirs = [torch.zeros_like(t) for t in base]
            dirs[which] = cpu_randn(*base[which].shape, seed=seed, dtype=torch.float64).to(gpu)
            h = 1e-4
            diff = (loss([a + h * b for a, b in zip(base, dirs)]) - loss([a - h * b for a, b in zip(base, dirs)])) / (2 * h)
            got = (grads[which].double() * dirs[which]).sum()
            bound = 1e-5 * (1 + (grads[which].double() * dirs[which]).abs().sum())
            assert (got - diff).abs() <= bound


def test_layouts_broadcasts_and_one_weight_for_both(gpu):
    from low_bit_fake_quant import qk_norm_rope
    B, S, hq, hk, d = 2, 9, 6, 2, 128
    q, k, wq, wk, cos, sin, pos = case(gpu, B, S, hq, hk, d, torch.bfloat16)
    want = qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    packed = torch.cat([q, k, k], 2)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=gpu)[1:].view(q.shape).copy_(q)
    strided = k.transpose(2, 3).contiguous().transpose(2, 3)
    heads = q.transpose(1, 2).contiguous().transpose(1, 2)
    for a, b, p in ((packed[:, :, :hq], packed[:, :, hq:hq + hk], pos.int()), (odd, strided, pos), (heads, k, pos)):
        got = qk_norm_rope(a, b, wq, wk, cos, sin, p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = qk_norm_rope(q.flatten(0, 1), k.flatten(0, 1), wq, wk, cos, sin, pos.flatten())
    assert torch.equal(got[0].view(q.shape), want[0]) and torch.equal(got[1].view(k.shape), want[1])
    at = torch.arange(S, device=gpu)
    for p in (None, at, at.expand(B, S)):
        got = qk_norm_rope(q, k, None, None, cos, sin, p)
        check_forward(q, None, got[0], cos, sin, at.expand(B, S), "adjacent")
        check_forward(k, None, got[1], cos, sin, at.expand(B, S), "adjacent")

    # one row for the whole batch, one weight for Q and K, expanded gradients: each leaf gets the sum
    row = q[:1, :, :1].detach().float().requires_grad_()
    w = wq.detach().clone().requires_grad_()
    yq, yk = qk_norm_rope(row.expand(B, S, hq, d), row.expand(B, S, hk, d), w, w, cos, sin, pos)
    (yq.sum() + 2 * yk.sum()).backward()
    c, s = cos.double()[pos], sin.double()[pos]
    x = row.detach().double()
    parts = [ref.norm_rope_grad(x.expand(B, S, h, d), w.detach().double(),
                                torch.full((B, S, h, d), g, dtype=torch.float64, device=gpu), c, s, "adjacent", EPS)
             for h, g in ((hq, 1.0), (hk, 2.0))]
    dx = sum(p[0].sum((0, 2), keepdim=True) for p in parts)
    size = sum(p[0].abs().sum((0, 2), keepdim=True) for p in parts) + 1
    ref.check(row.grad, dx, 128 * 2.0 ** -24 * size, "broadcast dx")
    ref.check(w.grad, sum(p[1] for p in parts), 600 * 2.0 ** -24 * (sum(p[2] for p in parts) + 1), "shared dw")


def test_only_what_is_asked_for(gpu):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, wk, cos, sin, pos = case(gpu, 1, 6, 4, 4, 64, torch.float32)
    all_ = gradients((q, k, wq, wk, cos, sin, pos), q, torch.zeros_like(k))
    x = q.detach().clone().requires_grad_()
    y, yk = qk_norm_rope(x, k, wq, wk, cos, sin, pos)
    (g,) = torch.autograd.grad(y, x, q)  # K's output is not used
    assert torch.equal(g, all_[0])
    w = wq.detach().clone().requires_grad_()
    (g,) = torch.autograd.grad(qk_norm_rope(q, k, w, None, cos, sin, pos)[0], w, q)
    assert torch.equal(g, all_[2])
    zero = gradients((q, k, wq, wk, cos, sin, pos), torch.zeros_like(q), k)
    w = wk.detach().clone().requires_grad_()
    (g,) = torch.autograd.grad(qk_norm_rope(q, k, None, w, cos, sin, pos)[1], w, k)  # the first weight is not given
    assert torch.equal(g, zero[3])
    with torch.no_grad():
        assert not qk_norm_rope(x, k, w, wk, cos, sin, pos)[0].requires_grad


def test_a_second_derivative_is_refused(gpu):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, _, cos, sin, pos = case(gpu, 1, 6, 4, 4, 64, torch.float32)
    q.requires_grad_()
    wq.requires_grad_()
    yq, yk = qk_norm_rope(q, k, wq, None, cos, sin, pos)
    (plain,) = torch.autograd.grad(yq.square().sum() + yk.sum(), q, retain_graph=True)
    (g,) = torch.autograd.grad(yq.square().sum() + yk.sum(), q, create_graph=True)
    assert torch.equal(g, plain)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_backward_on_a_side_stream_and_in_threads(gpu):
    """The backward pass runs on the forward's stream, in autograd's own thread, from several callers at once."""
    import threading
    args = case(gpu, 2, 300, 6, 2, 128, torch.bfloat16)
    dq, dk = torch.ones_like(args[0]), torch.ones_like(args[1])
    want = gradients(args, dq, dk)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream(device=gpu)
        with torch.cuda.stream(s):
            for _ in range(20):
                got = gradients(args, dq, dk)
                s.synchronize()
                bad.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_padding_positions_and_positions_past_the_table(gpu):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, wk, cos, sin, pos = case(gpu, 1, 5, 2, 2, 64, torch.float32, rot=32)
    pos[0, 1], pos[0, 3] = -1, cos.shape[0]
    yq, yk = qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    n = q.double() / (q.double().square().mean(-1, keepdim=True) + EPS).sqrt() * wq.double()
    ref.check(yq[0, 1], n[0, 1], 32 * 2.0 ** -24 * n[0, 1].abs(), "not rotated")
    assert torch.isnan(yq[0, 3, :, :32]).all() and torch.isfinite(yq[0, 3, :, 32:]).all()
    assert torch.isfinite(yq[0, [0, 1, 2, 4]]).all() and torch.isfinite(yk[0, [0, 1, 2, 4]]).all()


def test_zero_rows_and_empty_calls(gpu):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, wk, cos, sin, pos = case(gpu, 1, 4, 2, 1, 128, torch.bfloat16)
    q.zero_()
    dq, dk, dwq, dwk = gradients((q, k, wq, wk, cos, sin, pos), torch.ones_like(q), torch.ones_like(k))
    assert torch.isfinite(dq.float()).all() and not dwq.any()
    assert not qk_norm_rope(q, k, wq, wk, cos, sin, pos)[0].any()
    e, f = q[:, :0], k[:, :0]
    dq, dk, dwq, dwk = gradients((e, f, wq, wk, cos, sin, pos[:, :0]), e, f)
    assert dq.shape == e.shape and not dwq.any() and not dwk.any()


def test_graph_replays_of_a_training_step(gpu):
    """Forward and backward captured together, replayed on new inputs between eager
    calls (of other leaves: an eager graph of the captured ones may not live then)."""
    from low_bit_fake_quant import qk_norm_rope
    args = case(gpu, 2, 40, 6, 2, 128, torch.bfloat16)
    dyq, dyk = torch.ones_like(args[0]), torch.ones_like(args[1])

    def step(leaves):
        yq, yk = qk_norm_rope(*leaves, *args[4:])
        return (yq, yk) + torch.autograd.grad((yq, yk), leaves, (dyq, dyk))

    fresh = lambda: tuple(t.detach().clone().requires_grad_() for t in args[:4])  # noqa: E731
    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream(gpu).wait_stream(side)
    torch.cuda.synchronize()
    leaves = fresh()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = [t.detach() for t in step(leaves)]
    for rep in range(4):
        for i in (0, 1, 2):
            new = cpu_randn(*leaves[i].shape, seed=30 + 4 * rep + i, dtype=torch.float32).to(leaves[i].dtype).to(gpu)
            args[i].copy_(new)
            leaves[i].data.copy_(new)
        g.replay()
        want = step(fresh())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), rep


def test_refusals(gpu):
    from low_bit_fake_quant import qk_norm_rope, rotary_table
    q, k, wq, wk, cos, sin, pos = case(gpu, 2, 5, 4, 2, 64, torch.bfloat16)
    bad = [
        (dict(q=q[0]), ValueError, "both be"), (dict(q=q.cpu(), k=k.cpu()), ValueError, "one CUDA device"),
        (dict(k=k.float()), TypeError, "one dtype"), (dict(q=q.double(), k=k.double()), TypeError, "unsupported dtype"),
        (dict(q=q[..., :32], k=k[..., :32]), ValueError, "D must be"), (dict(k=k[:, :4]), ValueError, "must agree"),
        (dict(k=k[:, :, :0]), ValueError, "must agree"),
        (dict(wq=wq[:3]), ValueError, "q_weight must have"), (dict(wk=wk.cpu()), ValueError, "k_weight must live"),
        (dict(cos=cos[:, :4], sin=sin[:, :4]), ValueError, "multiple of 16"), (dict(cos=cos.double()), TypeError, "float32"),
        (dict(sin=sin[:3]), ValueError, "cos and sin must be"), (dict(cos=cos.cpu(), sin=sin.cpu()), ValueError, "live on"),
        (dict(pos=pos.float()), TypeError, "positions must be int32"), (dict(pos=pos[:1]), ValueError, "positions must have"),
        (dict(pos=pos.cpu()), ValueError, "positions must live"),
        (dict(pos=None, cos=cos[:4], sin=sin[:4]), ValueError, "the table has 4"),
    ]
    names = ("q", "k", "wq", "wk", "cos", "sin", "pos")
    for kw, err, msg in bad:
        with pytest.raises(err, match=msg):
            qk_norm_rope(*(kw.get(n, x) for n, x in zip(names, (q, k, wq, wk, cos, sin, pos))))
    with pytest.raises(ValueError, match="pairs must be"):
        qk_norm_rope(q, k, wq, wk, cos, sin, pos, pairs="neither")
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rope(q, k, wq, wk, cos, sin, pos, eps=math.nan)
    with pytest.raises(ValueError, match="no gradient for cos"):
        qk_norm_rope(q, k, wq, wk, cos.requires_grad_(), sin, pos)
    with pytest.raises(ValueError, match="rot must be"):
        rotary_table(4, 3)
    x = q.detach().requires_grad_()
    y, _ = qk_norm_rope(x, k, wq, wk, cos.detach(), sin, pos)
    (g,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()  # no second derivative
