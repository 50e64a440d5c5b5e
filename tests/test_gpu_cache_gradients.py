"""What the cache operators do with inputs that ask for a derivative which they do not form: they say so."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_paged_attention import problem

pytestmark = pytest.mark.gpu


def norm_inputs(dev):
    from low_bit_fake_quant import rotary_table
    g = torch.Generator().manual_seed(0)
    x = [torch.randn(5, h, 64, generator=g).to(dev) for h in (4, 2)] + [torch.randn(64, generator=g).to(dev) for _ in (0, 1)]
    return x + list(rotary_table(5, 64, device=dev))


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("also_backward", [False, True])
def test_norm_refuses_tangents(gpu, which, also_backward):
    """q, k, the weights and the table, also where another input has a gradient of the ordinary kind."""
    from low_bit_fake_quant import qk_norm_rope
    x = norm_inputs(gpu)
    if also_backward:
        x[1 if which == 0 else 0].requires_grad_()
    with forward_ad.dual_level():
        x[which] = forward_ad.make_dual(x[which].detach(), torch.ones_like(x[which]))
        for mode in (torch.enable_grad, torch.no_grad):  # (no_grad leaves forward mode on)
            with mode(), pytest.raises(ValueError, match="forward-mode"):
                qk_norm_rope(*x)
        with forward_ad._set_fwd_grad_enabled(False):
            qk_norm_rope(*x)
    # behind the level there is no tangent any more
    qk_norm_rope(*x)


def test_cache_calls_refuse_tangents(gpu):
    from low_bit_fake_quant import paged_attention, write_kv_cache
    q, cache, table, lens, starts = problem(gpu, lens=[20], counts=[2])
    k = torch.randn(2, 2, 128, device=gpu)
    slots = torch.arange(2, device=gpu)
    before = [t.view(torch.uint8).clone() for t in cache]
    with forward_ad.dual_level(), torch.no_grad():
        dk, dq = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (k, q))
        out = forward_ad.make_dual(torch.zeros_like(q), torch.ones_like(q))
        for call in (lambda: write_kv_cache(dk, k, cache, slots), lambda: write_kv_cache(k, dk, cache, slots),
                     lambda: paged_attention(dq, cache, table, lens, starts),
                     lambda: paged_attention(q, cache, table, lens, starts, out=out)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b)


def test_function_transforms_are_refused(gpu):
    from low_bit_fake_quant import qk_norm_rope
    q, k, wq, wk, cos, sin = norm_inputs(gpu)
    f = lambda q: qk_norm_rope(q, k, wq, wk, cos, sin)[0].sum()  # noqa: E731
    for call in (lambda: torch.func.grad(f)(q), lambda: torch.func.jvp(f, (q,), (q,)), lambda: torch.func.vmap(f)(q[None])):
        with pytest.raises((RuntimeError, ValueError)):
            call()


def test_a_cache_write_counts_as_a_change_in_place(gpu):
    """A backward pass that needs what a cache tensor held before says so."""
    from low_bit_fake_quant import empty_kv_cache, write_kv_cache
    cache = empty_kv_cache(2, 16, 2, 64, device=gpu)
    k, slots = torch.randn(3, 2, 64, device=gpu), torch.arange(3, device=gpu)
    w = torch.ones(cache.k_scale.shape, device=gpu, requires_grad=True)
    y = (w * cache.k_scale).sum()
    versions = [t._version for t in cache]
    write_kv_cache(k[:0], k[:0], cache, slots[:0])
    assert [t._version for t in cache] == versions  # nothing written
    write_kv_cache(k, k, cache, slots)
    assert all(t._version > v for t, v in zip(cache, versions))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():  # tensors of that mode have no counter
        own = empty_kv_cache(2, 16, 2, 64, device=gpu)
        write_kv_cache(k, k, own, slots)
        write_kv_cache(k, k, cache, slots)
    write_kv_cache(k, k, own, slots)
    for a, b in zip(own, cache):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("which", ["k_codes", "v_codes"])
def test_a_cache_that_asks_for_a_gradient_is_refused(gpu, which):
    from low_bit_fake_quant import paged_attention, read_kv_cache, write_kv_cache
    q, cache, table, lens, starts = problem(gpu, lens=[20], counts=[2])
    k, slots = torch.randn(2, 2, 128, device=gpu), torch.arange(2, device=gpu)
    want = paged_attention(q, cache, table, lens, starts)
    cache = cache._replace(**{which: getattr(cache, which).clone().requires_grad_()})
    for call in (lambda: write_kv_cache(k, k, cache, slots), lambda: read_kv_cache(cache, table, lens, 20),
                 lambda: paged_attention(q, cache, table, lens, starts)):
        with pytest.raises(ValueError, match="no backward pass"):
            call()
    with torch.no_grad():
        assert torch.equal(paged_attention(q, cache, table, lens, starts), want)
        read_kv_cache(cache, table, lens, 20)
