"""The cache in 4 bits from its definition, in 64 bits; what reads it is checked as for 8
bits, on the 8-bit cache of the same values (every E2M1 value is an E4M3 value)."""

import torch

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def encode(x):
    """(..., D) -> values of the E2M1 codes (fp64) and the scales' exponents (int64), finite x."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1).clamp_min(float(torch.tensor(1e-4, dtype=torch.float32)))
    m, e = torch.frexp(top / 6.0)
    e = (e.long() - (m == 0.5).long()).clamp(max=125)
    q = (g / torch.exp2(e.double())[..., None]).clamp(-6.0, 6.0)
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(1.0))) - 1.0)
    return (torch.round(q / step) * step).flatten(-2), e


def values(codes):
    """fp64 values of the codes, without their scales: (..., D / 2) -> (..., D)."""
    c = codes.view(torch.uint8).long()
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=c.device)
    return table[c]


def widen(cache):
    """The 8-bit cache of the same values."""
    k, v = (values(c).to(torch.float8_e4m3fn) for c in (cache[0], cache[2]))
    return type(cache)(k, cache[1].clone(), v, cache[3].clone())


def garbage(pages, page, h, d, dev, seed=3):
    """A cache of arbitrary bytes, scales of 255 among them."""
    from low_bit_fake_quant import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    by = lambda w: torch.randint(0, 256, (pages, h, page, w), generator=g, dtype=torch.uint8).to(dev)  # noqa: E731
    f4 = torch.float4_e2m1fn_x2
    return PagedKVCache(by(d // 2).view(f4), by(d // 32), by(d // 2).view(f4), by(d // 32))
