"""The cache operators from their definitions, in 64 bits, on whatever device the inputs are.

``mx_encode`` / ``mx_decode``: the MXFP8 rows of the cache; ``norm_rope`` and its
gradient; ``attend``: paged attention with the error bounds of the kernels'
roundings (see there)."""

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def mx_encode(x):
    """(..., D) -> values of the E4M3 codes (fp64) and the scales' exponents (int64), finite x."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1).clamp_min(float(torch.tensor(1e-4, dtype=torch.float32)))
    m, e = torch.frexp(top / 448.0)
    e = e.long() - (m == 0.5).long()
    q = g / torch.exp2(e.double())[..., None]
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3.0)
    return (torch.round(q / step) * step).flatten(-2), e


def mx_decode(codes, scale):
    """Values (fp64) of float8_e4m3fn codes and E8M0 bytes."""
    c = codes.view(torch.uint8).long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8.0 + m) * torch.exp2(e.double() - 10.0))
    v = torch.where(c > 127, -v, v)
    return v * torch.exp2(scale.double() - 127.0).repeat_interleave(32, -1)


def rows_of(codes, scale, table_row, length):
    """(length, H, D) fp64 of one sequence; rows of pages that are not there are NaN."""
    n, h, page, d = codes.shape
    length = min(length, table_row.numel() * page)
    out = torch.full((length, h, d), math.nan, dtype=torch.float64, device=codes.device)
    for i in range(-(-length // page)):
        pid, take = int(table_row[i]), min(page, length - i * page)
        if 0 <= pid < n:
            x = mx_decode(codes[pid:pid + 1].contiguous(), scale[pid:pid + 1])[0]
            out[i * page:i * page + take] = x.transpose(0, 1)[:take]
    return out


def visible(n, length, causal, window, device):
    """(n, length) bool."""
    at = length - n + torch.arange(n, device=device)[:, None]
    j = torch.arange(length, device=device)
    see = torch.ones(n, length, dtype=torch.bool, device=device)
    if causal:
        see &= j <= at
    if window:
        see &= j > at - window
    return see


def attend(q, cache, table, lens, starts, *, causal=True, window=None, sm_scale=None):
    """-> out, lse (fp64; rows of no sequence 0 / -inf) and their bounds.

    For a row with weights p_j (sum l) and A = sum p_j |V_j| / l, the kernels'
    result is off by at most
      u_out |o|                 the output's rounding
      + A 2^-10.9               P rounded to 11 bits (2^-11), for numerator only
      + 2 A ds                  scores off by ds: fp32 sums of exact products, in any order, and the exponent's
                                argument rounded: (D + 8) 2^-24 sum |q k| scale + 2^-22 max |s|
      + 2 A (N + 64) 2^-24      fp32 sums over N keys and the rescaling, in any order
    and its lse by ds + (N + 64) 2^-24 + 2^-22 |lse|.
    """
    T, hq, d = q.shape
    hk = cache[0].shape[1]
    sm = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    out = torch.zeros(T, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(table.shape[0]):
        r0, r1 = int(starts[b]), int(starts[b + 1])
        n = r1 - r0
        k = rows_of(cache[0], cache[1], table[b], int(lens[b]))
        v = rows_of(cache[2], cache[3], table[b], int(lens[b]))
        L = k.shape[0]
        if n == 0 or L == 0:
            continue
        see = visible(n, L, causal, window, q.device)
        there = ~torch.isnan(k).any(-1).any(-1) & ~torch.isnan(v).any(-1).any(-1)
        # a key on a missing page is not seen; any other NaN would be a mistake of the test
        see = see & there
        k, v = torch.nan_to_num(k), torch.nan_to_num(v)
        qq = q[r0:r1].double().transpose(0, 1)
        kk = k.transpose(0, 1).repeat_interleave(hq // hk, 0)
        vv = v.transpose(0, 1).repeat_interleave(hq // hk, 0)
        kt = kk.transpose(1, 2).contiguous()
        s = torch.bmm(qq, kt) * sm
        size = torch.bmm(qq.abs(), kt.abs()) * sm
        s = torch.where(see, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        some = top > -math.inf
        top = torch.where(some, top, 0.0)
        p = torch.exp(s - top)
        l = p.sum(-1, keepdim=True)
        l1 = torch.where(some, l, 1.0)
        o = torch.bmm(p, vv.contiguous()) / l1
        a = torch.bmm(p, vv.abs().contiguous()) / l1
        ds = ((d + 8) * 2.0 ** -24 * torch.where(see, size, 0.0) + 2.0 ** -22 * torch.where(see, s, 0.0).abs()).amax(
            -1, keepdim=True)
        sums = (L + 64) * 2.0 ** -24
        out[r0:r1] = o.transpose(0, 1)
        tol[r0:r1] = (U[q.dtype] * o.abs() + a * (2.0 ** -10.9 + 2 * ds + 2 * sums)).transpose(0, 1)
        z = torch.where(some, top + torch.log(l1), -math.inf)
        lse[r0:r1] = z[..., 0].t()
        ltol[r0:r1] = (ds + sums + 2.0 ** -22 * torch.where(some, z, 0.0).abs())[..., 0].t()
    # values below the output type's normal range round by its smallest step
    tiny = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[q.dtype]
    return out, lse, tol + tiny, ltol


def check(got, want, tol, what):
    """Each value within its bound.  Rounding to nearest gives infinity from half a step
    past the type's largest value on (fp16: 65504 + 16); a value whose bound reaches
    that far may come out as that infinity."""
    top = torch.finfo(got.dtype).max
    over = want.abs() + tol >= top * (1 + torch.finfo(got.dtype).eps / 4)
    got = got.double()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    bad = ~((got == want) | ((got - want).abs() <= tol) | (over & (got == torch.sign(want) * math.inf)))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at "
                           f"{tuple(int(i) for i in bad.nonzero()[0])}: {got[bad][0].item()} for {want[bad][0].item()} "
                           f"(bound {tol.expand_as(want)[bad][0].item():.3g})")


def rotate(n, cos, sin, pairs, back=False):
    rot = 2 * cos.shape[-1]
    if back:
        sin = -sin
    n = n.clone()
    if pairs == "adjacent":
        ia, ib = slice(0, rot, 2), slice(1, rot, 2)
    else:
        ia, ib = slice(0, rot // 2), slice(rot // 2, rot)
    a, b = n[..., ia].clone(), n[..., ib].clone()
    n[..., ia], n[..., ib] = a * cos - b * sin, a * sin + b * cos
    return n


def norm_rope(x, w, cos, sin, pairs, eps):
    """x (..., H, D), cos / sin (..., R/2) of each token, in fp64 -> y."""
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return rotate(n if w is None else n * w, cos[..., None, :], sin[..., None, :], pairs)


def norm_rope_grad(x, w, dy, cos, sin, pairs, eps):
    """-> dx, dw, and sum |terms| of dw."""
    r = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    dn = rotate(dy, cos[..., None, :], sin[..., None, :], pairs, back=True)
    g = dn if w is None else dn * w
    dx = r * (g - x * r * (g * x * r).mean(-1, keepdim=True))
    t = (dn * x * r).flatten(0, -2)
    return dx, t.sum(0), t.abs().sum(0)
