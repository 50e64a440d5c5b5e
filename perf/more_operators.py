"""Appending rotated keys to the paged cache, and the cache in 4 bits: calls, plain forms, exact values.

``listed()`` names calls that a model which keeps its keys and values in a
quantised cache makes, from one token to a whole prompt; ``draw(rng)`` gives
further ones of the same ranges.  A case is a dict of plain values:

* ``op``: ``append`` (append_kv_cache), ``store`` (write_kv_cache, then read_kv_cache: K and V as attention sees
  them), ``read`` (read_kv_cache) or ``attend`` (paged_attention);
* ``bits`` of the cache's codes: 4, or (append) 8.  An append to 4 bits is read back, as ``store`` is; one to 8
  bits returns the cache itself;
* ``Hq, Hk, D, dtype``: query heads, key heads, head size, the caller's dtype; ``page`` rows of a page;
* ``B`` sequences of up to ``L`` tokens (``_lengths``), of which up to ``n`` are new;
* append: ``rot`` rotated columns, ``pairs`` (``adjacent`` or ``halves``), ``packed`` (q, k, v are views of one
  projection's output);
* attend: ``causal``, ``window`` (0: none), ``tail`` rows behind the last sequence.

The cache holds, for every 32 columns of a row, one E8M0 byte e for the factor
2^(e - 127) = 2^ceil(log2(max(amax, 1e-4) / top)) and codes that round to
nearest, ties to even: E4M3 with top = 448, or E2M1 (0, 1/2, 1, 3/2, 2, 3, 4, 6
and a sign, two to a byte, the even column in the low half) with top = 6.  A
rotated key is fp32, each product and the sum rounded, before it is quantised.
"""

import functools
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@functools.lru_cache(maxsize=None)
def _package():
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "low-bit-attention-fake-quant_amd"))
    import low_bit_fake_quant
    return low_bit_fake_quant


# ---- cases -----------------------------------------------------------------------------------------


def _append(B, n, L, Hq, Hk, D, dtype="bf16", bits=4, page=64, rot=None, pairs="halves", packed=True):
    return dict(op="append", bits=bits, B=B, n=n, L=L, Hq=Hq, Hk=Hk, D=D, dtype=dtype, page=page, rot=rot or D,
                pairs=pairs, packed=packed)


def _store(B, n, L, Hk, D, dtype="bf16", page=64):
    return dict(op="store", bits=4, B=B, n=n, L=L, Hk=Hk, D=D, dtype=dtype, page=page)


def _read(B, L, Hk, D, dtype="bf16", page=64):
    return dict(op="read", bits=4, B=B, L=L, Hk=Hk, D=D, dtype=dtype, page=page)


def _attend(B, n, L, Hq, Hk, D, dtype="bf16", page=64, causal=True, window=0, tail=0):
    return dict(op="attend", bits=4, B=B, n=n, L=L, Hq=Hq, Hk=Hk, D=D, dtype=dtype, page=page, causal=causal,
                window=window, tail=tail)


def listed():
    return [
        # one decoding step of a batch: a few rows, launches and latency
        dict(_append(24, 1, 4000, 32, 8, 128, bits=8, page=16), name="append_decode_24"),
        # odd chunks of new tokens after unequal pasts, heads of 64 of which half is rotated, fp16
        dict(_append(5, 777, 3001, 28, 4, 64, "fp16", 8, 32, 32, "adjacent"), name="append_chunks_5x777_fp16"),
        # all tokens of a Wan2.1-14B layer into 4 bits, and the cache handed on as whole tensors
        dict(_append(1, 32760, 32760, 40, 40, 128, pairs="adjacent"), name="append_wan14b"),
        # a few short prompts into small pages and back
        dict(_store(8, 100, 100, 8, 128, "fp16", 16), name="store_8x100_fp16"),
        # all keys and values of a Wan2.1-1.3B layer, as 4 bits hold them
        dict(_store(1, 32760, 32760, 12, 128), name="store_wan1.3b"),
        # a few short ragged sequences looked at in fp32
        dict(_read(5, 777, 4, 64, "fp32", 16), name="read_5x777_fp32"),
        # the cache of a batch handed to an attention that takes whole tensors
        dict(_read(8, 16384, 8, 128), name="read_8x16384"),
        # one token of one sequence: a single user
        dict(_attend(1, 1, 5003, 32, 8, 128), name="attend_one_5003"),
        # one token of each sequence of a large ragged batch, an empty one among them
        dict(_attend(48, 1, 16000, 32, 8, 128, page=32), name="attend_decode_48x16000"),
        # odd chunks of new tokens after unequal pasts, a sliding window, fp16, rows behind the last sequence
        dict(_attend(4, 509, 9001, 28, 4, 64, "fp16", 16, window=4096, tail=3), name="attend_chunks_4x509_fp16"),
        # a whole prompt at once
        dict(_attend(1, 8192, 8192, 32, 8, 128), name="attend_prompt_8192"),
        # three latent frames of a Wan2.1-1.3B video over all frames up to them, each token seeing all
        dict(_attend(1, 4680, 32760, 12, 12, 128, causal=False), name="attend_wan1.3b_frames"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((12, 12), (32, 8), (8, 1), (28, 4), (5, 5), (24, 8), (16, 2), (40, 40), (32, 2))


def draw(rng):
    op = rng.choice(("append", "append", "store", "read", "attend", "attend", "attend"))
    Hq, Hk = rng.choice(HEADS)
    D = rng.choice((64, 128, 128))
    page = rng.choice((16, 32, 64, 128))
    if op != "attend":
        B = _log_uniform(rng, 1, 32)
        L = _log_uniform(rng, 1, max(1, min(20000, 600000 // (B * (Hk if op != "append" else (Hq + 2 * Hk) // 2)))))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        n = rng.choice((1, L, _log_uniform(rng, 1, L)))
        if op == "append":
            return _append(B, n, L, Hq, Hk, D, dtype, rng.choice((4, 8)), page, rng.choice((D, D, D // 2)),
                           rng.choice(("adjacent", "halves")), rng.random() < 0.6)
        return _store(B, n, L, Hk, D, dtype, page) if op == "store" else _read(B, L, Hk, D, dtype, page)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    window = 0 if rng.random() < 0.7 else _log_uniform(rng, 1, 4000)
    tail = rng.choice((0, 0, 1, 5))
    if rng.random() < 0.5:
        B = _log_uniform(rng, 1, 48)
        L = _log_uniform(rng, 1, max(1, min(30000, 4000000 // (B * Hk))))
        return _attend(B, rng.choice((1, 1, 1, 2, 4)), L, Hq, Hk, D, dtype, page, True, window, tail)
    B = _log_uniform(rng, 1, 6)
    n = _log_uniform(rng, 2, 3000)
    L = n + _log_uniform(rng, 1, max(2, min(20000, 1200000000 // (B * Hq * n)))) - 1
    return _attend(B, n, L, Hq, Hk, D, dtype, page, rng.random() < 0.6, window, tail)


def _lengths(case):
    """[(new tokens, all tokens)] of each sequence.  The first has the case's sizes, the others fewer; of three or more
    one is empty, of four or more one holds fewer tokens than it asks for (its first queries see nothing)."""
    B, L, n = case["B"], case["L"], case.get("n", 1)
    writes = case["op"] in ("append", "store")
    r = random.Random("%d %d %d" % (B, n, L))
    got = []
    for b in range(B):
        nb = n if b == 0 else r.randint(1, n)
        lb = L if b == 0 else nb if n == L else r.randint(max(1, L // 2), L)
        if not writes:
            lb = 0 if b == 1 and B >= 3 else min(lb, (nb + 1) // 2) if b == 3 else lb
        got.append((min(nb, lb) if writes else nb, lb))
    return got


# ---- inputs ----------------------------------------------------------------------------------------


def _rand(seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return gen, lambda *s: torch.randn(*s, generator=gen, device="cuda")


def _table(P, rot):
    """cos and sin of position * 10000^(-2i/rot), angles in 64 bits."""
    f = 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
    a = torch.arange(P, device="cuda", dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _pages(case, gen):
    """A pool of shuffled pages, some more than needed, and each sequence's row of it."""
    per = -(-max(l for _, l in _lengths(case)) // case["page"]) or 1
    B = case["B"]
    order = torch.randperm(B * per + 3, generator=gen, device="cuda").to(torch.int32)
    return B * per + 3, order[:B * per].view(B, per).contiguous()


@functools.lru_cache(maxsize=None)
def _edges():
    """From which size on each E2M1 code but the first holds (a middle goes to the even code)."""
    up = lambda v: float(torch.nextafter(torch.tensor(v), torch.tensor(9.0)))  # noqa: E731
    return torch.tensor([up(0.25), 0.75, up(1.25), 1.75, up(2.5), 3.5, up(5.0)], device="cuda")


@functools.lru_cache(maxsize=None)
def _pairs():
    """The two values of each byte."""
    v = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    v += [-x for x in v]
    return torch.tensor([[v[b & 15], v[b >> 4]] for b in range(256)], device="cuda")


def _encode(x, bits):
    """fp32 rows: bytes of codes and scales."""
    top = 448.0 if bits == 8 else 6.0
    g = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(g.abs().amax(-1).clamp_min(1e-4))
    m0, e0 = math.frexp(top)
    e = e - e0 + (m > m0).to(e.dtype)
    q = (g * torch.exp2(-e.double()).float()[..., None]).clamp(-top, top).flatten(-2)
    if bits == 8:
        c = q.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        c = torch.bucketize(q.abs(), _edges(), right=True, out_int32=True) + 8 * torch.signbit(q)
        c = (c[..., ::2] + 16 * c[..., 1::2]).to(torch.uint8)
    return c, (e + 127).to(torch.uint8)


def _filled(N, case, rand):
    """Bytes of codes and scales of N pages of keys (channel biases, some large channels) or values."""
    shape = (N, case["Hk"], case["page"], case["D"])
    bias, big = 2.0 * rand(1, shape[1], 1, shape[3]), 1.0 + 9.0 * (rand(1, shape[1], 1, shape[3]) > 1.5)
    kc, ks = _encode((rand(*shape) + bias) * big / 3.0, case["bits"])
    vc, vs = _encode(rand(*shape) + rand(1, shape[1], 1, shape[3]), case["bits"])
    return kc, ks, vc, vs


def prepare(case, seed):
    gen, rand = _rand(seed)
    t, D = DTYPES[case["dtype"]], case["D"]
    s = dict(case)
    N, table = _pages(case, gen)
    lens = _lengths(case)
    kc, ks, vc, vs = _filled(N, case, rand)
    # (a cache of 4 bits has two values to an element)
    code = torch.float8_e4m3fn if case["bits"] == 8 else torch.float4_e2m1fn_x2
    s["cache"] = (kc.view(code), ks, vc.view(code), vs)
    s["block_table"] = table
    s["seq_lens"] = torch.tensor([l for _, l in lens], dtype=torch.int32, device="cuda")
    if case["op"] in ("append", "store"):
        T = sum(n for n, _ in lens)
        seq = torch.tensor([b for b, (n, _) in enumerate(lens) for _ in range(n)], device="cuda")
        at = torch.tensor([l - n + i for n, l in lens for i in range(n)], device="cuda")
        s["slots"] = table[seq, at // case["page"]].long() * case["page"] + at % case["page"]
        Hk, Hq = case["Hk"], case.get("Hq", 0)
        x = rand(T, Hq + 2 * Hk, D)
        x[:, Hq:Hq + Hk] += 2.0 * rand(1, Hk, D)
        x = x.to(t)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]
        s.update(k=k, v=v)
        if case["op"] == "append":
            s["cos"], s["sin"] = _table(case["L"], case["rot"])
            s["positions"], s["q"] = at, q
            if not case["packed"]:
                s.update(q=q.contiguous(), k=k.contiguous(), v=v.contiguous())
    elif case["op"] == "attend":
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        s["query_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["q"] = (1.5 * rand(starts[-1] + case["tail"], case["Hq"], D)).to(t)
    return s


# ---- one pass --------------------------------------------------------------------------------------


def run(s):
    return (_own if own else _plain)[s["op"]](s)


def _own_read(s):
    p = _package()
    k, v = p.read_kv_cache(p.PagedKVCache(*s["cache"]), s["block_table"], s["seq_lens"], s["L"],
                           dtype=_back(s))
    return dict(k=k, v=v)


def _back(s):
    """The dtype that values are read back in: the caller's (after a rotation in fp32, where a value next to a
    border goes by the last bit of it, 16 bits)."""
    return torch.bfloat16 if s["op"] == "append" and s["dtype"] == "fp32" else DTYPES[s["dtype"]]


def _own_append(s):
    p = _package()
    cache = p.PagedKVCache(*s["cache"])
    q = p.append_kv_cache(s["q"], s["k"], s["v"], cache, s["slots"], s["cos"], s["sin"], s["positions"], pairs=s["pairs"])
    if s["bits"] == 4:
        return dict(q=q, **_own_read(s))
    return dict(q=q, k=cache.k_codes, k_scale=cache.k_scale, v=cache.v_codes, v_scale=cache.v_scale)


def _own_store(s):
    p = _package()
    p.write_kv_cache(s["k"], s["v"], p.PagedKVCache(*s["cache"]), s["slots"])
    return _own_read(s)


def _own_attend(s):
    p = _package()
    out, lse = p.paged_attention(s["q"], p.PagedKVCache(*s["cache"]), s["block_table"], s["seq_lens"],
                                 s["query_starts"], max_query_len=s["n"], causal=s["causal"],
                                 window=s["window"] or None, return_lse=True)
    return dict(out=out, lse=lse)


_own = dict(append=_own_append, store=_own_store, read=_own_read, attend=_own_attend)


def _rotate(x, cos, sin, pairs):
    """The rotation of the first columns of x."""
    rot = 2 * cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    if pairs == "adjacent":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _put(s, k, v):
    """Rows of fp32 into their slots."""
    page, row = s["slots"] // s["page"], s["slots"] % s["page"]
    for x, codes, scale in ((k, *s["cache"][:2]), (v, *s["cache"][2:])):
        c, e = _encode(x, s["bits"])
        codes.view(torch.uint8)[page, :, row] = c
        scale[page, :, row] = e


def _plain_append(s):
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _rotate(s["q"].float(), cos, sin, s["pairs"]).to(s["q"].dtype)
    _put(s, _rotate(s["k"].float(), cos, sin, s["pairs"]), s["v"].float())
    if s["bits"] == 4:
        return dict(q=q, **_plain_read(s))
    kc, ks, vc, vs = s["cache"]
    return dict(q=q, k=kc, k_scale=ks, v=vc, v_scale=vs)


def _plain_store(s):
    _put(s, s["k"].float(), s["v"].float())
    return _plain_read(s)


def _decoded(codes, scale, table, L):
    """Rows 0 .. L - 1 of each sequence's pages of 4-bit codes: fp32 (B, L, Hk, D)."""
    x = _pairs()[codes.view(torch.uint8)[table.long()].int()].flatten(-2).unflatten(-1, (-1, 32))
    x = (x * torch.exp2(scale[table.long()].float() - 127.0)[..., None]).flatten(-2)
    return x.permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :L]


def _plain_read(s):
    kc, ks, vc, vs = s["cache"]
    there = torch.arange(s["L"], device="cuda") < s["seq_lens"][:, None]
    return {name: torch.where(there[:, :, None, None], _decoded(c, e, s["block_table"], s["L"]), 0.0).to(_back(s))
            for name, c, e in (("k", kc, ks), ("v", vc, vs))}


def _plain_attend(s):
    kc, ks, vc, vs = s["cache"]
    q, starts, L, n, B = s["q"], s["query_starts"].long(), s["L"], s["n"], s["B"]
    T, Hq, D = q.shape
    Hk = s["Hk"]
    k = _decoded(kc, ks, s["block_table"], L).permute(0, 2, 3, 1).contiguous()
    v = _decoded(vc, vs, s["block_table"], L).permute(0, 2, 1, 3).contiguous()
    length, count = s["seq_lens"].long()[:, None], (starts[1:] - starts[:-1])[:, None]
    i = torch.arange(n, device="cuda")
    rows = (starts[:-1, None] + i).clamp_max(T - 1)
    at = length - count + i
    j = torch.arange(L, device="cuda")
    see = (j < length)[:, None].expand(B, n, L)
    if s["causal"]:
        see = see & (j <= at[:, :, None])
    if s["window"]:
        see = see & (j > at[:, :, None] - s["window"])
    x = q.float()[rows].view(B, n, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    score = ((x / math.sqrt(D)) @ k).view(B, Hk, Hq // Hk, n, L).masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, -1, L) @ v).view(B, Hk, Hq // Hk, n, D) / torch.where(total == 0.0, 1.0, total)
    lse = top + total.log()
    # rows of sequence b go to starts[b] .. starts[b + 1]; those past its own are put on a spare row
    to = torch.where(i < count, rows, T).flatten()
    out = torch.zeros(T + 1, Hq, D, device="cuda")
    out[to] = o.permute(0, 3, 1, 2, 4).reshape(-1, Hq, D)
    end = torch.full((T + 1, Hq), -math.inf, device="cuda")
    end[to] = lse.permute(0, 3, 1, 2, 4).reshape(-1, Hq)
    return dict(out=out[:T].to(q.dtype), lse=end[:T].contiguous())


_plain = dict(append=_plain_append, store=_plain_store, read=_plain_read, attend=_plain_attend)


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    D, Hk, size = case["D"], case["Hk"], DTYPES[case["dtype"]].itemsize
    lens = _lengths(case)
    row = Hk * (D * case["bits"] // 8 + D // 32) * 2.0  # K and V of one cached token
    if case["op"] != "attend":
        moved = flops = 0.0
        if case["op"] != "read":
            T = sum(n for n, _ in lens)
            moved += T * (row + 2.0 * Hk * D * size + 8)
            flops += T * Hk * D * 6.0
        if case["op"] == "append":
            moved += T * (2.0 * case["Hq"] * D * size + 4 * case["rot"] + 8)
            flops += T * (case["Hq"] + Hk) * case["rot"] * 3.0
        if case["bits"] == 4:  # and read (back)
            T = sum(l for _, l in lens)
            moved += T * row + 2.0 * case["B"] * case["L"] * Hk * D * _back(case).itemsize
            flops += T * Hk * D * 2.0
        return dict(bytes=moved, flops=flops)
    moved = flops = 0.0
    for n, l in lens:
        at = [l - n + i for i in range(n)]
        hi = [max(0, min(l, p + 1)) if case["causal"] else l for p in at]
        lo = [max(0, p - case["window"] + 1) if case["window"] else 0 for p in at]
        flops += 4.0 * D * case["Hq"] * sum(max(0, h - o) for h, o in zip(hi, lo))
        moved += row * max(0, max(hi) - min(lo)) + n * case["Hq"] * (2.0 * D * size + 4)
    return dict(bytes=moved, flops=flops)


# ---- the definitions in 64 bits, row by row of the formulas ----------------------------------------


def _rounded(x, bits):
    """x rounded to E4M3 (steps of 2^-3 of the binade, of 2^-9 below 2^-6) or E2M1 (of 2^-1, of 2^-1 below 1)."""
    least, digits = (2.0 ** -6, 3.0) if bits == 8 else (1.0, 1.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(least))) - digits)
    return torch.round(x / step) * step


def _value(codes, scale, bits):
    c = codes.view(torch.uint8).long()
    if bits == 8:
        e, m = (c >> 3) & 15, (c & 7).double()
        mag = torch.where(e == 0, m * 2.0 ** -9, (8.0 + m) * torch.exp2(e.double() - 10.0))
        neg = c > 127
    else:
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
        e, m = (c >> 1) & 3, (c & 1).double()
        mag = torch.where(e == 0, m * 0.5, (2.0 + m) * torch.exp2(e.double() - 2.0))
        neg = c > 7
    two = torch.exp2(scale.double() - 127.0).repeat_interleave(32, -1)
    return torch.where(neg, -mag, mag) * two


def exact(case, seed):
    s = prepare(case, seed)
    return dict(append=_exact_append, store=_exact_store, read=_exact_read, attend=_exact_attend)[case["op"]](s)


def _written(s, x, which):
    """Codes' values (without their factors) and scale bytes of x, in place of the rows that it goes to."""
    codes, scale = s["cache"][2 * which:2 * which + 2]
    top = 448.0 if s["bits"] == 8 else 6.0
    g = x.double().unflatten(-1, (-1, 32))
    big = g.abs().amax(-1).clamp_min(float(torch.tensor(1e-4)))
    e = torch.ceil(torch.log2(big / top))
    # the logarithm's own rounding next to a power of two
    e = torch.where(top * torch.exp2(e - 1) >= big, e - 1, torch.where(top * torch.exp2(e) < big, e + 1, e))
    two = scale.clone()
    val = _value(codes, torch.full_like(scale, 127), s["bits"])
    N, H, P, D = val.shape
    flat = (s["slots"][:, None] // P * H + torch.arange(H, device="cuda")) * P + s["slots"][:, None] % P
    val.view(-1, D)[flat] = _rounded(g / torch.exp2(e)[..., None], s["bits"]).flatten(-2)
    two.view(-1, D // 32)[flat] = (e + 127).to(torch.uint8)
    return val, two


def _sequences(s, val, two):
    """(B, L, Hk, D) of the sequences' rows, zero behind their ends."""
    out = torch.zeros(s["B"], s["L"], s["Hk"], s["D"], dtype=torch.float64, device="cuda")
    for b, (_, l) in enumerate(_lengths(s)):
        pages = s["block_table"][b, :-(-l // s["page"])].long()
        x = val[pages] * torch.exp2(two[pages].double() - 127.0).repeat_interleave(32, -1)
        out[b, :l] = x.transpose(1, 2).reshape(-1, s["Hk"], s["D"])[:l]
    return out


def _exact_append(s):
    rot = s["rot"]
    c = torch.arange(rot // 2, device="cuda")
    first, second = (2 * c, 2 * c + 1) if s["pairs"] == "adjacent" else (c, c + rot // 2)
    z = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]

    def turned(x):
        y = x.double().clone()
        pair = torch.complex(y[..., first], y[..., second]) * z
        y[..., first], y[..., second] = pair.real, pair.imag
        return y

    k, ks = _written(s, turned(s["k"]), 0)
    v, vs = _written(s, s["v"], 1)
    if s["bits"] == 4:
        return dict(q=turned(s["q"]), k=_sequences(s, k, ks), v=_sequences(s, v, vs))
    return dict(q=turned(s["q"]), k=k, k_scale=None, v=v, v_scale=None)


def _exact_store(s):
    return {name: _sequences(s, *_written(s, s[name], which)) for which, name in enumerate(("k", "v"))}


def _exact_read(s):
    return {name: _sequences(s, _value(s["cache"][2 * which], torch.full_like(s["cache"][2 * which + 1], 127), 4),
                             s["cache"][2 * which + 1]) for which, name in enumerate(("k", "v"))}


def _rows(s, b, which):
    """Keys (0) or values (1) of sequence b in 64 bits: (length, Hk, D)."""
    l = _lengths(s)[b][1]
    pages = s["block_table"][b, :-(-l // s["page"])].long()
    x = _value(s["cache"][2 * which].view(torch.uint8)[pages], s["cache"][2 * which + 1][pages], s["bits"])
    return x.transpose(1, 2).reshape(-1, s["Hk"], s["D"])[:l]


def _exact_attend(s):
    T, Hq, D = s["q"].shape
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device="cuda")
    r0 = 0
    for b, (n, l) in enumerate(_lengths(s)):
        k, v = _rows(s, b, 0), _rows(s, b, 1)
        at = l - n + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(l, device="cuda")
        hide = torch.zeros(n, l, dtype=torch.bool, device="cuda")
        if s["causal"]:
            hide |= j > at
        if s["window"]:
            hide |= j <= at - s["window"]
        for h in range(Hq if l else 0):
            kh = h // (Hq // s["Hk"])
            for i in range(0, n, 4096):
                r = slice(r0 + i, r0 + min(i + 4096, n))
                a = s["q"][r, h].double() @ k[:, kh].t().contiguous() / math.sqrt(D)
                a = a.masked_fill(hide[i:i + 4096], -math.inf)
                z = torch.logsumexp(a, -1, keepdim=True)
                lse[r, h] = z[:, 0]
                out[r, h] = torch.exp(a - torch.where(z == -math.inf, 0.0, z)) @ v[:, kh].contiguous()
        r0 += n
    return dict(out=out, lse=lse)
