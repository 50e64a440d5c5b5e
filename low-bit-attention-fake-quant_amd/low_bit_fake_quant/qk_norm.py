"""RMS norm of each query and key head with the position rotation, on gfx950.

What a transformer layer does to its projected Q and K before attention, in
one launch for both, with a backward pass.  The outputs feed
``fake_quant_attention`` or, token by token, ``kv_cache.write_kv_cache`` and
``kv_cache.paged_attention``.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from ._ops import _dt

PAIRS = ("adjacent", "halves")


def rows_16b(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself if its last dimension is contiguous and every row starts on a
    16-byte boundary (any other strides are passed to the kernel), else a copy."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t  # rows of 64 or 128 values of at least 16 bits
        *outer, last = t.stride()
        step = 16 // t.element_size()
        if last == 1:
            for st, n in zip(outer, t.shape):
                if st % step and n != 1:
                    break
            else:
                return t
    return t.clone(memory_format=torch.contiguous_format)


def row_strides(t: torch.Tensor) -> list[int]:
    """Strides of all dimensions but the last; of one of a single entry, whose stride may be anything, 0."""
    return [st if n > 1 else 0 for st, n in zip(t.stride()[:-1], t.shape)]


class _Here:
    """The context of a launch on the current device."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_device(index: int):
    """Launches go to the tensors' device, whichever is current."""
    return _HERE if index == torch.cuda.current_device() else torch.cuda.device(index)


def rotary_table(length: int, rot: int, theta: float = 10000.0, *, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin (fp32, (length, rot / 2)) of position * theta^(-2 i / rot); the
    angles are formed in 64 bits, where those of far positions keep their fraction."""
    if rot <= 0 or rot % 2:
        raise ValueError(f"rot must be positive and even; got {rot}")
    f = float(theta) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    a = torch.arange(length, dtype=torch.float64, device=device)[:, None] * f
    return a.cos().float(), a.sin().float()


def _params(q, k, q_weight, k_weight, cos, sin, positions, eps, halves) -> _lib.QkNormParams:
    code = _lib.DTYPE_CODE
    p = _lib.QkNormParams()
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.dtype = code[q.dtype]
    p.B, p.S, p.Hq, p.D = q.shape
    p.Hk = k.shape[2]
    p.q_b, p.q_s, p.q_h = row_strides(q)
    p.k_b, p.k_s, p.k_h = row_strides(k)
    if q_weight is not None:
        p.q_weight = q_weight.data_ptr(); p.q_weight_dtype = code[q_weight.dtype]
    if k_weight is not None:
        p.k_weight = k_weight.data_ptr(); p.k_weight_dtype = code[k_weight.dtype]
    p.cos = cos.data_ptr(); p.sin = sin.data_ptr()
    p.table_len, half = cos.shape
    p.rot = 2 * half
    if positions is not None:
        p.positions = positions.data_ptr()
        p.positions_i64 = 1 if positions.dtype == torch.int64 else 0
        st = positions.stride()
        p.pos_s = st[-1]
        p.pos_b = st[0] if len(st) == 2 else 0
    p.eps = eps; p.halves = 1 if halves else 0
    return p


def _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, halves):
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    if q.numel():
        p = _params(q, k, q_weight, k_weight, cos, sin, positions, eps, halves)
        p.q_out = q_out.data_ptr(); p.k_out = k_out.data_ptr()
        with on_device(q.get_device()):
            _lib.check(_lib.load().lbfq_qk_norm_rope(p, _lib.stream_handle(q.device)), "lbfq_qk_norm_rope")
    return q_out, k_out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, halves):
        q, k = rows_16b(q), rows_16b(k)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps, ctx.halves = eps, halves
        return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, halves)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        want = ctx.needs_input_grad
        dq = torch.empty_like(q, memory_format=torch.contiguous_format)
        dk = torch.empty_like(k, memory_format=torch.contiguous_format)
        empty = q.numel() == 0
        new = torch.zeros_like if empty else torch.empty_like
        dqw = new(q_weight) if want[2] else None
        dkw = new(k_weight) if want[3] else None
        if not empty:
            lib = _lib.load()
            dyq, dyk = rows_16b(dyq), rows_16b(dyk)
            p = _params(q, k, q_weight, k_weight, cos, sin, positions, ctx.eps, ctx.halves)
            g = _lib.QkNormGrads()
            g.dyq = dyq.data_ptr(); g.dyk = dyk.data_ptr()
            g.dyq_b, g.dyq_s, g.dyq_h = row_strides(dyq)
            g.dyk_b, g.dyk_s, g.dyk_h = row_strides(dyk)
            g.dq = dq.data_ptr(); g.dk = dk.data_ptr()
            g.dq_weight = _lib.ptr(dqw); g.dk_weight = _lib.ptr(dkw)
            with on_device(q.get_device()):
                partial = None
                if dqw is not None or dkw is not None:
                    rows = int(lib.lbfq_qk_norm_rope_bwd_rows(p))
                    partial = torch.empty(rows * 2 * p.D, dtype=torch.float32, device=q.device)
                    g.partial = partial.data_ptr()
                _lib.check(lib.lbfq_qk_norm_rope_bwd(p, g, _lib.stream_handle(q.device)), "lbfq_qk_norm_rope_bwd")
        return dq if want[0] else None, dk if want[1] else None, dqw, dkw, None, None, None, None, None


def _check_weight(w, name, d, index):
    if w is None:
        return None
    if w.shape != (d,):
        raise ValueError(f"{name} must have shape {(d,)}; got {tuple(w.shape)}")
    if w.get_device() != index:
        raise ValueError(f"{name} must live on cuda:{index}; got {w.device}")
    _dt(w)
    return w.contiguous()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None, *, eps: float = 1e-6,
                 pairs: str = "adjacent") -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head's row of Q and K and the rotation by its position.

    ``q`` is (B, S, Hq, D) and ``k`` (B, S, Hk, D), or (T, Hq, D) and (T, Hk, D),
    with D 64 or 128, in fp32, fp16 or bf16; views of a joint projection are
    read where they are (rows that are not contiguous and 16-byte aligned are
    copied).  A row x becomes ``n = x * w / sqrt(mean(x^2) + eps)`` with
    ``q_weight`` / ``k_weight`` (D,) of any of these dtypes (None: ones), and the
    first R columns of n are rotated in pairs, ``(2i, 2i + 1)`` for
    ``pairs="adjacent"`` or ``(i, i + R/2)`` for ``"halves"``:
    ``(a cos - b sin, a sin + b cos)``.  ``cos`` and ``sin`` are fp32 (P, R/2), R a
    multiple of 16 up to D (``rotary_table``).  ``positions`` (int32 or int64, (S,)
    or (B, S); (T,) for three dimensions) picks the table's row of each token;
    without it token s takes row s.  A negative position is normalised and not
    rotated (padding); one past the table comes out as NaN.

    Arithmetic is fp32 with one rounding at the end.  Gradients reach q, k and the
    weights (``cos`` and ``sin`` take none); the weights' sums have a fixed order.
    Returns new contiguous tensors of the inputs' shapes and dtype.
    """
    shape, kshape = q.shape, k.shape
    if len(shape) not in (3, 4) or len(kshape) != len(shape):
        raise ValueError(f"q and k must both be (B, S, H, D) or (T, H, D); got {tuple(shape)} and {tuple(kshape)}")
    index = q.get_device()
    if not q.is_cuda or k.get_device() != index:
        raise ValueError(f"q and k must live on one CUDA device; got {q.device} and {k.device}")
    if k.dtype != q.dtype:
        raise TypeError(f"q and k must have one dtype; got {q.dtype} and {k.dtype}")
    _dt(q)
    flat = len(shape) == 3
    if flat:
        q, k = q.unsqueeze(0), k.unsqueeze(0)
        shape, kshape = q.shape, k.shape
    b, s, hq, d = shape
    kb, ks, hk, kd = kshape
    if d not in (64, 128):
        raise ValueError(f"D must be 64 or 128; got {d}")
    if kb != b or ks != s or kd != d or hq == 0 or hk == 0:
        raise ValueError(f"q and k must agree in all but their heads; got {tuple(shape)} and {tuple(kshape)}")
    if pairs not in PAIRS:
        raise ValueError(f"pairs must be one of {PAIRS}; got {pairs!r}")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative; got {eps}")
    if cos.ndim != 2 or sin.shape != cos.shape:
        raise ValueError(f"cos and sin must be (P, R/2); got {tuple(cos.shape)} and {tuple(sin.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError(f"cos and sin must be float32; got {cos.dtype} and {sin.dtype}")
    length, half = cos.shape
    if half == 0 or half % 8 or 2 * half > d:
        raise ValueError(f"R must be a multiple of 16 up to D={d}; got {2 * half}")
    if cos.get_device() != index or sin.get_device() != index:
        raise ValueError(f"cos and sin must live on {q.device}")
    if positions is None:
        if s > length:
            raise ValueError(f"the table has {length} positions, q has {s}")
    else:
        if positions.dtype != torch.int64 and positions.dtype != torch.int32:
            raise TypeError(f"positions must be int32 or int64; got {positions.dtype}")
        if positions.get_device() != index:
            raise ValueError(f"positions must live on {q.device}; got {positions.device}")
        if positions.shape != (s,) and (flat or positions.shape != (b, s)):
            raise ValueError(f"positions must have shape {(s,)}{'' if flat else f' or {(b, s)}'}; "
                             f"got {tuple(positions.shape)}")
    q_weight = _check_weight(q_weight, "q_weight", d, index)
    k_weight = _check_weight(k_weight, "k_weight", d, index)
    halves = pairs == "halves"
    cos, sin = cos.contiguous(), sin.contiguous()
    if cos.data_ptr() % 16 or sin.data_ptr() % 16:
        cos, sin = cos.clone(), sin.clone()
    if torch.is_grad_enabled():
        if cos.requires_grad or sin.requires_grad:
            raise ValueError("qk_norm_rope has no gradient for cos and sin; detach them")
        if q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad) or (
                k_weight is not None and k_weight.requires_grad):
            out = _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, halves)
            return (out[0][0], out[1][0]) if flat else out
    out = _forward(rows_16b(q), rows_16b(k), q_weight, k_weight, cos, sin, positions, eps, halves)
    return (out[0][0], out[1][0]) if flat else out


__all__ = ["qk_norm_rope", "rotary_table"]
