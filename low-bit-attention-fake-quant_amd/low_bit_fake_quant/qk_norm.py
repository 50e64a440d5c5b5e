"""RMS norm of each query and key head with the position rotation, on gfx950.

What a transformer layer does to its projected Q and K before attention, in
one launch for both, with a backward pass.  The outputs feed
``fake_quant_attention`` or, token by token, ``kv_cache.write_kv_cache`` and
``kv_cache.paged_attention``.  Arguments are checked in ``csrc/lbfq_torch.cpp``.
"""

from __future__ import annotations

import torch

from . import _lib


def rotary_table(length: int, rot: int, theta: float = 10000.0, *, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin (fp32, (length, rot / 2)) of position * theta^(-2 i / rot); the
    angles are formed in 64 bits, where those of far positions keep their fraction."""
    if rot <= 0 or rot % 2:
        raise ValueError(f"rot must be positive and even; got {rot}")
    f = float(theta) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    a = torch.arange(length, dtype=torch.float64, device=device)[:, None] * f
    return a.cos().float(), a.sin().float()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None, *, eps: float = 1e-6,
                 pairs: str = "adjacent") -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head's row of Q and K and the rotation by its position.

    ``q`` is (B, S, Hq, D) and ``k`` (B, S, Hk, D), or (T, Hq, D) and (T, Hk, D),
    with D 64 or 128, in fp32, fp16 or bf16 (every head by itself; a norm over all of a
    token's heads at once is another operator); views of a joint projection are
    read where they are (rows that are not contiguous and 16-byte aligned are
    copied).  A row x becomes ``n = x * w / sqrt(mean(x^2) + eps)`` with
    ``q_weight`` / ``k_weight`` (D,) of any of these dtypes (None: ones), and the
    first R columns of n are rotated in pairs, ``(2i, 2i + 1)`` for
    ``pairs="adjacent"`` or ``(i, i + R/2)`` for ``"halves"``:
    ``(a cos - b sin, a sin + b cos)``.  ``cos`` and ``sin`` are fp32 (P, R/2), R a
    multiple of 16 up to D (``rotary_table``).  ``positions`` (int32 or int64, (S,)
    or (B, S); (T,) for three dimensions) picks the table's row of each token;
    without it token s takes row s.  A negative position is normalised and not
    rotated (padding); one past the table comes out as NaN.  Columns that are not
    rotated do not reach each other.

    Arithmetic is fp32 with one rounding at the end.  Gradients reach q, k and the
    weights (``cos`` and ``sin`` take none); the weights' sums have a fixed order.  A
    second derivative and forward mode are refused.
    Returns new contiguous tensors of the inputs' shapes and dtype.
    """
    return _lib.torch_ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, pairs)


__all__ = ["qk_norm_rope", "rotary_table"]
