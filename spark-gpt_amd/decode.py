"""The mixture-of-experts layer for a few tokens, on gfx950 kernels: what a
generation step runs in the place of ``fp8_routed_experts``.

The grouped experts pad each expert's rows to 256; with a token or a few of them
the layer is bound by the weights of the experts that are taken.  Here those
are read from memory once, from bf16 or from 4-bit weights.  No counterpart in
the reference, which runs its grouped path at every size (train.py:2262-2299).
There is no CPU fallback.
"""
from __future__ import annotations

import torch

from . import torch_ops
from .mxfp4 import MXFP4, _is_mxfp4, _no_tangent

MAX_TOKENS = 64


def decode_routed_experts(x: torch.Tensor, router: torch.Tensor, w_gu, w_down, top_k: int, *, score: str = "softmax",
                          bias: torch.Tensor | None = None, mask: torch.Tensor | None = None, groups: int = 1,
                          top_groups: int | None = None, group_best: int = 1, renormalize: bool = True,
                          scale: float = 1.0):
    """The layer from its router on: ``(out [T, D] bf16, selected int64 [T, top_k])``.

    ``x`` [T, D] bf16 (any strides), T <= 64; ``router`` [E, D] fp32 or bf16;
    ``w_gu`` [E, 2I, D] (gate rows first) and ``w_down`` [E, D, I] both bf16 or
    both ``MXFP4``; D and I multiples of 8.

    The logits are x router^T, summed in 64 bits; ``top_k`` and the keyword
    arguments are those of ``route_tokens``, and the experts are ordered by the
    64-bit values (not by logits rounded to 32).  h = silu(x Wg^T) * (x Wu^T), and
    out is the sum over the chosen experts of weight * h Wd^T, with h and the sums
    in 32 bits and one rounding at the end; 4-bit weights multiply x in bf16 as the
    values they stand for.  Masked tokens give rows of zeros and -1.  An infinity
    in w_down makes its column of its expert's tokens NaN (h meets it in parts,
    some of them zero).

    No gradient is taken: with gradients enabled, inputs that require one are
    refused, and so are inputs with a forward-mode tangent."""
    quantized = isinstance(w_gu, MXFP4)
    if quantized != isinstance(w_down, MXFP4):
        raise TypeError("w_gu and w_down must be both bf16 tensors or both MXFP4")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, router, bias)
                                       + (() if quantized else (w_gu, w_down))):
        raise ValueError("decode_routed_experts takes no gradient: call it under torch.no_grad(), or train through "
                         "route_tokens and the grouped experts")
    _no_tangent("decode_routed_experts", x, router, bias, w_gu, w_down)
    if quantized:
        _is_mxfp4("w_gu", w_gu, (3,))
        _is_mxfp4("w_down", w_down, (3,))
        shapes = (tuple(w_gu.shape), tuple(w_down.shape))
        parts = (w_gu.codes, w_gu.scales, w_down.codes, w_down.scales)
    else:
        if w_gu.dim() != 3 or w_down.dim() != 3:
            raise ValueError(f"w_gu must be [E, 2I, D] and w_down [E, D, I], got {tuple(w_gu.shape)} and "
                             f"{tuple(w_down.shape)}")
        shapes = (tuple(w_gu.shape), tuple(w_down.shape))
        parts = (w_gu, None, w_down, None)
    E, D, I = shapes[1]
    if shapes[0] != (E, 2 * I, D) or x.dim() != 2 or x.shape[1] != D:
        raise ValueError(f"x [T, D], w_gu [E, 2I, D] and w_down [E, D, I] do not fit: {tuple(x.shape)}, {shapes[0]}, "
                         f"{shapes[1]}")
    if router.dim() != 2 or tuple(router.shape) != (E, D):
        raise ValueError(f"router must be [{E}, {D}], got {tuple(router.shape)}")
    return torch_ops.op("moe_decode")(x, router, *parts, I, bias, mask, score, groups,
                                      groups if top_groups is None else top_groups, group_best, top_k, renormalize,
                                      float(scale))
