"""Microscaled 4-bit floating point (OCP MX, "MXFP4") on gfx950 kernels:
quantisation, products of quantised matrices, and a linear layer on them.

* ``MXFP4``                                  a quantised matrix, or a batch of them
* ``mxfp4_quantize(x, along=...)``           codes of x, of its transpose, or both from one read
* ``mxfp4_dequantize(q, dtype)``             the values they stand for
* ``mxfp4_matmul(a, b, dtype)``              a b^T over those values
* ``mxfp4_linear(x, w)``                     x w^T with x and w quantised, with gradients; or w kept as MXFP4

32 values of a row share one power of two, 2^(floor(log2(largest |value|)) - 2)
and not below 2^-127, and each is held as the nearest e2m1 code (0, 0.5, 1, 1.5,
2, 3, 4, 6 and a sign; ties to the even code, what is past 6 becomes 6).  A block
with an infinity or a NaN is NaN as a whole.  No counterpart in the reference.
Nothing here synchronises the device, and there is no CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops, torch_ops

BLOCK = 32  # values that share a scale
SLAB = 128  # values of a row that lie together
ROW_ALIGN = 16
ROWS_MAX_N = (1 << 27) - 16  # columns of a product whose rows are quantised on the way
_DIRECTIONS = {"rows": (True, False), "columns": (False, True), "both": (True, True)}


class MXFP4(NamedTuple):
    """A matrix [R, C], or E of them [E, R, C], in 4-bit codes.

    ``codes`` uint8 [(E,) ceil(C / 128), ceil(R / 16) * 16, 64]: 128 values of a
    row in 64 bytes, the lower value in the lower half of a byte; ``scales`` uint8
    [(E,) ceil(C / 128), ceil(R / 16) * 16, 4]: the exponents (bias 127, 255 =
    NaN) of their four blocks.  What is beyond R and C is zero."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple

    @staticmethod
    def from_rows(codes: torch.Tensor, scales: torch.Tensor, columns: int) -> "MXFP4":
        """From rows as checkpoints hold them: codes uint8 [(E,) R, ceil(columns /
        2)] (two values a byte, the lower in the lower half), scales uint8 [(E,) R,
        ceil(columns / 32)].  A copy, once per weight."""
        if not (codes.dtype == scales.dtype == torch.uint8 and codes.dim() == scales.dim() and codes.dim() in (2, 3)):
            raise ValueError("codes and scales must be uint8 matrices, or batches of them")
        if (codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != -(-columns // 2)
                or scales.shape[-1] != -(-columns // BLOCK) or codes.device != scales.device):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not those of rows of "
                             f"{columns} values on one device")
        *lead, rows, _ = codes.shape
        slabs, padded = -(-columns // SLAB), -(-rows // ROW_ALIGN) * ROW_ALIGN
        full = codes.new_zeros(*lead, padded, slabs * 64)
        full[..., :rows, :codes.shape[-1]] = codes
        if columns % 2:
            full[..., :rows, columns // 2] &= 15
        full_scales = scales.new_zeros(*lead, padded, slabs * 4)
        full_scales[..., :rows, :scales.shape[-1]] = scales
        return MXFP4(full.unflatten(-1, (slabs, 64)).transpose(-3, -2).contiguous(),
                     full_scales.unflatten(-1, (slabs, 4)).transpose(-3, -2).contiguous(), (*lead, rows, columns))

    def rows(self):
        """(codes, scales) as rows, what ``from_rows`` takes."""
        rows, columns = self.shape[-2:]
        codes = self.codes.transpose(-3, -2).flatten(-2)[..., :rows, :-(-columns // 2)]
        scales = self.scales.transpose(-3, -2).flatten(-2)[..., :rows, :-(-columns // BLOCK)]
        return codes.contiguous(), scales.contiguous()


def _is_mxfp4(name: str, q, dims=(2,)) -> None:
    if not isinstance(q, MXFP4):
        raise TypeError(f"{name} must be an MXFP4, got {type(q).__name__}")
    if len(q.shape) not in dims:
        raise ValueError(f"{name} must be {' or '.join(f'{d}-D' for d in dims)}, got shape {tuple(q.shape)}")
    if q.codes.dim() != len(q.shape) + 1 or (len(q.shape) == 3 and q.codes.shape[0] != q.shape[0]):
        raise ValueError(f"{name}: codes {tuple(q.codes.shape)} do not fit the shape {tuple(q.shape)}")


def _no_tangent(what: str, *tensors) -> None:
    """Refuses inputs of forward-mode differentiation: a dual tensor needs no gradient, so the paths without a node
    would drop its tangent."""
    if forward_ad._current_level >= 0 and not torch.compiler.is_compiling() and any(
            isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _quantized(x: torch.Tensor, rows: bool, columns: bool):
    """MXFP4 of x and of its transpose, None for the one that is not asked for."""
    parts = torch_ops.op("mxfp4_quantize")(x, rows, columns)
    by_row = MXFP4(parts[0], parts[1], tuple(x.shape)) if rows else None
    by_column = MXFP4(parts[-2], parts[-1], (*x.shape[:-2], x.shape[-1], x.shape[-2])) if columns else None
    return by_row, by_column


def mxfp4_quantize(x: torch.Tensor, along: str = "rows"):
    """MXFP4 of x [R, C] or [E, R, C] (fp32, bf16 or fp16; any strides, copied
    where values of a row do not lie side by side).

    ``along``: ``"rows"`` (blocks of 32 values of a row, what a product over C
    reads), ``"columns"`` (of the transpose [C, R], what a product over R reads) or
    ``"both"`` (the pair of them from one read).  Not differentiable: the codes
    carry no gradient."""
    if along not in _DIRECTIONS:
        raise ValueError(f"along must be 'rows', 'columns' or 'both', got {along!r}")
    by_row, by_column = _quantized(x.detach(), *_DIRECTIONS[along])
    return (by_row, by_column) if along == "both" else by_row if along == "rows" else by_column


def mxfp4_dequantize(q: MXFP4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of q, rounded to ``dtype`` (bf16 and fp32 hold them all, but
    for those past their largest)."""
    _is_mxfp4("q", q, (2, 3))
    return torch_ops.op("mxfp4_dequantize")(q.codes, q.scales, q.shape[-2], q.shape[-1], dtype)


def mxfp4_matmul(a: MXFP4, b: MXFP4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b^T [M, N] for a [M, K] and b [N, K], both along their rows: the values'
    products summed in 32 bits and rounded once to ``dtype`` (fp32, bf16, fp16)."""
    _is_mxfp4("a", a)
    _is_mxfp4("b", b)
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} must have rows of one length")
    return torch_ops.op("mxfp4_matmul")(a.codes, a.scales, b.codes, b.scales, a.shape[0], b.shape[0], a.shape[1], dtype)


class _MXFP4Linear(torch.autograd.Function):
    """x w^T on quantised operands in a compiled graph (an eager call makes the
    same node in C++).  Each of the three products quantises its
    operands along the dimension that it sums over; gradients pass the
    quantisation as if it were not there.  What is kept for the backward pass is
    in 4 bits: the codes of x along its rows' dimension and of w along its."""

    @staticmethod
    def forward(ctx, x, w):
        need_x, need_w = ctx.needs_input_grad
        xr, xc = _quantized(x, True, need_w)
        wr, wc = _quantized(w, True, need_x)
        kept = [t for q in (xc, wc) if q is not None for t in q[:2]]
        ctx.save_for_backward(*kept)
        ctx.size = (*x.shape, w.shape[0])
        ctx.types = (x.dtype, w.dtype)
        return mxfp4_matmul(xr, wr, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w = ctx.needs_input_grad
        T, K, N = ctx.size
        kept = ctx.saved_tensors
        dx = dw = None
        dr, dc = _quantized(dy, need_x, need_w)
        if need_x:
            dx = mxfp4_matmul(dr, MXFP4(kept[-2], kept[-1], (K, N)), ctx.types[0])
        if need_w:
            dw = mxfp4_matmul(dc, MXFP4(kept[0], kept[1], (K, T)), ctx.types[1])
        return dx, dw


def mxfp4_linear(x: torch.Tensor, w) -> torch.Tensor:
    """x w^T for x [..., K] (fp32, bf16 or fp16), in x's type.

    ``w`` [N, K] a tensor (a master in fp32, bf16 or fp16): both are quantised
    along K, and the gradients are dx = q(dy) q(w) over blocks along N and dw =
    q(dy)^T q(x) over blocks along the tokens, in the types of x and w.  Zero
    tokens give a zero gradient of w.

    ``w`` an ``MXFP4`` [N, K] (weights kept in 4 bits): no gradient is taken.  Up
    to 16 tokens without a gradient are quantised within the product's kernel,
    with the same codes.

    Differentiable once, and not in forward mode."""
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    kept = isinstance(w, MXFP4)
    if kept:
        _is_mxfp4("w", w)
    elif w.dim() != 2:
        raise ValueError(f"w must be [N, K], got shape {tuple(w.shape)}")
    N, K = w.shape
    if x.shape[-1] != K:
        raise ValueError(f"x must be [..., {K}], got shape {tuple(x.shape)}")
    _no_tangent("mxfp4_linear", x, w)
    flat = x if x.dim() == 2 else x[None] if x.dim() == 1 else x.flatten(0, -2)
    if torch.is_grad_enabled() and (x.requires_grad or (not kept and w.requires_grad)):
        if kept:
            raise ValueError("weights kept as MXFP4 give no gradient of x: pass the master, or call without gradients")
        y = (_MXFP4Linear.apply if torch.compiler.is_compiling() else ops.mxfp4_linear)(flat, w)
    else:
        q = w if kept else _quantized(w, True, False)[0]
        if flat.shape[0] <= ROW_ALIGN and N <= ROWS_MAX_N:
            y = torch_ops.op("mxfp4_rows_matmul")(flat, q.codes, q.scales, N, x.dtype)
        else:
            y = mxfp4_matmul(_quantized(flat, True, False)[0], q, x.dtype)
    return y.view(*x.shape[:-1], N) if x.dim() != 2 else y
