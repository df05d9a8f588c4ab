"""The global gradient norm and clipping, on gfx950 kernels: what a training
step does between the backward pass and the optimizer (whose momentum stage is
``muon.py``).

* ``grad_norm(grads)``                      the 2-norm over all gradients
* ``clip_grads(grads, max_norm, out=None)`` the same, and the gradients scaled
  by min(1, max_norm / (norm + 1e-6)), in place or into ``out``
* ``clip_grad_norm_(parameters, max_norm)`` the same on the parameters' ``.grad``:
  the call and the factor of torch.nn.utils.clip_grad_norm_

Gradients are fp32, bf16 or fp16, mixed as they come, on one device, each
dense in some order of its dimensions.  The squares are summed in 64 bits, in
an order that sizes and types alone give: the same gradients give the same norm,
bit for bit, wherever they lie.  A norm that is infinite or NaN goes into the
factor as it is, as in torch.  Nothing synchronises the device unless
``error_if_nonfinite`` asks.
"""
from __future__ import annotations

from typing import Iterable, Sequence

import torch

from . import ops


def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """sqrt(sum of squares over every element of ``grads``), an fp32 scalar tensor."""
    return ops.grad_norm(list(grads))


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """Scales ``grads`` to a norm of at most ``max_norm`` and returns the norm
    they had (an fp32 scalar tensor).  In place, or into ``out``: tensors of the
    same types, shapes and strides.  Tensors that are written must not overlap
    each other or another gradient: a gradient that is listed twice is refused."""
    return ops.clip_grads(list(grads), float(max_norm), None if out is None else list(out))


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """``clip_grads`` in place on the gradients of ``parameters`` (those that have
    one); a zero when none has.  The arguments are torch's: of the norms only the
    2-norm is offered, ``foreach`` changes nothing.  Unlike there, a gradient that
    is listed twice is refused, and all are on one device."""
    if float(norm_type) != 2.0:
        raise ValueError(f"clip_grad_norm_ offers the 2-norm alone, got norm_type {norm_type}")
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = grad_norm(grads)
        if not torch.isfinite(norm):
            raise RuntimeError(f"the norm of the gradients is {float(norm)}: they are not clipped")
    return clip_grads(grads, max_norm)
