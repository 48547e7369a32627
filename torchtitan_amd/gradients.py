"""The global norm of a model's gradients, and their clipping, before the optimizer step.

Counterpart of the clipping step of the reference's trainer (torchtitan/distributed/utils.py:466-472 and the function
around it), with torch's own signatures.  bf16 and float32 gradients on a GPU run in two passes over all of them, in as few
launches as tables of 160 tensors take; everything else runs through torch's functions.
"""
from __future__ import annotations

import torch

from . import _lib, ops


def _ours(grads, norm_type: float) -> bool:
    device = grads[0].device
    return norm_type in ops.GRAD_NORMS and ops.plain_rows(*grads) and all(
        t.device == device and t.layout == torch.strided for t in grads)


def get_total_norm(tensors, norm_type: float = 2.0, error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """The norm of all tensors taken as one vector, as ``torch.nn.utils.get_total_norm``; float32 whatever their type, summed
    in float64, where they are bf16 or float32 tensors on one GPU and the norm is 2, 1 or infinity."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    norm_type = float(norm_type)
    if not tensors or not _ours(tensors, norm_type):
        return torch.nn.utils.get_total_norm(tensors, norm_type, error_if_nonfinite, foreach)
    with torch.no_grad():
        norm = ops.grad_norm([t if ops.is_dense(t) else t.contiguous() for t in tensors], norm_type)
    if error_if_nonfinite and not bool(norm.isfinite()):
        raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it cannot be "
                           "clipped. To disable this error and scale the gradients by the non-finite norm anyway, set "
                           "`error_if_nonfinite=False`")
    return norm


def _grads(parameters):
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    return [p.grad for p in parameters if p.grad is not None]


def _apart(tensors) -> bool:
    """No element of one lies between the first and the last of another."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
                   for t in tensors if t.numel())
    return all(end <= start for (_, end), (start, _) in zip(spans, spans[1:]))


def clip_grads_with_norm_(parameters, max_norm: float, total_norm: torch.Tensor, foreach: bool | None = None) -> None:
    """Scales the parameters' gradients in place by min(1, max_norm / (total_norm + 1e-6)), as
    ``torch.nn.utils.clip_grads_with_norm_``; nothing is read or written where that is exactly 1 (a gradient that is not one
    run of memory is copied and written back either way)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = _grads(parameters)
    if not grads:
        return
    if not _ours(grads, 2.0) or type(total_norm) is not torch.Tensor:
        torch.nn.utils.clip_grads_with_norm_(parameters, max_norm, total_norm, foreach)
        return
    with torch.no_grad():
        total_norm = total_norm.to(device=grads[0].device, dtype=torch.float32)
        # copies that share memory with another gradient are written back before the next one is read
        together = [grads] if all(ops.is_dense(t) for t in grads) or _apart(grads) else [[t] for t in grads]
        for some in together:
            runs = [t if ops.is_dense(t) else t.contiguous() for t in some]
            ops.grad_scale_(runs, total_norm, float(max_norm))
            for t, run in zip(some, runs):
                if run is not t:
                    t.copy_(run)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: bool | None = None) -> torch.Tensor:
    """Clips the gradients of `parameters` in place by their norm taken as one vector and returns that norm, as
    ``torch.nn.utils.clip_grad_norm_``.  A caller whose gradients are spread over ranks adds up the powers of
    ``get_total_norm`` and calls ``clip_grads_with_norm_`` with the result."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if parameters and norm_type in ops.GRAD_NORMS and not error_if_nonfinite and ops.native_rows(parameters[0]):
        norm = _lib.blocks().clip_gradients(parameters, max_norm, ops.GRAD_NORMS[norm_type])
        if norm is not None:
            return norm
    total_norm = get_total_norm(_grads(parameters), norm_type, error_if_nonfinite, foreach)
    clip_grads_with_norm_(parameters, max_norm, total_norm, foreach)
    return total_norm
