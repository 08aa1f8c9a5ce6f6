"""The global gradient norm over many tensors, and clipping by it, for B200.

* ``grad_norm(grads, norm_type)`` -- the norm, an fp32 scalar on the device;
* ``clip_grads(grads, max_norm, norm_type, out)`` -- the norm, and every
  gradient times ``min(1, max_norm / (norm + 1e-6))``, in place or into ``out``
  (e.g. the fp32 main gradients of bf16 ones);
* ``clip_grad_norm_(parameters, max_norm, norm_type, error_if_nonfinite)`` --
  the same on ``parameter.grad``, with torch.nn.utils' arguments.

``norm_type`` is 2 or inf.  fp32, fp16 and bf16 may be mixed in one list; all
tensors are on one GPU.  Nothing synchronises (``error_if_nonfinite=True``
reads the norm and does).  A NaN gradient makes the norm and every output NaN;
an infinite norm scales by zero.  Equal inputs give equal bits.  Tensors with
holes between their elements are clipped through a dense copy.  A tensor may
stand in the list once.  Every written tensor counts a new version, whether or
not its values change, so autograd refuses a graph that saved it before.
Tensors with a forward-mode tangent raise NotImplementedError.
"""
from __future__ import annotations

import math
from collections.abc import Iterable

import torch

from bevk import load_extension

CLIP_EPS = 1e-6

_ext = None


def _load_ext():
    global _ext
    if _ext is None:
        _ext = load_extension("_bevk_train_ext")
    return _ext


def _is_inf(norm_type) -> bool:
    norm_type = float(norm_type)
    if norm_type == 2.0:
        return False
    if norm_type == math.inf:
        return True
    raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """Norm over all elements of the tensors, an fp32 scalar tensor."""
    return _load_ext().grad_clip(list(grads), None, CLIP_EPS, _is_inf(norm_type), None)


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None) -> torch.Tensor:
    """Scales the gradients (in place, or into the tensors of ``out``) to a norm
    of at most ``max_norm``; returns the norm before that."""
    return _load_ext().grad_clip(list(grads), float(max_norm), CLIP_EPS, _is_inf(norm_type),
                                 None if out is None else list(out))


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the gradients of ``parameters`` (a tensor or an iterable of them)
    in place and returns their norm.  With ``error_if_nonfinite`` a norm that is
    not finite raises RuntimeError and leaves the gradients as they were."""
    inf_norm = _is_inf(norm_type)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    elif not isinstance(parameters, Iterable):
        raise TypeError("parameters must be a tensor or an iterable of tensors")
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the gradients' norm of order {float(norm_type)} is not finite; "
                               "pass error_if_nonfinite=False to scale them all the same")
    return _load_ext().grad_clip(grads, float(max_norm), CLIP_EPS, inf_norm, None)


__all__ = ["grad_norm", "clip_grads", "clip_grad_norm_", "CLIP_EPS"]
