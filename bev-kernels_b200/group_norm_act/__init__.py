"""Group norm with a fused activation on channels-last tensors, for B200.

``y = act(weight * (x - mean) * rstd + bias)`` per (image, group), the norm
that follows a (deformable) convolution.  Channels-last outputs, as the
``*_nhwc`` functions of ``modulated_deform_conv`` and its Pack module on
channels-last input give them, go in as they are; ``modulated_deform_conv2d``,
the Pack with groups and the Pack on contiguous input return NCHW, which is
copied first.

* ``group_norm_act(input, num_groups, weight, bias, eps, act)`` -- with
  gradients (``GroupNormActFunction``); ``GroupNormAct`` is the module.
* ``group_norm_act_forward`` / ``group_norm_act_backward`` -- the two passes
  for callers that keep the statistics themselves.

``input`` is [N, C, *spatial] in fp32, fp16 or bf16; ``weight`` and ``bias``
share its dtype or are fp32.  Statistics and sums are fp32 and the result is
rounded once.  Channels-last memory (also with a wider pixel stride, e.g. a
channel slice) is read in place; any other layout is first copied to it by
torch, input and gradient alike (6x256x58x100 bf16: 14 us become 50, the
backward's 26 become 97).  The output and ``grad_input`` are channels-last.
Every image takes an SM of its own while it is worked on, so thousands of
images of a few pixels are slow (20000 x 256 x 1 x 1: 567 us).  ``act`` is
"none", "relu" or "silu".  CUDA tensors only; there is no forward-mode
derivative (a tangent raises NotImplementedError).
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from bevk import load_extension

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}

_ext = None


def _load_ext():
    global _ext
    if _ext is None:
        _ext = load_extension("_bevk_train_ext")
    return _ext


def _act(act: str) -> int:
    try:
        return ACTIVATIONS[act]
    except (KeyError, TypeError):
        raise ValueError(f"act must be one of {sorted(ACTIVATIONS)}, got {act!r}") from None


def group_norm_act_forward(input: torch.Tensor, num_groups: int,
                           weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, eps: float = 1e-5,
                           act: str = "none"):
    """-> (output, mean, rstd); mean and rstd are fp32 [N, num_groups]."""
    return _load_ext().group_norm_act_forward(input, num_groups, weight, bias, eps, _act(act),
                                              True)


def group_norm_act_backward(grad_output: torch.Tensor, input: torch.Tensor, mean: torch.Tensor,
                            rstd: torch.Tensor, num_groups: int,
                            weight: torch.Tensor | None = None,
                            bias: torch.Tensor | None = None, act: str = "none",
                            needs=(True, True, True)):
    """-> (grad_input, grad_weight, grad_bias) from the statistics that the
    forward returned.  ``needs`` says which to compute (None in the place of
    the others, and of the gradient of a weight or bias that is None)."""
    return _load_ext().group_norm_act_backward(
        grad_output, input, mean, rstd, num_groups, weight, bias, _act(act), bool(needs[0]),
        bool(needs[1]) and weight is not None, bool(needs[2]) and bias is not None)


class GroupNormActFunction(Function):
    """autograd Function of (input, num_groups, weight, bias, eps, act)."""

    @staticmethod
    def forward(ctx, input, num_groups, weight, bias, eps, act):
        output, mean, rstd = group_norm_act_forward(input, num_groups, weight, bias, eps, act)
        ctx.num_groups, ctx.act = num_groups, act
        ctx.save_for_backward(input, mean, rstd, weight, bias)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        input, mean, rstd, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = group_norm_act_backward(grad_output, input, mean, rstd, ctx.num_groups, weight,
                                        bias, ctx.act, (need[0], need[2], need[3]))
        return grads[0], None, grads[1], grads[2], None, None


def group_norm_act(input: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5,
                   act: str = "none") -> torch.Tensor:
    """Group norm and activation; differentiable in input, weight and bias."""
    if torch.is_grad_enabled() and (input.requires_grad
                                    or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return GroupNormActFunction.apply(input, num_groups, weight, bias, eps, act)
    return _load_ext().group_norm_act_forward(input, num_groups, weight, bias, eps, _act(act),
                                              False)[0]


class GroupNormAct(nn.Module):
    """``torch.nn.GroupNorm`` (parameter names, initialisation) with an
    activation behind it."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5,
                 affine: bool = True, act: str = "none"):
        super().__init__()
        if num_groups <= 0 or num_channels % num_groups:
            raise ValueError("num_channels must be divisible by num_groups")
        _act(act)
        self.num_groups, self.num_channels, self.eps, self.act = num_groups, num_channels, eps, act
        self.affine = affine
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels))
            self.bias = nn.Parameter(torch.zeros(num_channels))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return group_norm_act(input, self.num_groups, self.weight, self.bias, self.eps, self.act)

    def extra_repr(self) -> str:
        return (f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.affine}, "
                f"act={self.act!r}")


__all__ = ["group_norm_act_forward", "group_norm_act_backward", "GroupNormActFunction",
           "group_norm_act", "GroupNormAct", "ACTIVATIONS"]
