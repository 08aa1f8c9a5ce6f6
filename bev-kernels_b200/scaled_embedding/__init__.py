"""Embedding lookup with scaling and its gradient, for B200: learned positions,
bird's-eye-view and object queries, token tables.

* ``scaled_embedding(ids, weight, scale, padding_idx)`` -- ``scale * weight[ids]``
  with a gradient (``ScaledEmbeddingFunction``); ``ScaledEmbedding`` is the module.
* ``scaled_embedding_forward`` / ``scaled_embedding_backward`` -- the two passes;
  the backward can add into an existing gradient (e.g. an fp32 main gradient of a
  bf16 table), touching only the rows that ids name.

ids are int64 or int32 of any shape; the table is fp32, fp16 or bf16.  An id
outside [0, rows) reads as a row of zeros and gives no gradient; the row
``padding_idx`` is read as any other and gets no gradient.  Sums are fp32 and
their order is fixed by the ids alone, so equal inputs give equal bits.  CUDA
tensors only; there is no forward-mode derivative (a tangent raises
NotImplementedError).
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from bevk import load_extension

_ext = None


def _load_ext():
    global _ext
    if _ext is None:
        _ext = load_extension("_bevk_train_ext")
    return _ext


def _padding(padding_idx, rows: int) -> int:
    """padding_idx as a row number (negative ones count from the end), -1: none."""
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"padding_idx {padding_idx} is not a row of {rows}")
    return padding_idx % rows


def scaled_embedding_forward(weight: torch.Tensor, ids: torch.Tensor,
                             scale: float = 1.0) -> torch.Tensor:
    """weight [rows, dim], ids [*] -> scale * weight[ids], [*, dim]."""
    return _load_ext().embedding_forward(weight, ids, scale)


def scaled_embedding_backward(grad_output: torch.Tensor, ids: torch.Tensor, num_embeddings: int,
                              scale: float = 1.0, padding_idx: int | None = None,
                              grad_weight: torch.Tensor | None = None) -> torch.Tensor:
    """-> the weight's gradient [num_embeddings, dim] in grad_output's dtype, with
    zeros in the rows that no id names.  Where ``grad_weight`` (grad_output's dtype
    or fp32) is given, the gradient is added to it instead, in place, and it is
    returned; it counts a new version."""
    return _load_ext().embedding_backward(grad_output, ids, num_embeddings, scale,
                                          _padding(padding_idx, num_embeddings), grad_weight)


class ScaledEmbeddingFunction(Function):
    """autograd Function of (ids, weight, scale, padding_idx)."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.rows, ctx.scale, ctx.padding_idx = weight.size(0), scale, padding_idx
        ctx.save_for_backward(ids)
        return scaled_embedding_forward(weight, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        ids, = ctx.saved_tensors
        return None, scaled_embedding_backward(grad_output, ids, ctx.rows, ctx.scale,
                                               ctx.padding_idx), None, None


def scaled_embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None) -> torch.Tensor:
    """scale * weight[ids]; differentiable in weight."""
    _padding(padding_idx, weight.size(0))
    return ScaledEmbeddingFunction.apply(ids, weight, scale, padding_idx)


class ScaledEmbedding(nn.Module):
    """``torch.nn.Embedding`` (parameter name, initialisation) whose rows are
    multiplied by ``scale`` when they are looked up."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None,
                 scale: float = 1.0):
        super().__init__()
        _padding(padding_idx, num_embeddings)
        self.num_embeddings, self.embedding_dim = num_embeddings, embedding_dim
        self.padding_idx, self.scale = padding_idx, scale
        self.weight = nn.Parameter(torch.empty(num_embeddings, embedding_dim))
        nn.init.normal_(self.weight)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].fill_(0)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return scaled_embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        s = f"{self.num_embeddings}, {self.embedding_dim}"
        if self.padding_idx is not None:
            s += f", padding_idx={self.padding_idx}"
        return s + f", scale={self.scale}"


__all__ = ["scaled_embedding_forward", "scaled_embedding_backward", "ScaledEmbeddingFunction",
           "scaled_embedding", "ScaledEmbedding"]
