"""Cross entropy of a large vocabulary, straight from the hidden states.

``loss_n = log sum_v exp(hidden_n . weight_v) - hidden_n . weight_target(n)``.
The logits of all tokens are never stored: the forward pass keeps a maximum
and a sum for each tile of the vocabulary, and the backward pass goes over the
vocabulary in pieces and computes each piece's logits again.
"""

from __future__ import annotations

from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from . import _native
from ._native import LOSS_ARGS, TYPES


def _rows(x):
    """Innermost stride 1, a width that is a multiple of 8, and rows at
    multiples of 16 bytes; copied (with zeros behind) if need be."""
    d = x.shape[1]
    if (d % 8 == 0 and x.stride(1) == 1 and x.stride(0) % 8 == 0 and d <= x.stride(0) <= 1 << 21
            and x.data_ptr() % 16 == 0):
        return x
    y = x.new_zeros((x.shape[0], -(-d // 8) * 8))
    y[:, :d] = x
    return y


def _checked(hidden, weight, targets):
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError(f"hidden is [tokens, width] and weight [vocab, width], got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}.")
    if weight.shape[0] < 1 or not 1 <= weight.shape[1] <= 1 << 20:
        raise ValueError("at least one class, and a width of 1 to 2^20.")
    if hidden.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"the loss takes bf16 and fp16, got {hidden.dtype}.")
    if weight.dtype != hidden.dtype:
        raise ValueError("hidden and weight have one type.")
    if targets.dtype != torch.int64 or targets.shape != hidden.shape[:1]:
        raise ValueError(f"targets are int64 [{hidden.shape[0]}].")
    if not hidden.is_cuda or weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError("hidden, weight and targets are on one GPU.")


@lru_cache(maxsize=4096)
def _workspace_bytes(dims, backward):
    """What a call of these sizes needs (the plan depends on nothing else)."""
    args = LOSS_ARGS.pack(*([0] * 10), *dims, 0, 0, 0)
    return _native.query(_native.lib.clear_loss_workspace, args, backward)


def _run(fn, backward, hidden, weight, targets, ptrs, ignore_index):
    """ptrs: loss, lse, dloss, dhidden, dweight."""
    n, d = hidden.shape
    dims = (TYPES[hidden.dtype], n, weight.shape[0], d)
    need = _workspace_bytes(dims, backward)
    ws = hidden.new_empty(need, dtype=torch.uint8)
    args = LOSS_ARGS.pack(hidden.data_ptr(), weight.data_ptr(), targets.data_ptr(), *ptrs,
                          ws.data_ptr(), need, *dims, ignore_index, hidden.stride(0),
                          weight.stride(0))
    _native.call(fn, args, hidden.device.index)


def linear_cross_entropy_forward(hidden, weight, targets, *, ignore_index: int = -100):
    """(loss, lse), fp32 [N], of hidden [N, D] through weight [V, D] at the int64
    targets [N].  Where the target is ``ignore_index`` both are 0; where it is
    no class the loss is NaN.  No graph is kept: tensors that require gradients
    go through ``linear_cross_entropy``."""
    _native.without_graph("linear_cross_entropy", hidden, weight)
    _checked(hidden, weight, targets)
    n = hidden.shape[0]
    loss = hidden.new_empty(n, dtype=torch.float32)
    lse = hidden.new_empty(n, dtype=torch.float32)
    if n:
        hidden, weight, targets = _rows(hidden), _rows(weight), targets.contiguous()
        _run(_native.lib.clear_loss_forward, False, hidden, weight, targets,
             (loss.data_ptr(), lse.data_ptr(), 0, 0, 0), int(ignore_index))
    return loss, lse


def linear_cross_entropy_backward(dloss, hidden, weight, targets, lse, *,
                                  ignore_index: int = -100):
    """(dhidden, dweight), in the inputs' type, from the gradient of the losses
    (fp32 [N]) and the forward's lse.  Tokens with ``ignore_index`` add nothing,
    whatever their dloss holds; in fp16 the gradients' range is the caller's
    (scale dloss)."""
    _checked(hidden, weight, targets)
    n, d = hidden.shape
    for name, x in (("dloss", dloss), ("lse", lse)):
        if x.dtype != torch.float32 or x.shape != (n,) or x.device != hidden.device:
            raise ValueError(f"{name} is fp32 [{n}] on hidden's device.")
    if n == 0:
        return torch.empty_like(hidden), torch.zeros_like(weight)
    hidden, weight, targets = _rows(hidden), _rows(weight), targets.contiguous()
    dloss, lse = dloss.contiguous(), lse.contiguous()
    wide = hidden.shape[1]
    dh = hidden.new_empty((n, wide))
    dw = hidden.new_empty((weight.shape[0], wide))
    _run(_native.lib.clear_loss_backward, True, hidden, weight, targets,
         (0, lse.data_ptr(), dloss.data_ptr(), dh.data_ptr(), dw.data_ptr()), int(ignore_index))
    if wide != d:
        dh, dw = dh[:, :d].contiguous(), dw[:, :d].contiguous()
    return dh, dw


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index):
        loss, lse = linear_cross_entropy_forward(hidden, weight, targets,
                                                 ignore_index=ignore_index)
        ctx.save_for_backward(hidden, weight, targets, lse)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        hidden, weight, targets, lse = ctx.saved_tensors
        return linear_cross_entropy_backward(dloss, hidden, weight, targets, lse,
                                             ignore_index=ctx.ignore_index) + (None, None)


def linear_cross_entropy(hidden, weight, targets, *, ignore_index: int = -100,
                         reduction: str = "mean"):
    """The loss with gradients: "mean" over the tokens that count (NaN where
    none does, as the quotient says), "sum", or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction is mean, sum or none, got {reduction!r}.")
    loss = _LinearCrossEntropy.apply(hidden, weight, targets, ignore_index)
    if reduction == "none":
        return loss
    if reduction == "sum":
        return loss.sum()
    return loss.sum() / (targets != ignore_index).sum()


__all__ = ["linear_cross_entropy", "linear_cross_entropy_backward",
           "linear_cross_entropy_forward"]
