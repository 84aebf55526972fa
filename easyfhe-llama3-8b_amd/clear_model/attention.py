"""Grouped attention of the clear decoder (reference approx/attention.py:134-173
over repeated heads, without lengths or gradients).

``out_i = sum_j softmax_j(scale q_i . k_j) v_j`` over the keys that query i
sees: j below the sequence's length, and where ``causal`` not behind the
query.  No scores are stored; the backward pass computes the probabilities
again from the forward's log-sum-exp.  Gradients of shared key heads are summed
in one fixed order, so equal inputs give equal bits.
"""

from __future__ import annotations

from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from . import _native
from ._native import ATTENTION_ARGS, TYPES


def _rows(x):
    """x and its strides, innermost stride 1, tokens that do not overlap, and
    rows at multiples of 16 bytes; copied if need be."""
    s = x.stride()
    if (s[3] == 1 and not (s[0] | s[1] | s[2]) & 7 and x.shape[3] <= s[1] <= 1 << 23
            and not x.data_ptr() & 15):
        return x, s
    # contiguous() hands back the tensor itself if it is contiguous but misaligned
    x = x.clone(memory_format=torch.contiguous_format)
    return x, x.stride()


def _checked(q, k, v, kv_lens, q_start, scale):
    qs, ks, dtype, dev = q.shape, k.shape, q.dtype, q.device
    if len(qs) != 4 or len(ks) != 4:
        raise ValueError("q is [batch, tokens, heads, dim], k and v [batch, tokens, kv heads, dim].")
    b, n, h, d = qs
    if ks != v.shape or ks[0] != b or ks[3] != d:
        raise ValueError(f"k and v are [{b}, tokens, kv heads, {d}], got {tuple(ks)} and "
                         f"{tuple(v.shape)}.")
    if ks[2] < 1 or h < 1 or h % ks[2]:
        raise ValueError("the query heads are a multiple of the key heads.")
    if d < 8 or d % 8 or d > 128:
        raise ValueError("the head is a multiple of 8, at most 128.")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"attention takes bf16 and fp16, got {dtype}.")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v have one type.")
    if not q.is_cuda or k.device != dev or v.device != dev:
        raise ValueError("q, k and v are on one GPU.")
    lens = starts = 0
    if kv_lens is not None:
        kv_lens = _per_sequence("kv_lens", kv_lens, b, dev)
        lens = kv_lens.data_ptr()
    if q_start is not None:
        q_start = _per_sequence("q_start", q_start, b, dev)
        starts = q_start.data_ptr()
    scale = d ** -0.5 if scale is None else float(scale)
    if not 1.1754943508222875e-38 <= scale < 1e30:
        raise ValueError("the scale is positive and finite in fp32.")
    # the tensors are returned too: they live until the call has been made
    return lens, starts, scale, (kv_lens, q_start)


def _per_sequence(name, x, b, device):
    if x.dtype is not torch.int32 or x.shape != (b,) or x.device != device:
        raise ValueError(f"{name} is int32 [{b}] on q's device.")
    return x.contiguous()


def _pack(q, k, v, ptrs, dims, scale, strides, workspace=0, workspace_bytes=0):
    """ptrs: out, lse, kv_lens, q_start, dout, dq, dk, dv."""
    return ATTENTION_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *ptrs, workspace,
                               workspace_bytes, *dims, scale, *strides)


@lru_cache(maxsize=4096)
def _workspace_bytes(dims, backward):
    """What a call of these sizes needs (the plan depends on nothing else)."""
    args = ATTENTION_ARGS.pack(*([0] * 12), 0, *dims, 1.0, *([0] * 12))
    return _native.query(_native.lib.clear_attention_workspace, args, backward)


def attention_forward(q, k, v, *, causal: bool, kv_lens=None, q_start=None, scale=None):
    """(out, lse) of q [B, Tq, H, D] over k, v [B, Tk, Hk, D]: out is [B, Tq, H, D]
    in q's type, lse fp32 [B, H, Tq].

    Query i of sequence b sees key j where j < kv_lens[b] (int32, all Tk
    without it; what a cache holds beyond is not read into the result) and,
    where ``causal``, j <= i + q_start[b] (int32; Tk - Tq without it, which
    puts the last query at the last key).  A query that sees nothing gets
    zeros and lse = -inf.  ``scale`` is 1/sqrt(D) unless given.  No graph is
    kept: tensors that require gradients go through ``attention``."""
    _native.without_graph("attention", q, k, v)
    lens, starts, scale, _held = _checked(q, k, v, kv_lens, q_start, scale)
    q, qs = _rows(q)
    k, ks = _rows(k)
    v, vs = _rows(v)
    b, n, h, d = shape = q.shape
    dims = (TYPES[q.dtype], b, n, k.shape[1], h, k.shape[2], d, bool(causal))
    out = q.new_empty(shape)
    lse = q.new_empty((b, h, n), dtype=torch.float32)
    need = _workspace_bytes(dims, False)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    args = _pack(q, k, v, (out.data_ptr(), lse.data_ptr(), lens, starts, 0, 0, 0, 0), dims, scale,
                 (qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], 0, 0, 0),
                 ws.data_ptr() if need else 0, need)
    _native.call(_native.lib.clear_attention_forward, args, q.device.index)
    return out, lse


def attention_backward(dout, q, k, v, out, lse, *, causal: bool, kv_lens=None, q_start=None,
                       scale=None):
    """(dq, dk, dv) from the gradient of ``attention_forward``'s output, its
    inputs, and what it returned.  Keys beyond a sequence's length and queries
    that see nothing have gradients of zero."""
    lens, starts, scale, _held = _checked(q, k, v, kv_lens, q_start, scale)
    b, n, h, d = shape = q.shape
    dtype, dev = q.dtype, q.device
    for name, x in (("dout", dout), ("out", out)):
        if x.shape != shape or x.dtype is not dtype or x.device != dev:
            raise ValueError(f"{name} has q's shape, type and device.")
    if lse.shape != (b, h, n) or lse.dtype is not torch.float32 or lse.device != dev:
        raise ValueError(f"lse is fp32 [{b}, {h}, {n}] on q's device.")
    q, qs = _rows(q)
    k, ks = _rows(k)
    v, vs = _rows(v)
    dout, ds = _rows(dout)
    out, lse = out.contiguous(), lse.contiguous()
    if out.data_ptr() & 15:
        out = out.clone()
    dims = (TYPES[dtype], b, n, k.shape[1], h, k.shape[2], d, bool(causal))
    dq, dk, dv = q.new_empty(shape), k.new_empty(k.shape), v.new_empty(v.shape)
    need = _workspace_bytes(dims, True)
    ws = q.new_empty(need, dtype=torch.uint8)
    args = _pack(q, k, v, (out.data_ptr(), lse.data_ptr(), lens, starts, dout.data_ptr(),
                           dq.data_ptr(), dk.data_ptr(), dv.data_ptr()), dims, scale,
                 (qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], ds[0], ds[1],
                  ds[2]), ws.data_ptr(), need)
    _native.call(_native.lib.clear_attention_backward, args, dev.index)
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, kv_lens, q_start, scale):
        out, lse = attention_forward(q, k, v, causal=causal, kv_lens=kv_lens, q_start=q_start,
                                     scale=scale)
        ctx.save_for_backward(q, k, v, out, lse, kv_lens, q_start)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, kv_lens, q_start = ctx.saved_tensors
        grads = attention_backward(dout, q, k, v, out, lse, causal=ctx.causal, kv_lens=kv_lens,
                                   q_start=q_start, scale=ctx.scale)
        return grads + (None, None, None, None)


def attention(q, k, v, *, causal: bool, kv_lens=None, q_start=None, scale=None):
    """``attention_forward``'s output, with gradients."""
    return _Attention.apply(q, k, v, causal, kv_lens, q_start, scale)


__all__ = ["attention", "attention_backward", "attention_forward"]
