"""The decoder in the clear: the layers that the encrypted programs evaluate
(reference approx/layer.py:64-149 with exact RMSNorm, SiLU and softmax), in
bf16 or fp16 on the device, with a cache for generating and gradients for
adapting.

Weights have the encrypted layers' form: [out, in] projections q, k, v, o,
gate, up, down, and RMSNorms without weights of their own (the encrypted
programs take them into the projections behind) unless some are given.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.nn import functional as F

from .attention import attention, attention_forward
from .loss import linear_cross_entropy, linear_cross_entropy_forward
from .rope import RopeTable, apply_rope, rope

PROJECTIONS = ("q", "k", "v", "o", "gate", "up", "down")


@dataclass
class ClearCache:
    """Keys and values of every layer, [B, capacity, Hk, D] each, and how many of
    a sequence's places hold one.

    ``bound`` is the most places that the host knows a sequence to hold; None
    where it knows nothing, as where the caller has filled the cache (whoever
    writes ``lens`` sets it to None).  The lengths are read from the device only
    where the bound leaves no room."""

    keys: list
    values: list
    lens: torch.Tensor
    bound: int | None = None

    @property
    def capacity(self) -> int:
        return self.keys[0].shape[1]

    def _check_batch(self, b: int) -> None:
        if self.lens.shape != (b,):
            raise ValueError(f"{b} sequences, a cache of {len(self.lens)}.")

    def _take_place(self) -> None:
        """Counts one more token a sequence, or refuses it.  A captured call has no
        host to ask when it is replayed: `decode` keeps those inside the cache."""
        if self.lens.is_cuda and torch.cuda.is_current_stream_capturing():
            self.bound = None
            return
        if self.bound is None or self.bound >= self.capacity:
            self.bound = int(self.lens.max()) if len(self.lens) else 0
        if self.bound >= self.capacity:
            raise ValueError(f"a sequence has no room in its cache of {self.capacity}.")
        self.bound += 1


def rms_norm(x, weight=None, eps: float = 1e-5):
    """x / sqrt(mean x^2 + eps), in fp32, rounded once."""
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    return y.to(x.dtype)


def _linear(x, w):
    """x @ w^T over the last axis, as one product of two matrices."""
    return (x.reshape(-1, x.shape[-1]) @ w.t()).reshape(*x.shape[:-1], w.shape[0])


class ClearDecoder:
    """``layers``: one mapping a layer with the seven projections and optionally
    "input_norm" and "post_attention_norm"; ``embedding`` and ``lm_head``
    [vocab, hidden].  Tensors are used as they are: leaves that require
    gradients get them."""

    def __init__(self, layers, embedding, lm_head, *, heads: int, kv_heads: int, head_dim: int,
                 table: RopeTable | None = None, final_norm=None, eps: float = 1e-5):
        self.layers = [dict(w) for w in layers]
        if not self.layers:
            raise ValueError("no layers.")
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("the query heads are a multiple of the key heads.")
        width = embedding.shape[1]
        rows = dict(q=heads * head_dim, k=kv_heads * head_dim, v=kv_heads * head_dim, o=width)
        for w in self.layers:
            for name in PROJECTIONS:
                if name not in w:
                    raise ValueError(f"a layer has no {name!r} projection.")
            for name, n in rows.items():
                if w[name].shape[0] != n:
                    raise ValueError(f"{name} has {w[name].shape[0]} rows, not {n}.")
        if lm_head.shape != embedding.shape:
            raise ValueError("the embedding and the LM head are [vocab, hidden].")
        self.embedding, self.lm_head, self.final_norm = embedding, lm_head, final_norm
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, head_dim, float(eps)
        self.table = RopeTable(head_dim) if table is None else table
        if self.table.dim != head_dim:
            raise ValueError("the rotary table is for another head.")

    # ------------------------------------------------------------- layers

    def _qkv(self, w, x):
        n = rms_norm(x, w.get("input_norm"), self.eps)
        split = lambda y, h: y.reshape(*x.shape[:2], h, self.head_dim)  # noqa: E731
        return (split(_linear(n, w["q"]), self.heads), split(_linear(n, w["k"]), self.kv_heads),
                split(_linear(n, w["v"]), self.kv_heads))

    def _rest(self, w, x, att):
        h = x + _linear(att.reshape(*x.shape[:2], -1), w["o"])
        n = rms_norm(h, w.get("post_attention_norm"), self.eps)
        return h + _linear(F.silu(_linear(n, w["gate"])) * _linear(n, w["up"]), w["down"])

    def _ids(self, ids):
        if ids.dim() != 2 or ids.dtype != torch.int64:
            raise ValueError("token ids are int64 [batch, tokens].")
        return F.embedding(ids, self.embedding)

    def hidden(self, ids, lens=None):
        """The layers' output [B, T, hidden] before the final norm, with gradients;
        ``lens`` (int32 [B]) hides a sequence's padding."""
        x = self._ids(ids)
        places = torch.arange(ids.shape[1], device=ids.device, dtype=torch.int32)
        for w in self.layers:
            q, k, v = self._qkv(w, x)
            q, k = apply_rope(self.table, q, k, positions=places)
            x = self._rest(w, x, attention(q, k, v, causal=True, kv_lens=lens))
        return x

    # ------------------------------------------------------ training, scoring

    def loss(self, ids, targets, lens=None, *, ignore_index: int = -100, reduction: str = "mean"):
        """Cross entropy of ``targets`` [B, T], with gradients."""
        x = rms_norm(self.hidden(ids, lens), self.final_norm, self.eps)
        return linear_cross_entropy(x.reshape(-1, x.shape[-1]), self.lm_head, targets.reshape(-1),
                                    ignore_index=ignore_index, reduction=reduction)

    @torch.no_grad()
    def score(self, hidden, targets, *, ignore_index: int = -100):
        """Losses [N] of final hidden states [N, hidden], such as a decrypted
        prefill's, before the final norm: normed in fp32, then rounded once."""
        x = rms_norm(torch.as_tensor(hidden).to(self.lm_head.device, torch.float32),
                     self.final_norm, self.eps).to(self.lm_head.dtype)
        return linear_cross_entropy_forward(x, self.lm_head, targets, ignore_index=ignore_index)[0]

    # ------------------------------------------------------------ generating

    def cache(self, batch: int, capacity: int) -> ClearCache:
        new = lambda: self.embedding.new_zeros(batch, capacity, self.kv_heads, self.head_dim)  # noqa: E731
        return ClearCache([new() for _ in self.layers], [new() for _ in self.layers],
                          torch.zeros(batch, dtype=torch.int32, device=self.embedding.device), 0)

    def logits(self, hidden):
        return _linear(rms_norm(hidden, self.final_norm, self.eps), self.lm_head)

    @torch.no_grad()
    def prefill(self, ids, cache: ClearCache, lens=None):
        """Fills an empty cache with the prompts [B, T] of the given lengths (int32
        [B]; taken as 0 below and as T beyond), and returns the logits [B, vocab]
        behind each prompt's last token."""
        x = self._ids(ids)
        b, t = ids.shape
        cache._check_batch(b)
        if t > cache.capacity or t < 1:
            raise ValueError(f"prompts of {t} tokens, a cache of {cache.capacity}.")
        if lens is None:
            lens = torch.full((b,), t, dtype=torch.int32, device=ids.device)
        elif lens.shape != (b,) or lens.dtype != torch.int32 or lens.device != ids.device:
            raise ValueError(f"lens is int32 [{b}] on the ids' device.")
        else:
            lens = lens.clamp(0, t)
        places = torch.arange(t, device=ids.device, dtype=torch.int32)
        for w, ck, cv in zip(self.layers, cache.keys, cache.values):
            q, k, v = self._qkv(w, x)
            q, k = rope(self.table, q, k, positions=places)
            ck[:, :t], cv[:, :t] = k, v
            x = self._rest(w, x, attention_forward(q, k, v, causal=True, kv_lens=lens)[0])
        cache.lens.copy_(lens)
        cache.bound = t
        at = (lens.long() - 1).clamp(min=0)
        return self.logits(x[torch.arange(b, device=ids.device), at])

    @torch.no_grad()
    def decode(self, ids, cache: ClearCache):
        """One more token [B] a sequence: its logits [B, vocab].  Refused where a
        sequence has no room left; in a replayed graph, which the host does not
        see, a full sequence's last place is written again."""
        x = self._ids(ids[:, None])
        cache._check_batch(len(ids))
        cache._take_place()
        places = cache.lens.clamp(0, cache.capacity - 1)
        rows, at, lens = torch.arange(len(ids), device=ids.device), places.long(), places + 1
        places = places[:, None]
        for w, ck, cv in zip(self.layers, cache.keys, cache.values):
            q, k, v = self._qkv(w, x)
            q, k = rope(self.table, q, k, positions=places)
            ck[rows, at], cv[rows, at] = k[:, 0], v[:, 0]
            x = self._rest(w, x, attention_forward(q, ck, cv, causal=False, kv_lens=lens)[0])
        cache.lens.copy_(lens)
        return self.logits(x[:, 0])


__all__ = ["ClearCache", "ClearDecoder", "rms_norm"]
