"""The keys and values of the tokens that a model has seen, in pages, for generating text one token at a time."""
from __future__ import annotations

from typing import Optional

import torch

from .. import ops


class PagedKVCache:
    """One cache for all layers of a model and ``batch`` sequences of up to ``max_len`` tokens (rounded up to whole pages).  A
    sequence that outgrows its pages raises IndexError on the CPU; on the GPU the token is not kept, and
    ``parallel.health.check_device_status()`` raises.

    ``k`` and ``v`` are [n_layer, pages, n_kv_head, page_size, head_dim]; ``page_table`` (int32 [batch, pages of a sequence]) and
    ``lengths`` (int32 [batch], tokens held) live on the device, so that a captured decoding step stays correct.

    With ``window`` (and ``sinks``) a sequence keeps only what the next token sees: the pages of its sinks and a ring of
    ``ceil(window / page_size) + 1`` pages, whatever ``max_len`` is.

    A model's ``forward(idx, cache=cache)`` appends the tokens and returns the logits of the next ones (see ``models``)::

        cache = model.new_cache(batch, max_len)
        logits = model(prompts, cache=cache, counts=counts)     # [batch, vocab_size]
        logits = model(logits.argmax(-1, keepdim=True), cache=cache)
    """

    def __init__(self, n_layer: int, batch: int, max_len: int, n_kv_head: int, head_dim: int, page_size: int = 64,
                 window: Optional[int] = None, sinks: int = 0, device=None, dtype=torch.float32):
        if min(n_layer, batch, max_len, n_kv_head, head_dim, page_size) < 1:
            raise ValueError("PagedKVCache: sizes must be positive")
        if (window is not None and window < 1) or sinks < 0:
            raise ValueError("PagedKVCache: window must be at least 1 and sinks must not be negative")
        self.batch, self.max_len, self.page_size = batch, max_len, page_size
        self.window, self.sinks = window, sinks
        width = (max_len + page_size - 1) // page_size
        slots = torch.arange(width, dtype=torch.int32)
        held = width
        if window is not None:
            first = (sinks + page_size - 1) // page_size
            ring = (window + page_size - 1) // page_size + 1
            if first + ring < width:
                held = first + ring
                slots = torch.where(slots < first, slots, first + (slots - first) % ring)
        table = slots[None, :] + held * torch.arange(batch, dtype=torch.int32)[:, None]
        self.page_table = table.to(device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        # zeros, not garbage: rows that no token was written to are not read, but may be printed or saved
        self.k = torch.zeros(n_layer, batch * held, n_kv_head, page_size, head_dim, device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self._empty = True
        self._starts = self._ends = self._counts = None

    def bytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()

    def reset(self) -> None:
        """Forgets all tokens."""
        self.lengths.zero_()
        self._empty = True

    def begin(self, idx: torch.Tensor, counts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Called by a model before its layers: the positions of the new tokens idx [batch, T], int64 [batch, T].  ``counts``
        (int32 [batch]): how many of the T tokens of a sequence are real, the others being padding behind them; a count outside
        0 .. T is taken as the nearer of the two."""
        B, T = idx.shape
        if B != self.batch:
            raise ValueError(f"PagedKVCache: a batch of {B} for a cache of {self.batch} sequences")
        if T < 1 or T > self.max_len:
            raise ValueError(f"PagedKVCache: {T} tokens for a cache of {self.max_len} positions")
        if T > 1 and not self._empty:
            raise ValueError("PagedKVCache: several tokens at once go into an empty cache only; reset() it, or feed them one by one")
        if counts is not None and (counts.dtype != torch.int32 or counts.shape != (B,) or counts.device != self.lengths.device):
            raise ValueError(f"PagedKVCache: counts must be an int32 tensor of {B} elements on {self.lengths.device}")
        if counts is not None:
            counts = counts.clamp(0, T)     # a larger one would count rows that no token was written to
        self._starts, self._counts = self.lengths, counts
        self._ends = self.lengths + (T if counts is None else counts)
        return self.lengths[:, None].long() + torch.arange(T, device=idx.device)

    def attend(self, layer: int, qkv: torch.Tensor, n_head: int, theta: Optional[float] = None) -> torch.Tensor:
        """Appends the tokens of the projection qkv [batch, T, (n_head + 2 n_kv_head) * head_dim] to a layer's pages and returns
        their attention [batch, T, n_head, head_dim]: a prompt's over itself, a single token's over the cache."""
        k, v = self.k[layer], self.v[layer]
        n_kv, hd = k.shape[1], k.shape[3]
        T = qkv.shape[1]
        out = ops.cache_append(qkv, k, v, self.page_table, self._starts, n_head, n_kv, theta=theta, counts=self._counts,
                               window=self.window, sinks=self.sinks, return_k=T > 1)
        if T == 1:
            return ops.paged_attention(out[:, 0], k, v, self.page_table, self._ends, self.window, self.sinks)[:, None]
        # Without a window ops.causal_attention gives the same sums: with heads of 64 it takes 35 us where this takes 54 (a prompt
        # of 1999, 32 / 8 heads; 374 and 463 us at 8192), with heads of 128 50 and 46 (580 each; 9.0 and 10 ms at 32768).  It
        # rounds the probabilities of bf16 models and lets a NaN reach earlier rows; here a prompt is as exact as the tokens behind it.
        values = qkv.unflatten(-1, (n_head + 2 * n_kv, hd))[:, :, n_head + n_kv:]
        return ops.window_attention(*out, values, self.window, self.sinks)

    def end(self) -> None:
        """Called by a model behind its layers."""
        self.lengths.copy_(self._ends)
        self._empty = False
        self._starts = self._ends = self._counts = None

    def last_rows(self, x: torch.Tensor) -> torch.Tensor:
        """Of the hidden states x [batch, T, C] of the tokens in hand those of each sequence's last real one, [batch, C]."""
        if x.shape[1] == 1:
            return x[:, 0]
        if self._counts is None:
            return x[:, -1]
        last = (self._counts.long() - 1).clamp_(min=0)
        return x[torch.arange(x.shape[0], device=x.device), last]
