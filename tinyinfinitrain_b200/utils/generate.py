"""Text generation over a key-value cache: the captured decoding step and a loop around it."""
from __future__ import annotations

from typing import Callable, List, Optional, Sequence

import torch

from ..parallel.health import check_device_status


class DecodeStep:
    """One new token of every sequence of a cache: ``step(tokens)`` with tokens int64 [batch] appends them and returns the
    logits of the next ones, [batch, vocab_size].  On the GPU the step is captured in a CUDA graph at its first call and
    replayed after that; the logits are then a buffer that the next call overwrites."""

    def __init__(self, model, cache, use_graph: bool = True):
        self.model, self.cache = model, cache
        self.device = cache.lengths.device
        self.idx = torch.zeros(cache.batch, 1, dtype=torch.int64, device=self.device)
        self.use_graph = use_graph and self.idx.is_cuda
        self.graph = self.logits = None

    def _capture(self) -> None:
        # the steps before the capture append at the position that the first real one writes again
        cache = self.cache
        lengths, empty = cache.lengths.clone(), cache._empty
        # kernels are launched on the cache's device, whichever the current one is: the capture has to be there too
        with torch.cuda.device(self.device):
            side = torch.cuda.Stream(device=self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(side):
                self.model(self.idx, cache=cache)
                cache.lengths.copy_(lengths)
            torch.cuda.current_stream(self.device).wait_stream(side)
            torch.cuda.synchronize(self.device)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                self.logits = self.model(self.idx, cache=cache)
        self.graph = graph     # whole: a capture that failed is made again by the next call
        cache._empty = empty

    def __call__(self, tokens: torch.Tensor) -> torch.Tensor:
        if tokens.dim() == 0 or tokens.shape[0] != self.cache.batch or tokens.numel() != self.cache.batch:
            raise ValueError(f"DecodeStep: tokens of shape {tuple(tokens.shape)} for a cache of {self.cache.batch} sequences")
        if tokens.is_floating_point():
            raise ValueError(f"DecodeStep: tokens must be integers, got {tokens.dtype}")
        self.idx.copy_(tokens.reshape(-1, 1), non_blocking=True)
        if not self.use_graph:
            return self.model(self.idx, cache=self.cache)
        if self.graph is None:
            self._capture()
        with torch.cuda.device(self.device):
            self.graph.replay()
        self.cache._empty = False
        return self.logits


@torch.no_grad()
def generate(model, prompts: Sequence[Sequence[int]], max_new_tokens: int,
             sample: Optional[Callable[[torch.Tensor], torch.Tensor]] = None, page_size: int = 64,
             use_graph: bool = True) -> List[List[int]]:
    """``max_new_tokens`` tokens behind each of the prompts (lists of token ids, of any lengths from one on).  ``sample`` maps the
    logits [batch, vocab_size] to the next tokens, int64 [batch]; by default the most likely one.  Raises if a kernel has reported an
    error on the GPU (``parallel.health.check_device_status``)."""
    if not prompts or min(len(p) for p in prompts) < 1 or max_new_tokens < 0:
        raise ValueError("generate: every prompt needs a token, and max_new_tokens must not be negative")
    if max_new_tokens == 0:
        return [[] for _ in prompts]
    sample = sample or (lambda logits: logits.argmax(-1))
    device = model.lm_head.weight.device
    longest = max(len(p) for p in prompts)
    cache = model.new_cache(len(prompts), longest + max_new_tokens - 1, page_size)     # the last token is not fed back
    idx = torch.zeros(len(prompts), longest, dtype=torch.int64)
    for row, p in zip(idx, prompts):
        row[:len(p)] = torch.as_tensor(p, dtype=torch.int64)
    counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device)
    tokens = sample(model(idx.to(device), cache=cache, counts=counts))
    out = [tokens]
    step = DecodeStep(model, cache, use_graph)
    for _ in range(max_new_tokens - 1):
        tokens = sample(step(tokens))
        out.append(tokens)
    out = torch.stack(out, dim=1).tolist()
    if device.type == "cuda":
        with torch.cuda.device(device):
            check_device_status()
    return out
