"""Attention over a bounded context and a paged key-value cache: what is timed, and the plain forms it is timed against.

Three operators:

* ``window`` -- causal attention in which a query sees the last ``window`` positions and the first ``sinks`` ones
  (``ops.window_attention``, ``ops.window_attention_qkv``): a training step (output and gradients) or a prompt (output).
* ``append`` -- rotary embedding of new queries and keys, the keys and values written into the pages of a cache
  (``ops.cache_append``).
* ``paged``  -- attention of one new token of each sequence over its pages (``ops.paged_attention``).

The head counts are those of the presets of ``models``: GPT-2 (12 heads of 64), GPT-2 XL (25 of 64), LLaMA-3 1B (32 and 8 of
64) and 8B (32 and 8 of 128).
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------- the cases
def _window(name, batch, seq, heads, kv_heads, head_dim, window, sinks, dtype="bf16", train=True, fused=True):
    case = {"do": "window", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "window": window, "sinks": sinks, "dtype": dtype, "train": train, "fused": fused}
    return {"name": name, **case} if name else case


def _append(name, batch, seq, heads, kv_heads, head_dim, before, page, dtype="bf16", theta=0.0, window=0, sinks=0):
    case = {"do": "append", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "before": before, "page": page, "dtype": dtype, "theta": theta, "window": window, "sinks": sinks}
    return {"name": name, **case} if name else case


def _paged(name, batch, longest, heads, kv_heads, head_dim, page, dtype="bf16", window=0, sinks=0, ragged=True):
    case = {"do": "paged", "batch": batch, "longest": longest, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype, "window": window, "sinks": sinks, "ragged": ragged}
    return {"name": name, **case} if name else case


def listed():
    return [
        # long-context training of the 8B shape: a window of an eighth of the sequence, read in place from the projection
        _window("window step 1x8192 llama3-8b", 1, 8192, 32, 8, 128, 1024, 4),
        # sequences of an odd length, odd head count, a window that is no multiple of a tile, tensors of their own
        _window("window step 3x777 gpt2-xl", 3, 777, 25, 25, 64, 100, 1, fused=False),
        # fp32 training, the precision of the end-to-end check
        _window("window fp32 step 2x512 gpt2", 2, 512, 12, 12, 64, 128, 2, dtype="fp32"),
        # a prompt of an odd length before generation starts
        _window("window prompt 1x1999 llama3-1b", 1, 1999, 32, 8, 64, 512, 4, train=False, fused=False),
        # the prompts of two conversations, the second shorter, into an empty cache
        _append("append prompt 2x1999 llama3-8b", 2, 1999, 32, 8, 128, 0, 64, theta=500000.0),
        # one new token each of a serving batch, at positions up to 131071
        _append("append token 64 llama3-8b", 64, 1, 32, 8, 128, 131000, 64, theta=500000.0),
        # one new token each at the command line's batch: no rotation, latency
        _append("append token 4 gpt2 fp32", 4, 1, 12, 12, 64, 60, 16, dtype="fp32"),
        # one step of sampling at the command line's default batch and length: latency
        _paged("paged 4x64 gpt2", 4, 64, 12, 12, 64, 16),
        # one conversation with a long cache: only a split over its length keeps the card busy
        _paged("paged 1x131071 llama3-8b", 1, 131071, 32, 8, 128, 64, ragged=False),
        # a serving batch of very different lengths, one slot of it idle
        _paged("paged 64x8192 llama3-8b", 64, 8192, 32, 8, 128, 64),
        # many conversations, each reading its window and its sinks only
        _paged("paged window 192x32768 llama3-1b", 192, 32768, 32, 8, 64, 32, window=1024, sinks=4),
        # the fp32 model's cache
        _paged("paged fp32 4x777 gpt2", 4, 777, 12, 12, 64, 16, dtype="fp32"),
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(12, 12, 64), (25, 25, 64), (32, 8, 64), (8, 2, 64), (32, 8, 128), (8, 1, 128), (4, 4, 128)]


def draw(rng):
    do = rng.choice(["window", "window", "append", "paged", "paged"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if do == "window":
        seq = _between(rng, 1, 512 if dtype == "fp32" else 8192)
        # tokens x heads x head size no more than the largest listed case has
        batch = rng.randint(1, max(1, min(8, (8192 * 32 * 128) // (seq * heads * head_dim))))
        if dtype == "fp32":
            batch = min(batch, 2)
        return _window(None, batch, seq, heads, kv_heads, head_dim, min(_between(rng, 1, 880), seq),
                       rng.choice([0, 1, 4, 16, 130]), dtype, rng.random() < 0.7, rng.random() < 0.5)
    page = rng.choice([16, 32, 64, 128])
    theta = rng.choice([0.0, 10000.0, 500000.0])
    window, sinks = (_between(rng, 16, 4096), rng.choice([0, 1, 4, 64])) if rng.random() < 0.4 else (0, 0)
    if do == "append":
        if rng.random() < 0.5:
            return _append(None, _between(rng, 1, 192), 1, heads, kv_heads, head_dim, _between(rng, 1, 131000), page, dtype,
                           theta)
        batch = rng.randint(1, 4)
        seq = _between(rng, 2, (1999 if dtype == "fp32" else 3998) // batch)
        return _append(None, batch, seq, heads, kv_heads, head_dim, rng.choice([0, 0, 17, 900]), page, dtype, theta, window,
                       sinks)
    # as many cached bytes as the largest listed cases read and hold, at most
    width = kv_heads * head_dim * (2 if dtype == "fp32" else 1)
    longest = _between(rng, 1, min(131071, 131071 * 8 * 128 // width))
    seen = min(longest, window + sinks) if window else longest
    most = min(131071 * 8 * 128 // (seen * width), 64 * 32768 * 8 * 64 // (longest * width))
    return _paged(None, _between(rng, 1, max(1, min(192, most))), longest, heads, kv_heads, head_dim, page, dtype, window, sinks,
                  rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------- what is in hand
def _lengths(case, seed):
    """Cached positions of each sequence, the new token's among them: spread over the logarithm, the longest among them, and in
    a large batch a slot that holds none."""
    rng = random.Random(seed * 7919 + 11)
    B, top = case["batch"], case["longest"]
    if not case["ragged"]:
        return [top] * B
    lengths = [_between(rng, max(1, top // 64), top) for _ in range(B)]
    lengths[rng.randrange(B)] = top
    if B >= 16:
        lengths[lengths.index(min(lengths))] = 0
    return lengths


def _pages(case, lengths, gen):
    """A page table over pages in random order, as an allocator leaves them after a while, and how many pages there are."""
    page = case["page"]
    need = [(n + page - 1) // page for n in lengths]
    width = max(max(need), 1)
    # pages of other conversations lie between them; entries behind a sequence's last page point at page 0, which is nobody's
    total = sum(need) + 1 + sum(need) // 8
    order = torch.randperm(total - 1, device=DEVICE, generator=gen).to(torch.int32) + 1
    table = torch.zeros(case["batch"], width, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    Hq, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen, dtype=dtype)

    if case["do"] == "window":
        B, T = case["batch"], case["seq"]
        # scores of a trained model spread over a few units, and its first tokens draw more attention than others
        q, k, v = normal(B, T, Hq, hd) * 2.0, normal(B, T, Hkv, hd), normal(B, T, Hkv, hd)
        k[:, :4] *= 1.5
        state = {"case": case, "do": normal(B, T, Hq, hd)}
        if case["fused"]:
            state["qkv"] = torch.cat([q, k, v], dim=2).flatten(2).requires_grad_(case["train"])
        else:
            state.update((name, t.requires_grad_(case["train"])) for name, t in (("q", q), ("k", k), ("v", v)))
        return state
    if case["do"] == "append":
        B, T = case["batch"], case["seq"]
        rng = random.Random(seed * 104729 + 5)
        before, counts = [], []
        for b in range(B):
            # prompts of a batch are padded behind to the longest one's length
            counts.append(T if b == 0 or T == 1 else rng.randint((T + 1) // 2, T))
            before.append(_between(rng, max(1, case["before"] // 2), case["before"]) if case["before"] else 0)
        table, total = _tail_pages(case, before, counts, gen)
        return {"case": case, "qkv": normal(B, T, (Hq + 2 * Hkv) * hd), "k_cache": normal(total, Hkv, case["page"], hd),
                "v_cache": normal(total, Hkv, case["page"], hd), "page_table": table,
                "starts": torch.tensor(before, dtype=torch.int32, device=DEVICE),
                "counts": torch.tensor(counts, dtype=torch.int32, device=DEVICE), "host": (before, counts)}
    lengths = _lengths(case, seed)
    table, total = _pages(case, lengths, gen)
    q = normal(case["batch"], Hq, hd) * 2.0
    return {"case": case, "q": q, "k_cache": normal(total, Hkv, case["page"], hd),
            "v_cache": normal(total, Hkv, case["page"], hd), "page_table": table,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE), "longest": max(lengths)}


def _tail_pages(case, before, counts, gen):
    """The pages that new tokens go to, in random order, and how many pages there are; the entries of the pages before them,
    which nothing here reads, point at page 0, which is nobody's."""
    page, B = case["page"], case["batch"]
    most = (case["seq"] + page - 1) // page + 1
    total = B * most + 1
    order = torch.randperm(total - 1, device=DEVICE, generator=gen).to(torch.int32) + 1
    table = torch.zeros(B, (case["before"] + case["seq"] + page - 1) // page, dtype=torch.int32, device=DEVICE)
    for b in range(B):
        first, last = before[b] // page, (before[b] + counts[b] + page - 1) // page
        table[b, first:last] = order[b * most:b * most + last - first]
    return table, total


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    do = state["case"]["do"]
    if own:
        return {"window": _own_window, "append": _own_append, "paged": _own_paged}[do](state)
    return {"window": _plain_window, "append": _plain_append, "paged": _plain_paged}[do](state)


def _own_window(state):
    from tinyinfinitrain_b200 import ops

    case = state["case"]
    leaves = [state["qkv"]] if case["fused"] else [state["q"], state["k"], state["v"]]

    def forward():
        if case["fused"]:
            return ops.window_attention_qkv(leaves[0], case["heads"], case["kv_heads"], case["window"], case["sinks"])
        return ops.window_attention(*leaves, case["window"], case["sinks"])

    if not case["train"]:
        with torch.no_grad():
            return forward()
    for t in leaves:
        t.grad = None
    out = forward()
    out.backward(state["do"])
    return (out.detach(), *(t.grad for t in leaves))


def _own_append(state):
    from tinyinfinitrain_b200 import ops

    case = state["case"]
    prompt = case["seq"] > 1
    with torch.no_grad():
        # a prompt's attention reads the rotated keys themselves, a single token's the cache
        out = ops.cache_append(state["qkv"], state["k_cache"], state["v_cache"], state["page_table"], state["starts"],
                               case["heads"], case["kv_heads"], theta=case["theta"] or None,
                               counts=state["counts"] if prompt else None, window=case["window"] or None,
                               sinks=case["sinks"], return_k=prompt)
    return (*(out if prompt else (out,)), state["k_cache"], state["v_cache"])


def _own_paged(state):
    from tinyinfinitrain_b200 import ops

    case = state["case"]
    with torch.no_grad():
        return ops.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"], state["lengths"],
                                   window=case["window"] or None, sinks=case["sinks"])


# ------------------------------------------------------------------------------------------------- plain forms
def _heads_of(state):
    """q, k, v of a window case as [B, T, H, hd] views."""
    case = state["case"]
    if not case["fused"]:
        return state["q"].detach(), state["k"].detach(), state["v"].detach()
    Hq, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    x = state["qkv"].detach().unflatten(-1, (Hq + 2 * Hkv, hd))
    return x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]


def _plain_window(state):
    """All scores of a sequence, masked; as many key heads and the query heads that share them at a time as about 1 GB holds."""
    case = state["case"]
    q, k, v = _heads_of(state)
    B, T, Hq, hd = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(hd)
    i = torch.arange(T, device=q.device)
    ahead = i[:, None] - i[None, :]
    hidden = ~((ahead >= 0) & ((ahead < case["window"]) | (i[None, :] < case["sinks"])))
    out = torch.empty(B, T, Hq, hd, device=q.device, dtype=q.dtype)
    train = case["train"]
    if train:
        dq, dk, dv = torch.empty_like(out), torch.empty_like(k, memory_format=torch.contiguous_format), \
            torch.empty_like(v, memory_format=torch.contiguous_format)
    some = max(1, min(Hkv, (1 << 30) // (4 * G * T * T)))
    for b in range(B):
        for h in range(0, Hkv, some):
            n = min(some, Hkv - h)
            mine = slice(h * G, (h + n) * G)
            qf = q[b, :, mine].float().view(T, n, G, hd).permute(1, 2, 0, 3)               # [n, G, T, hd]
            kf, vf = (t[b, :, h:h + n].float().transpose(0, 1)[:, None] for t in (k, v))   # [n, 1, T, hd]
            s = (qf @ kf.transpose(2, 3)).mul_(scale).masked_fill_(hidden, float("-inf"))
            s = s.sub_(s.amax(-1, keepdim=True)).exp_()
            p = s.div_(s.sum(-1, keepdim=True))
            o = p @ vf
            out[b, :, mine] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
            if train:
                g = state["do"][b, :, mine].float().view(T, n, G, hd).permute(1, 2, 0, 3)
                dv[b, :, h:h + n] = (p.transpose(2, 3) @ g).sum(1).transpose(0, 1).to(dv.dtype)
                ds = (g @ vf.transpose(2, 3)).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                dq[b, :, mine] = (ds @ kf).permute(2, 0, 1, 3).flatten(1, 2).to(dq.dtype)
                dk[b, :, h:h + n] = (ds.transpose(2, 3) @ qf).sum(1).transpose(0, 1).to(dk.dtype)
    if not train:
        return out
    if case["fused"]:
        return out, torch.cat([dq, dk, dv], dim=2).flatten(2)
    return out, dq, dk, dv


def _plain_append(state):
    case = state["case"]
    B, T, Hq, Hkv, hd = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    x = state["qkv"].unflatten(-1, (Hq + 2 * Hkv, hd))
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]
    if case["theta"]:
        half = hd // 2
        pos = state["starts"].double()[:, None] + torch.arange(T, device=DEVICE, dtype=torch.float64)
        angle = pos[..., None] * case["theta"] ** (torch.arange(half, device=DEVICE, dtype=torch.float64) * (-2.0 / hd))
        cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
        a, c = x[:, :, :Hq + Hkv, :half].float(), x[:, :, :Hq + Hkv, half:].float()
        turned = torch.cat([a * cos - c * sin, c * cos + a * sin], dim=-1).to(x.dtype)
        q, k = turned[:, :, :Hq], turned[:, :, Hq:]
    q, k = q.contiguous(), k.contiguous()
    page = case["page"]
    if T == 1:
        pos = state["starts"].long()
        pages = state["page_table"].gather(1, (pos // page)[:, None])[:, 0].long()
        state["k_cache"][pages, :, pos % page] = k[:, 0]
        state["v_cache"][pages, :, pos % page] = v[:, 0]
        return q, state["k_cache"], state["v_cache"]
    for b, (before, count) in enumerate(zip(*state["host"])):
        end = before + count
        # what the next token will not see is not kept
        spans = [(before, end)]
        if case["window"]:
            edge = max(before, end - case["window"])
            spans = [(before, min(end, case["sinks"], edge)), (edge, end)]
        for lo, hi in spans:
            if lo < hi:
                pos = torch.arange(lo, hi, device=DEVICE)
                pages = state["page_table"][b, pos // page].long()
                state["k_cache"][pages, :, pos % page] = k[b, lo - before:hi - before]
                state["v_cache"][pages, :, pos % page] = v[b, lo - before:hi - before]
    return q, k, state["k_cache"], state["v_cache"]


def _plain_paged(state):
    """All sequences at once, padded to the longest; positions that a sequence does not see are masked."""
    case = state["case"]
    q, table, lengths = state["q"], state["page_table"], state["lengths"].long()
    B, Hq, hd = q.shape
    Hkv, page = case["kv_heads"], case["page"]
    longest = state["longest"]
    pos = torch.arange(longest, device=q.device).expand(B, longest)
    seen = pos < lengths[:, None]
    if case["window"] and case["window"] + case["sinks"] < longest:
        window, sinks = case["window"], case["sinks"]
        first = torch.arange(sinks, device=q.device).expand(B, sinks)
        last = lengths[:, None] - window + torch.arange(window, device=q.device)
        pos = torch.cat([first, last], dim=1)
        # a sink that lies in the window counts once
        seen = torch.cat([(first < lengths[:, None]) & (first < lengths[:, None] - window), last >= 0], dim=1)
        pos = pos.clamp(min=0, max=longest - 1)
    elif case["window"]:
        seen = seen & ((pos >= lengths[:, None] - case["window"]) | (pos < case["sinks"]))
    pages = table.long().gather(1, pos // page)
    k = state["k_cache"][pages, :, pos % page].float()                   # [B, N, Hkv, hd]
    v = state["v_cache"][pages, :, pos % page].float()
    v = v.masked_fill_(~seen[:, :, None, None], 0.0)
    qf = q.float().view(B, Hkv, Hq // Hkv, hd)
    s = (qf @ k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(hd)).masked_fill_(~seen[:, None, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = s.sub_(top.masked_fill(top == float("-inf"), 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e @ v.permute(0, 2, 1, 3)) / total.masked_fill(total == 0, 1.0)
    return o.view(B, Hq, hd).to(q.dtype)


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"window": _exact_window, "append": _exact_append, "paged": _exact_paged}[case["do"]](case, state)


def _exact_window(case, state):
    """Per query head, from softmax(x)_j = e^(x_j - logsumexp(x)) and the chain rule."""
    q, k, v = (t.double() for t in _heads_of(state))
    do = state["do"].double()
    B, T, Hq, hd = q.shape
    G = Hq // k.shape[2]
    r, c = torch.meshgrid(torch.arange(T, device=q.device), torch.arange(T, device=q.device), indexing="ij")
    bias = torch.where((c > r) | ((r - c >= case["window"]) & (c >= case["sinks"])), -math.inf, 0.0).double()
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        for h in range(Hq):
            Q, K, V, D = q[b, :, h], k[b, :, h // G], v[b, :, h // G], do[b, :, h]
            logits = torch.addmm(bias, Q, K.t(), alpha=hd ** -0.5)
            prob = torch.exp(logits - torch.logsumexp(logits, dim=1, keepdim=True))
            del logits
            out[b, :, h] = prob @ V
            if case["train"]:
                dv[b, :, h // G] += prob.t() @ D
                dprob = D @ V.t()
                dlogit = prob * (dprob - (prob * dprob).sum(1, keepdim=True)) * hd ** -0.5
                dq[b, :, h] = dlogit @ K
                dk[b, :, h // G] += dlogit.t() @ Q
    if not case["train"]:
        return out
    if case["fused"]:
        return out, torch.cat([t.reshape(B, T, -1) for t in (dq, dk, dv)], dim=-1)
    return out, dq, dk, dv


def _exact_append(case, state):
    Hq, Hkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    B, T = case["batch"], case["seq"]
    qkv = state["qkv"].double().view(B, T, Hq + 2 * Hkv, hd)
    rotated = qkv[:, :, :Hq + Hkv].clone()
    starts, counts = state["host"]
    if case["theta"]:
        for i in range(hd // 2):
            turn = torch.tensor([[(s + t) * case["theta"] ** (-2.0 * i / hd) for t in range(T)] for s in starts],
                                dtype=torch.float64).to(DEVICE)
            z = torch.complex(qkv[:, :, :Hq + Hkv, i], qkv[:, :, :Hq + Hkv, i + hd // 2])
            z = z * torch.polar(torch.ones_like(turn), turn)[:, :, None]
            rotated[..., i], rotated[..., i + hd // 2] = z.real, z.imag
    q, k, v = rotated[:, :, :Hq], rotated[:, :, Hq:], qkv[:, :, Hq + Hkv:]
    k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
    table = state["page_table"].tolist()
    for b in range(B):
        end = starts[b] + counts[b]
        kept = [p for p in range(starts[b], end)
                if not case["window"] or p >= end - case["window"] or p < case["sinks"]]
        if kept:
            at = torch.tensor([table[b][p // page] for p in kept], device=DEVICE)
            row = torch.tensor([p % page for p in kept], device=DEVICE)
            src = torch.tensor([p - starts[b] for p in kept], device=DEVICE)
            k_cache[at, :, row] = k[b, src]
            v_cache[at, :, row] = v[b, src]
    return (q, k, k_cache, v_cache) if T > 1 else (q, k_cache, v_cache)


def _exact_paged(case, state):
    q = state["q"].double()
    B, Hq, hd = q.shape
    Hkv, page = case["kv_heads"], case["page"]
    out = torch.zeros_like(q)
    for b, n in enumerate(state["lengths"].tolist()):
        if n == 0:
            continue
        pages = state["page_table"][b, :(n + page - 1) // page].long()
        visible = torch.ones(n, dtype=torch.bool, device=q.device)
        if case["window"]:
            visible[case["sinks"]:max(case["sinks"], n - case["window"])] = False
        for h in range(Hkv):
            K = state["k_cache"][pages, h].reshape(-1, hd)[:n][visible].double()
            V = state["v_cache"][pages, h].reshape(-1, hd)[:n][visible].double()
            mine = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            logits = q[b, mine] @ K.t() * hd ** -0.5
            out[b, mine] = torch.softmax(logits, dim=1) @ V
    return out


# ------------------------------------------------------------------------------------------------- what it needs
def work(case):
    elem = 4 if case["dtype"] == "fp32" else 2
    Hq, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["do"] == "window":
        B, T = case["batch"], case["seq"]
        pairs = sum(min(i + 1, case["window"] + min(case["sinks"], max(0, i + 1 - case["window"]))) for i in range(T))
        # q k^T and p v; backward the scores again and four more products
        flops = (14.0 if case["train"] else 4.0) * hd * Hq * B * pairs
        # q, k, v in and o out; backward do in and three gradients out besides
        rows = (2 * Hq + 2 * Hkv) + (2 * Hq + 2 * Hkv if case["train"] else 0)
        return {"bytes": float(B * T * rows * hd * elem), "flops": flops}
    if case["do"] == "append":
        B, T = case["batch"], case["seq"]
        # the projection in; q (and for prompts k) out; keys and values into their pages
        rows = (Hq + 2 * Hkv) + Hq + (Hkv if T > 1 else 0) + 2 * Hkv
        return {"bytes": float(B * T * rows * hd * elem), "flops": 6.0 * B * T * (Hq + Hkv) * hd / 2 if case["theta"] else 0.0}
    lengths = _lengths(case, 0)
    seen = sum(min(n, case["window"] + min(case["sinks"], max(0, n - case["window"]))) if case["window"] else n
               for n in lengths)
    return {"bytes": float(2 * seen * Hkv * hd * elem + 2 * case["batch"] * Hq * hd * elem), "flops": 4.0 * seen * Hq * hd}
