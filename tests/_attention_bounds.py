"""Masked attention and its gradients in 64 bits, with elementwise bounds on what the kernels' arithmetic may add.

u is half a step of the tensors' type (bf16 2^-8, fp32 2^-24) and e = 2^-24.  A sum of n fp32 terms is off by at most
n e times the sum of their absolute values.

* scores: d_ij = hd e scale sum|q k| + 2 e |s|; the exponential, its argument and the row sum add 2^-20 + n e, and the row's
  maximum or log-sum-exp takes part with the error of its own scores: E_i = 2 max_j d_ij + (n + 8) e + 2^-20 relative to P_ij.
* O = P V, P rounded to the tensors' type before the product, O rounded:
  |dO| <= u |O| + (u + E_i + n e) (P |V|)
* dV = P^T dO, the same: u |dV| + P'^T |dO| with P' = (u + E_i + n e) P
* dS = scale P (dP - D), rounded; dP = dO V^T is off by hd e (|dO| |V|^T), D = rowsum(dO O) by hd e rowsum|dO O| and O's own error,
  of which the rounding counts with u^2: what it leaves is kept, rounded itself:
  |d dS| <= (u + E_i + 4 e) |dS| + scale P (hd e |dO||V|^T + |dO|.(|d O| - u |O| + u^2 |O|) + hd e |dO|.|O|)
* dQ = dS K and dK = dS^T Q: u |dQ| + (|d dS| + n e |dS|) |K|, and so for dK.
"""
import math

import torch

E = 2.0 ** -24


def visible(T, window, sinks):
    i = torch.arange(T)
    ahead = i[:, None] - i[None, :]
    return (ahead >= 0) & ((ahead < window) | (i[None, :] < sinks))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention64(q, k, v, do, mask, scale=None):
    """q [B,T,Hq,hd], k, v [B,S,Hkv,hd], do like q (or None), mask [T, S].  Returns {name: (value, bound)} in float64 on the CPU
    for o, dq, dk, dv (o alone without do)."""
    u = half_step(q.dtype)
    q, k, v = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v))
    B, Hq, T, hd = q.shape
    G = Hq // k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    kr, vr = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    hidden = ~mask.cpu()
    s = (q @ kr.transpose(2, 3)) * scale
    p = s.masked_fill(hidden, -math.inf).softmax(-1)
    p = torch.where(hidden, torch.zeros_like(p), p)        # a row that sees nothing
    n = mask.sum(-1).max().item()
    ds_abs = hd * E * scale * (q.abs() @ kr.abs().transpose(2, 3)) + 2 * E * s.abs()
    row = 2 * ds_abs.masked_fill(hidden, 0).amax(-1, keepdim=True) + (n + 8) * E + 2.0 ** -20
    o = p @ vr
    o_err = u * o.abs() + (u + row + n * E) * (p @ vr.abs())
    back = lambda t: t.transpose(1, 2)
    out = {"o": (back(o), back(o_err))}
    if do is None:
        return out
    g = do.detach().cpu().double().transpose(1, 2)
    share = lambda t: back(t.unflatten(1, (Hq // G, G)).sum(2))
    dv = share(p.transpose(2, 3) @ g)
    pe = (u + row + (G * n + T) * E) * p
    dv_err = u * dv.abs() + share(pe.transpose(2, 3) @ g.abs())
    dp = g @ vr.transpose(2, 3)
    delta = (g * o).sum(-1, keepdim=True)
    ds = scale * p * (dp - delta)
    ds_err = (u + row + 4 * E) * ds.abs() + scale * p * (
        hd * E * (g.abs() @ vr.abs().transpose(2, 3)) + (g.abs() * (o_err - (u - u * u) * o.abs())).sum(-1, keepdim=True)
        + hd * E * (g.abs() * o.abs()).sum(-1, keepdim=True))
    ds_all = ds_err + (n + G * T) * E * ds.abs()
    dq, dk = ds @ kr, share(ds.transpose(2, 3) @ q)
    out["dq"] = (back(dq), u * back(dq).abs() + back(ds_all @ kr.abs()))
    out["dk"] = (dk, u * dk.abs() + share(ds_all.transpose(2, 3) @ q.abs()))
    out["dv"] = (dv, dv_err)
    return out


def check(name, got, want):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    err = (got.detach().cpu().double() - value).abs()
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert (err <= bound).all(), f"{name}: off by {worst:.2f} times its bound"
    return worst
