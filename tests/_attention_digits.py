"""Bounds for masked attention whose product P V takes P rounded to the tensors' type and what that rounding left: the digits that a
bf16 output can have.

With u half a step of the type and e = 2^-24, as in _attention_bounds: the remainder is rounded itself, so of P's rounding u^2 is
left, and
  |dO| <= u |O| + (u^2 + E_i + n e) (P |V|)
Where P |V| is much larger than |O| the rounding of P alone, u (P |V|), is far outside.

norm_limit: the error's norm is that of rounding the exact values, moved by what is left of the other errors.  Those change which
way an element rounds, not how large a rounding is: over n elements the mean square of errors spread evenly over a step has a
deviation of 0.9 / sqrt(n) of itself, its root 0.45 / sqrt(n), and 3 % is 8 times that at 16384 elements.  P's rounding by itself
adds 7 % to the norm or more."""
import math

import torch

from _attention_bounds import E, half_step


def output64(q, k, v, mask, scale=None):
    """(value, bound) of the output, float64 on the device; arguments as of _attention_bounds.attention64."""
    u = half_step(q.dtype)
    q, k, v = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    G = q.shape[1] // k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    hidden, n, hd = ~mask.to(q.device), mask.sum(-1).max().item(), q.shape[-1]
    s = (q @ k.transpose(2, 3)) * scale
    p = s.masked_fill(hidden, -math.inf).softmax(-1)
    score_err = (hd * E * scale * (q.abs() @ k.abs().transpose(2, 3)) + 2 * E * s.abs()).masked_fill(hidden, 0)
    row = 2 * score_err.amax(-1, keepdim=True) + (n + 8) * E + 2.0 ** -20
    o = p @ v
    return o.transpose(1, 2), (u * o.abs() + (u * u + row + n * E) * (p @ v.abs())).transpose(1, 2)


def check_digits(name, got, value, bound):
    """Elementwise, and for 16384 elements or more the error's norm."""
    err = (got.double() - value).abs()
    worst = (err / bound.clamp_min(1e-300)).max().item()
    assert worst <= 1.0, f"{name}: off by {worst:.2f} times its bound"
    if got.numel() >= 16384:
        rounded = (value.to(got.dtype).double() - value).norm().item()
        assert err.norm().item() <= 1.03 * rounded, f"{name}: {err.norm().item() / rounded:.3f} times the error of its rounding"


def gradients64(q, k, v, do, mask, scale=None):
    """{name: (value, bound)} of dq, dk, dv where the output's error is that of output64 and what its own rounding left is kept
    (rounded itself, u^2).  The backward pass rounds P of dV and dS to the type, the choices that are left:
      |d dV| <= u |dV| + (u + E_i + n e) P^T |dO|
      |d dS| <= (u + E_i + 4 e) |dS| + scale P (hd e |dO||V|^T + |dO|.(|d O| - u |O| + u^2 |O|) + hd e |dO|.|O|)
      |d dQ| <= u |dQ| + (|d dS| + n e |dS|) |K|, and so for dK."""
    u = half_step(q.dtype)
    o, o_err = (t.transpose(1, 2) for t in output64(q, k, v, mask, scale))
    q, k, v, g = (t.detach().double().transpose(1, 2) for t in (q, k, v, do))
    B, Hq, T, hd = q.shape
    G = Hq // k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    kr, vr = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    hidden, n = ~mask.to(q.device), mask.sum(-1).max().item()
    s = (q @ kr.transpose(2, 3)) * scale
    p = s.masked_fill(hidden, -math.inf).softmax(-1)
    score_err = (hd * E * scale * (q.abs() @ kr.abs().transpose(2, 3)) + 2 * E * s.abs()).masked_fill(hidden, 0)
    row = 2 * score_err.amax(-1, keepdim=True) + (n + 8) * E + 2.0 ** -20
    share = lambda t: t.unflatten(1, (Hq // G, G)).sum(2)
    terms = n + G * T
    dv = share(p.transpose(2, 3) @ g)
    dv_err = u * dv.abs() + share(((u + row + terms * E) * p).transpose(2, 3) @ g.abs())
    ds = scale * p * (g @ vr.transpose(2, 3) - (g * o).sum(-1, keepdim=True))
    delta_err = (g.abs() * (o_err - u * o.abs() + u * u * o.abs())).sum(-1, keepdim=True)
    ds_err = (u + row + 4 * E) * ds.abs() + scale * p * (hd * E * (g.abs() @ vr.abs().transpose(2, 3)) + delta_err +
                                                         hd * E * (g.abs() * o.abs()).sum(-1, keepdim=True))
    ds_err = ds_err + terms * E * ds.abs()
    dq, dk = ds @ kr, share(ds.transpose(2, 3) @ q)
    back = lambda t: t.transpose(1, 2)
    return {"dq": (back(dq), back(u * dq.abs() + ds_err @ kr.abs())), "dv": (back(dv), back(dv_err)),
            "dk": (back(dk), back(u * dk.abs() + share(ds_err.transpose(2, 3) @ q.abs())))}
