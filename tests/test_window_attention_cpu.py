"""Window attention with sinks on the CPU: the plain path against 64-bit arithmetic, its gradients, and what is refused."""
import pytest
import torch

from tinyinfinitrain_b200 import ops

from _attention_bounds import attention64, check, visible

F32 = torch.float32


def _inputs(B, T, Hq, Hkv, hd, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda h: torch.randn(B, T, h, hd, generator=g).to(dtype)
    return r(Hq), r(Hkv), r(Hkv), r(Hq)


@pytest.mark.parametrize("T,window,sinks", [(1, 1, 0), (9, 1, 2), (40, 7, 0), (40, 7, 3), (40, 100, 1), (65, 16, 30)])
@pytest.mark.parametrize("fused", [False, True])
def test_against_64_bits(T, window, sinks, fused):
    q, k, v, do = _inputs(2, T, 4, 2, 16)
    want = attention64(q, k, v, do, visible(T, window, sinks))
    if fused:
        leaf = torch.cat([q, k, v], 2).flatten(2).requires_grad_()
        o = ops.window_attention_qkv(leaf, 4, 2, window, sinks)
        o.backward(do)
        got = (o, *leaf.grad.unflatten(-1, (8, 16)).split((4, 2, 2), 2))
    else:
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = ops.window_attention(*leaves, window, sinks)
        got = (o, *torch.autograd.grad(o, leaves, do))
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        check(name, t, want[name])


def test_the_bounds_follow_the_formula():
    """The 64-bit values themselves against autograd in 64 bits, to 1e-12: a mistake in them would move every bound."""
    q, k, v, do = (t.double() for t in _inputs(1, 30, 4, 2, 8))
    want = attention64(q, k, v, do, visible(30, 9, 2))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    s = torch.einsum("bihd,bjhd->bhij", leaves[0], leaves[1].repeat_interleave(2, 2)) / 8 ** 0.5
    p = s.masked_fill(~visible(30, 9, 2), float("-inf")).softmax(-1)
    o = torch.einsum("bhij,bjhd->bihd", p, leaves[2].repeat_interleave(2, 2))
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do))):
        assert (t - want[name][0]).abs().max() < 1e-12, name


def test_a_planted_mistake_is_seen():
    """One key too many in the oracle's mask fails the comparison."""
    q, k, v, do = _inputs(1, 30, 2, 2, 16)
    o = ops.window_attention(q, k, v, 9, 2)
    check("o", o, attention64(q, k, v, None, visible(30, 9, 2))["o"])
    with pytest.raises(AssertionError):
        check("o", o, attention64(q, k, v, None, visible(30, 10, 2))["o"])
    with pytest.raises(AssertionError):
        check("o", o, attention64(q, k, v, None, visible(30, 9, 3))["o"])


def test_no_bound_is_causal_attention():
    q, k, v, _ = _inputs(1, 12, 4, 2, 8)
    for window in (None, 12, 2 ** 40):
        assert torch.equal(ops.window_attention(q, k, v, window), ops.attention_ref(q, k, v))


def test_refusals():
    q, k, v, _ = _inputs(1, 8, 4, 2, 16)
    for args in ((q, k.double(), v, 4, 0), (q, k, v, 0, 0), (q, k, v, -1, 0), (q, k, v, 4, -1), (q[:, :4], k, v, 4, 0),
                 (q, k[:, :, :1], v, 4, 0), (q[:, :, :3], k, v, 4, 0), (q[0], k[0], v[0], 4, 0)):
        with pytest.raises(RuntimeError, match="titb200 window_attention"):
            ops.window_attention(*args)
    for scale in (0.0, -1.0, float("inf"), float("nan"), 1e-60, 1e60):
        with pytest.raises(RuntimeError, match="scale"):
            ops.window_attention(q, k, v, 4, scale=scale)
    with pytest.raises(RuntimeError, match="does not hold"):
        ops.window_attention_qkv(torch.zeros(1, 4, 101), 2, 1, 4)
