"""Window attention with sinks on the GPU against 64-bit arithmetic, with the bounds of _attention_bounds."""
import pytest
import torch

from tinyinfinitrain_b200 import ops
from tinyinfinitrain_b200._lib import C

from _attention_bounds import attention64, check, visible

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _inputs(B, T, Hq, Hkv, hd, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda h: torch.randn(B, T, h, hd, device=DEV, generator=g)
    return (2 * r(Hq)).to(dtype), r(Hkv).to(dtype), r(Hkv).to(dtype), r(Hq).to(dtype)


def _fused(q, k, v):
    return torch.cat([q, k, v], dim=2).flatten(2)


def _run(q, k, v, do, window, sinks, fused, scale=None):
    Hq, Hkv = q.shape[2], k.shape[2]
    if fused:
        leaf = _fused(q, k, v).requires_grad_()
        o = ops.window_attention_qkv(leaf, Hq, Hkv, window, sinks, scale)
        o.backward(do)
        return (o, *leaf.grad.unflatten(-1, (Hq + 2 * Hkv, q.shape[3])).split((Hq, Hkv, Hkv), dim=2))
    q, k, v = (t.clone().requires_grad_() for t in (q, k, v))
    o = ops.window_attention(q, k, v, window, sinks, scale)
    o.backward(do)
    return o, q.grad, k.grad, v.grad


def _compare(q, k, v, do, window, sinks, got, scale=None):
    T = q.shape[1]
    want = attention64(q, k, v, do, visible(T, T if window is None else window, sinks), scale)
    for name, t in zip(("o", "dq", "dk", "dv"), got):
        check(name, t, want[name])
    torch.cuda.synchronize()
    assert C.status_read(True) == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (2, 0), (64, 1), (100, 0), (128, 4), (129, 130), (300, 0), (1000, 5)])
@pytest.mark.parametrize("T", [1, 2, 63, 129, 300, 517])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_lengths_windows_and_sinks(T, window, sinks, dtype, hd):
    q, k, v, do = _inputs(2, T, 4, 2, hd, dtype, seed=T * 7 + window)
    _compare(q, k, v, do, window, sinks, _run(q, k, v, do, window, sinks, fused=True))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 5), (8, 1), (6, 3), (32, 8)])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 128)])
def test_head_layouts(Hq, Hkv, dtype, hd):
    q, k, v, do = _inputs(1, 260, Hq, Hkv, hd, dtype, seed=Hq)
    _compare(q, k, v, do, 90, 2, _run(q, k, v, do, 90, 2, fused=False))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd", [8, 16, 40, 72, 96, 120])
def test_other_head_sizes(hd, dtype):
    q, k, v, do = _inputs(2, 150, 4, 2, hd, dtype, seed=hd)
    _compare(q, k, v, do, 70, 3, _run(q, k, v, do, 70, 3, fused=hd % 16 == 0))


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64), (BF, 32)])
def test_sinks_far_behind_the_window(dtype, hd):
    """Many tiles between the sinks and the window, in several sink tiles, with shared heads."""
    for T, window, sinks in ((1500, 33, 1), (1300, 130, 300), (1111, 1, 128), (2049, 64, 4)):
        q, k, v, do = _inputs(1, T, 2, 1, hd, dtype, seed=T)
        _compare(q, k, v, do, window, sinks, _run(q, k, v, do, window, sinks, fused=True))


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (F32, 64)])
def test_no_bound_is_causal_attention(dtype, hd):
    q, k, v, do = _inputs(2, 333, 4, 2, hd, dtype)
    for window in (None, 333, 2 ** 40):
        _compare(q, k, v, do, None, 0, _run(q, k, v, do, window, 0, fused=True))


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_strides_orders_and_scale(dtype, hd):
    """Views of a wider buffer, transposed storage, an unaligned view, a broadcast gradient, a scale of one's own."""
    B, T, Hq, Hkv = 2, 140, 4, 2
    q, k, v, do = _inputs(B, T, Hq, Hkv, hd, dtype, seed=3)
    want = _run(q, k, v, do, 50, 2, fused=False, scale=0.3)
    _compare(q, k, v, do, 50, 2, want, scale=0.3)
    wide = torch.randn(B, T, 3 * hd * (Hq + 2 * Hkv), device=DEV).to(dtype)
    wide[..., hd:hd + Hq * hd] = q.flatten(2)
    layouts = [
        (wide[..., hd:hd + Hq * hd].unflatten(-1, (Hq, hd)), k.transpose(1, 2).contiguous().transpose(1, 2),
         torch.stack([v, v], dim=-1)[..., 0]),
        (torch.cat([q.flatten().new_zeros(1), q.flatten()])[1:].view_as(q), k.flip(0).flip(0), v),
    ]
    for ql, kl, vl in layouts:
        ql, kl, vl = (t.detach().requires_grad_() for t in (ql, kl, vl))
        o = ops.window_attention(ql, kl, vl, 50, 2, 0.3)
        got = torch.autograd.grad(o, (ql, kl, vl), do)
        for name, a, b in zip(("o", "dq", "dk", "dv"), (o, *got), want):
            if name == "dq" and dtype == BF:
                continue        # summed with atomics: the order differs from run to run
            assert torch.equal(a, b), name
    ones = torch.ones((), device=DEV, dtype=dtype).expand_as(q)
    ql, kl, vl = (t.clone().requires_grad_() for t in (q, k, v))
    o = ops.window_attention(ql, kl, vl, 50, 2)
    _compare(q, k, v, ones, 50, 2, (o, *torch.autograd.grad(o, (ql, kl, vl), ones)))


def test_gradients_against_differences():
    """fp32: the directional derivative along random directions.  A central difference of step h in fp32 is off by about
    h^2 / 6 times the third derivative plus 2^-24 |f| / h: with f of order 100 and h = 1e-2, a few 1e-3 of the derivative."""
    q, k, v, do = _inputs(1, 70, 2, 1, 16, F32, seed=9)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    f = lambda *x: (ops.window_attention(*x, 20, 2).double() * do.double()).sum()
    grads = torch.autograd.grad(ops.window_attention(q, k, v, 20, 2), (q, k, v), do)
    g = torch.Generator(device=DEV).manual_seed(1)
    for n, grad in enumerate(grads):
        x = [q.detach(), k.detach(), v.detach()]
        d = torch.randn(x[n].shape, device=DEV, generator=g)
        h = 1e-2
        plus, minus = list(x), list(x)
        plus[n], minus[n] = x[n] + h * d, x[n] - h * d
        slope = ((f(*plus) - f(*minus)) / (2 * h)).item()
        exact = (grad.double() * d.double()).sum().item()
        assert abs(slope - exact) <= 1e-2 * max(1.0, grad.double().norm().item())


def test_extreme_scores():
    """Scores of thousands, of both signs, and rows whose scores are all equal."""
    q, k, v, do = _inputs(1, 200, 2, 2, 64, BF, seed=4)
    q[:, 50:100] *= 300
    k[:, 20:60] *= 30
    q[:, 150:] = 0
    o = ops.window_attention(q, k, v, 64, 4)
    want = attention64(q, k, v, None, visible(200, 64, 4))
    check("o", o, want["o"])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_empty(dtype):
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        q = torch.zeros(shape, device=DEV, dtype=dtype, requires_grad=True)
        o = ops.window_attention(q, q, q, 3)
        o.sum().backward()
        assert o.shape == shape and q.grad.shape == shape


def test_refusals():
    q, k, v, _ = _inputs(1, 8, 4, 2, 64, BF)
    bad = [
        (q.half(), k.half(), v.half(), 4, 0), (q, k.float(), v, 4, 0), (q, k, v, 0, 0), (q, k, v, -1, 0), (q, k, v, 4, -1),
        (q[:, :4], k, v, 4, 0), (q, k[:, :, :1], v, 4, 0), (q[:, :, :3], k, v, 4, 0), (q[0], k[0], v[0], 4, 0),
        (q[..., :4], k[..., :4], v[..., :4], 4, 0), (q, k.cpu(), v, 4, 0),
    ]
    for args in bad:
        with pytest.raises(RuntimeError, match="titb200 window_attention"):
            ops.window_attention(*args)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="scale"):
            ops.window_attention(q, k, v, 4, scale=scale)
        with pytest.raises(RuntimeError, match="scale"):
            ops.window_attention_qkv(_fused(q, k, v), 4, 2, 4, scale=scale)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.window_attention(*(torch.zeros(1, 4, 2, 136, device=DEV, dtype=BF),) * 3, 4)
    with pytest.raises(RuntimeError, match="does not hold"):
        ops.window_attention_qkv(torch.zeros(1, 4, 101, device=DEV, dtype=BF), 2, 1, 4)


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_captured_step_beside_an_eager_one(dtype, hd):
    """Forward and backward in a CUDA graph, replayed with new inputs, and on another stream."""
    q, k, v, do = _inputs(1, 400, 4, 2, hd, dtype, seed=1)
    static = [t.clone() for t in (q, k, v)]
    sdo = do.clone()

    def step():
        leaves = [t.detach().requires_grad_() for t in static]
        o = ops.window_attention(*leaves, 100, 4)
        return (o.detach(), *torch.autograd.grad(o, leaves, sdo))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (5, 6):
        new = _inputs(1, 400, 4, 2, hd, dtype, seed=seed)
        for s, t in zip((*static, sdo), new):
            s.copy_(t)
        graph.replay()
        _compare(*new, 100, 4, captured)


@pytest.mark.parametrize("fused", [False, True])
def test_a_second_derivative_is_refused(fused):
    """The gradients of a recorded backward pass are values like any; differentiating them is an error."""
    q, k, v, do = _inputs(1, 20, 2, 1, 64, F32)
    leaves = [_fused(q, k, v).requires_grad_()] if fused else [t.requires_grad_() for t in (q, k, v)]
    o = ops.window_attention_qkv(leaves[0], 2, 1, 5) if fused else ops.window_attention(*leaves, 5)
    first = torch.autograd.grad(o, leaves, do, create_graph=True)
    again = torch.autograd.grad(ops.window_attention_qkv(leaves[0], 2, 1, 5) if fused else ops.window_attention(*leaves, 5), leaves, do)
    assert all(torch.equal(a.detach(), b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second derivative"):
        first[0].sum().backward()


def test_without_gradients_and_for_some_inputs_only():
    q, k, v, do = _inputs(1, 150, 4, 2, 64, BF)
    with torch.no_grad():
        plain = ops.window_attention(q, k, v, 30, 2)
    assert not plain.requires_grad
    v.requires_grad_()
    o = ops.window_attention(q, k, v, 30, 2)
    assert torch.equal(o.detach(), plain)
    o.backward(do)
    check("dv", v.grad, attention64(q, k, v, do, visible(150, 30, 2))["dv"])
    assert q.grad is None
    with torch.inference_mode():
        assert torch.equal(ops.window_attention(q, k, v, 30, 2), plain)
    # two backward passes of one forward, and an output changed in place by the caller
    o = ops.window_attention(q, k, v, 30, 2)
    a = torch.autograd.grad(o, v, do, retain_graph=True)[0]
    b = torch.autograd.grad(o, v, do)[0]
    assert torch.equal(a, b)
    o = ops.window_attention(q, k, v, 30, 2)
    o.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), 3e38])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64), (F32, 128), (BF, 40)])
@pytest.mark.parametrize("T,window,first,last", [(300, 40, 50, 250), (1100, 130, 300, 900)])
def test_what_a_row_does_not_see_may_be_anything(T, window, first, last, dtype, hd, fill):
    """Positions before `first` and from `last` on hold NaN, infinities or numbers whose products overflow, in q, k, v and the
    gradient.  Rows of o and dQ whose window holds none of them, and rows of dK and dV that no such query sees, are what the
    positions between them give by themselves."""
    q, k, v, do = _inputs(2, T, 4, 2, hd, dtype, seed=T)
    for t in (q, k, v, do):
        t[:, :first] = fill
        t[:, last:] = fill
    got = _run(q, k, v, do, window, 0, fused=False)
    lo, hi = first + window, last - window
    inner = [t[:, first:last] for t in (q, k, v, do)]
    want = attention64(*inner, visible(last - first, window, 0))
    for name, t, rows in zip(("o", "dq", "dk", "dv"), got, (slice(lo, last), slice(lo, last), slice(lo, hi), slice(lo, hi))):
        value, bound = (x[:, rows.start - first:rows.stop - first] for x in want[name])
        check(name, t[:, rows], (value, bound))


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_garbage_between_sinks_and_window(dtype, hd):
    """Garbage in the middle of a sequence: later rows see the sinks before it and the window behind it, and the sinks' gradients
    come from them alone where the queries beside the garbage have no gradient."""
    T, window, sinks = 900, 70, 3
    q, k, v, do = _inputs(1, T, 2, 1, hd, dtype, seed=2)
    k[:, 200:400], v[:, 200:400] = float("nan"), float("inf")
    got = _run(q, k, v, do, window, sinks, fused=True)
    keep = list(range(sinks)) + list(range(400, T))
    mask = visible(T, window, sinks)[470:][:, keep]
    n = T - 470
    want = attention64(q[:, 470:], k[:, keep], v[:, keep], do[:, 470:], mask)
    check("o", got[0][:, 470:], want["o"])
    check("dq", got[1][:, 470:], want["dq"])
    # keys from 470 on are seen by rows from 470 on only
    check("dk", got[2][:, 470:], tuple(x[:, -n:] for x in want["dk"]))
    check("dv", got[3][:, 470:], tuple(x[:, -n:] for x in want["dv"]))
    assert torch.isnan(got[0][:, 250]).all() and torch.isfinite(got[0][:, :200]).all()


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_a_visible_nan_shows(dtype, hd):
    q, k, v, do = _inputs(1, 300, 2, 1, hd, dtype, seed=2)
    k[:, 100] = float("nan")
    o, dq, dk, dv = _run(q, k, v, do, 40, 0, fused=True)
    assert torch.isnan(o[:, 100:140]).all() and torch.isfinite(o[:, :100]).all() and torch.isfinite(o[:, 140:]).all()
    assert torch.isnan(dq[:, 100:140]).all() and torch.isfinite(dq[:, :100]).all() and torch.isfinite(dq[:, 140:]).all()
    assert torch.isnan(dv[:, 61:140]).all() and torch.isfinite(dv[:, :61]).all() and torch.isfinite(dv[:, 140:]).all()
    v[:, 100] = float("inf")
    k[:, 100] = 0
    o = ops.window_attention(q, k, v, 40)
    assert torch.isinf(o[:, 100:140]).all() and torch.isfinite(o[:, :100]).all() and torch.isfinite(o[:, 140:]).all()
