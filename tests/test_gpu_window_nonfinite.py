"""Window attention on the GPU with NaN and infinities that rows see by right: every element is finite, +inf, -inf or NaN as the
definition says in 64 bits, and telling so does not crawl."""
import math

import pytest
import torch

from tinyinfinitrain_b200 import ops
from tinyinfinitrain_b200._lib import C

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _inputs(B, T, Hq, Hkv, hd, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda h: torch.randn(B, T, h, hd, device=DEV, generator=g).to(dtype)
    return r(Hq), r(Hkv), r(Hkv), r(Hq)


def _pairs64(q, k, v, do, window, sinks):
    """(value, sum of the terms' sizes) of o, dq, dk, dv from the definition: the terms of visible pairs alone are added."""
    B, T, Hq, hd = q.shape
    Hkv = k.shape[2]
    G, scale = Hq // Hkv, 1.0 / math.sqrt(hd)
    i = torch.arange(T, device=DEV)
    ahead = i[:, None] - i[None]
    see = (ahead >= 0) & ((ahead < (T if window is None else window)) | (i[None] < sinks))
    out = {n: [torch.zeros(B, T, h, hd, device=DEV, dtype=torch.float64) for _ in range(2)]
           for n, h in (("o", Hq), ("dq", Hq), ("dk", Hkv), ("dv", Hkv))}

    def add(name, b, h, weights, size, x):      # rows of `weights`: the rows of the result
        vis = see if name in ("o", "dq") else see.t()
        for c in range(0, hd, 16):
            terms = torch.where(vis[..., None], weights[..., None] * x[None, :, c:c + 16], 0.0)
            out[name][0][b, :, h, c:c + 16] += terms.sum(1)
            out[name][1][b, :, h, c:c + 16] += torch.where(vis[..., None], size[..., None] * x[None, :, c:c + 16].abs(), 0.0).sum(1)

    for b in range(B):
        for h in range(Hq):
            qb, kb, vb, gb = (t[b, :, n].double() for t, n in ((q, h), (k, h // G), (v, h // G), (do, h)))
            p = (qb @ kb.t() * scale).masked_fill(~see, -INF).softmax(-1)
            add("o", b, h, p, p, vb)
            o, o_size = out["o"][0][b, :, h], out["o"][1][b, :, h]
            ds = scale * p * (gb @ vb.t() - (gb * o).sum(-1, keepdim=True))
            size = scale * p * (gb.abs() @ vb.abs().t() + (gb.abs() * o_size).sum(-1, keepdim=True))
            add("dq", b, h, ds, size, kb)
            add("dk", b, h // G, ds.t(), size.t(), qb)
            add("dv", b, h // G, p.t(), p.t(), gb)
    return out


def _check(name, got, want):
    value, size = want
    assert torch.equal(torch.isnan(got), torch.isnan(value)), name
    for inf in (INF, -INF):
        assert torch.equal(got == inf, value == inf), (name, inf)
    # digits are held to account elsewhere: four roundings of a term at most (P or dS, o in delta, the sum), and the scores' own
    u = max(torch.finfo(got.dtype).eps / 2, 2.0 ** -16)
    ok = (got.double() - value).abs() <= 4 * u * size
    assert ok[torch.isfinite(value)].all(), name


def _spoil(case, q, k, v, do):
    T = q.shape[1]
    a, z = T // 5, T - T // 4
    if case == "one infinite value":
        v[:, a, 0, 3] = INF
    elif case == "both infinities in a column":
        v[:, a, 0, 3], v[:, a + 7, 0, 3], v[:, z, :, 5] = INF, -INF, -INF
    elif case == "an undefined value":
        v[:, a] = NAN
    elif case == "all values undefined":
        v.fill_(NAN)
    elif case == "all values infinite":
        v.fill_(INF)
    elif case == "one infinite gradient":
        do[:, z, 1, 2] = -INF
    elif case == "an undefined gradient":
        do[:, z, 0] = NAN
    elif case == "all gradients undefined":
        do.fill_(NAN)
    elif case == "a column of infinite gradients":
        do[..., 7] = INF
    elif case == "an infinite key":
        k[:, a, 0, 1] = INF
    elif case == "an undefined key":
        k[:, z, -1] = NAN
    elif case == "an infinite query":
        q[:, z, 0, 4] = INF
    elif case == "infinities that meet a weight of zero":
        # by sign of their query, rows see the second infinity of V, and keys that of dO, with a score of -inf
        v[:, a, 0, 3] = v[:, a + 9, 0, 3] = INF
        k[:, a + 9, 0, 1] = INF
        do[:, a + 20, :, 5] = do[:, a + 21, :, 5] = do[:, a + 22, :, 5] = -INF
    else:
        q[:, a, 0, 0], v[:, a + 3, -1, 1], do[:, z, :, 6], k[:, z + 5, 0, 2] = NAN, -INF, INF, INF


CASES = ["one infinite value", "both infinities in a column", "an undefined value", "all values undefined", "all values infinite",
         "one infinite gradient", "an undefined gradient", "all gradients undefined", "a column of infinite gradients",
         "an infinite key", "an undefined key", "an infinite query", "infinities that meet a weight of zero",
         "some of each"]


def _run(q, k, v, do, window, sinks):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = ops.window_attention(q, k, v, window, sinks)
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 0), (40, 3), (1, 0), (150, 130)])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64), (BF, 40), (F32, 120)])
def test_what_is_seen_shows_as_it_is(dtype, hd, window, sinks, case):
    q, k, v, do = _inputs(1, 277, 4, 2, hd, dtype, seed=hd)
    _spoil(case, q, k, v, do)
    want = _pairs64(q, k, v, do, window, sinks)
    for name, t in zip(("o", "dq", "dk", "dv"), _run(q, k, v, do, window, sinks)):
        _check(name, t, want[name])
    assert C.status_read(True) == 0


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_sinks_in_parts(dtype, hd, case):
    """A sequence whose sinks' gradients are sums of many parts."""
    q, k, v, do = _inputs(1, 1100, 2, 1, hd, dtype, seed=3)
    _spoil(case, q, k, v, do)
    want = _pairs64(q, k, v, do, 33, 2)
    for name, t in zip(("o", "dq", "dk", "dv"), _run(q, k, v, do, 33, 2)):
        _check(name, t, want[name])


def test_the_output_without_gradients_is_the_same():
    for case in CASES:
        for window in (None, 50):
            q, k, v, do = _inputs(1, 300, 2, 1, 64, BF, seed=5)
            _spoil(case, q, k, v, do)
            with torch.no_grad():
                plain = ops.window_attention(q, k, v, window)
            assert torch.equal(torch.nan_to_num(plain, 9.0, 8.0, 7.0), torch.nan_to_num(_run(q, k, v, do, window, 0)[0], 9.0, 8.0, 7.0))


def _ms(fn):
    for _ in range(2):
        fn()
    best = INF
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fn()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (256, 2)])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_a_pass_with_them_does_not_crawl(dtype, hd, window, sinks, case):
    """A pass over 1024 positions takes 0.13 ms when all is finite.  Warps that take rows again make it 1 to 5 ms; one thread a row made
    it 30 and more, growing with the square of what a row sees."""
    q, k, v, do = _inputs(1, 1024, 8, 2, hd, dtype, seed=1)
    fine = _ms(lambda: _run(q, k, v, do, window, sinks))
    _spoil(case, q, k, v, do)
    spoilt = _ms(lambda: _run(q, k, v, do, window, sinks))
    assert spoilt <= 100 * fine, (spoilt, fine)


@pytest.mark.parametrize("name,at", [("key", 100), ("value", 100), ("key", 127), ("value", 16)])
def test_beside_the_sinks(name, at):
    """A position that shares a tile with the sinks, which all later queries visit: those that do not see it are not taken again
    for it (that made a pass of 0.7 ms one of 59)."""
    T, window, sinks = 8192, 1024, 4
    q, k, v, do = _inputs(1, T, 32, 8, 128, BF, seed=2)
    fine = _ms(lambda: _run(q, k, v, do, window, sinks))
    whole = _run(q, k, v, do, window, sinks)
    (k if name == "key" else v)[:, at] = NAN
    spoilt = _ms(lambda: _run(q, k, v, do, window, sinks))
    o, dq, dk, dv = _run(q, k, v, do, window, sinks)
    first = (at + window + 127) // 128 * 128
    assert torch.equal(o[:, first:], whole[0][:, first:]) and torch.isfinite(dq[:, at + window:]).all()
    last = first + window       # keys that no spoilt query shares a tile with
    for got, want in ((dk, whole[2]), (dv, whole[3])):
        assert torch.equal(got[:, last:], want[:, last:])
    assert spoilt <= 30 * fine, (spoilt, fine)
