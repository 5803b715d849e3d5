"""The paged cache's operators on the GPU against 64-bit arithmetic."""
import math

import pytest
import torch

from tinyinfinitrain_b200 import ops
from tinyinfinitrain_b200._lib import C
from tinyinfinitrain_b200.parallel.health import check_device_status

from _attention_bounds import attention64, check, half_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _cache(lengths, Hkv, hd, page, dtype, seed=0, fill=float("nan"), slack=3):
    """Caches whose rows all hold `fill` but for the given positions, a page table in random order and the rows themselves."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lengths]
    total = sum(need) + slack
    order = torch.randperm(total, generator=g).to(torch.int32)
    width = max(max(need), 1)
    table = torch.full((len(lengths), width), -7, dtype=torch.int32)     # entries behind the last page are not followed
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    kc, vc = (torch.full((total, Hkv, page, hd), fill, dtype=dtype) for _ in range(2))
    rows = []
    for b, n in enumerate(lengths):
        k, v = (torch.randn(n, Hkv, hd, generator=g).to(dtype) for _ in range(2))
        pos = torch.arange(n)
        pages = table[b, pos // page].long()
        kc[pages, :, pos % page] = k
        vc[pages, :, pos % page] = v
        rows.append((k, v))
    return kc.to(DEV), vc.to(DEV), table.to(DEV), rows


def _expect(q, rows, lengths, window, sinks, scale=None):
    outs, bounds = [], []
    for b, n in enumerate(lengths):
        if n == 0:
            outs.append(torch.zeros(q.shape[1:], dtype=torch.float64))
            bounds.append(torch.zeros(q.shape[1:], dtype=torch.float64))
            continue
        p = torch.arange(n)
        seen = p < n if window is None else (p >= n - window) | (p < sinks)
        k, v = (t[seen][None] for t in rows[b])
        o, e = attention64(q[b][None, None], k, v, None, torch.ones(1, int(seen.sum()), dtype=torch.bool), scale)["o"]
        outs.append(o[0, 0])
        bounds.append(e[0, 0])
    return torch.stack(outs), torch.stack(bounds)


def _paged(lengths, Hq, Hkv, hd, page, dtype, window=None, sinks=0, seed=0, scale=None):
    kc, vc, table, rows = _cache(lengths, Hkv, hd, page, dtype, seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (2 * torch.randn(len(lengths), Hq, hd, device=DEV, generator=g)).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, kc, vc, table, n, window, sinks, scale)
    check("o", o, _expect(q, rows, lengths, window, sinks, scale))
    torch.cuda.synchronize()
    assert C.status_read(True) == 0
    return o


TYPES = [(BF, 64), (BF, 128), (F32, 64), (F32, 128)]


@pytest.mark.parametrize("dtype,hd", TYPES)
@pytest.mark.parametrize("lengths", [[1], [0], [2, 0, 1], [15, 16, 17, 63, 64, 65], [300, 1, 127, 128, 129, 0, 500], [4097, 3]])
def test_lengths(lengths, dtype, hd):
    _paged(lengths, 8, 2, hd, 16, dtype, seed=sum(lengths))


@pytest.mark.parametrize("dtype,hd", TYPES)
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (12, 12), (25, 25), (8, 1), (32, 8), (17, 1), (40, 1), (6, 2)])
def test_head_layouts(Hq, Hkv, dtype, hd):
    _paged([70, 333], Hq, Hkv, hd, 16, dtype, seed=Hq)


@pytest.mark.parametrize("dtype,hd", TYPES)
@pytest.mark.parametrize("page", [1, 3, 16, 48, 64, 100, 128, 1024])
def test_pages_that_end_inside_a_tile(page, dtype, hd):
    _paged([1, 99, 260, 1025], 4, 2, hd, page, dtype, seed=page)


@pytest.mark.parametrize("dtype,hd", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 0), (64, 4), (100, 70), (1000, 0), (333, 2), (2000, 3), (2 ** 40, 0)])
def test_window_and_sinks(window, sinks, dtype, hd):
    _paged([1, 64, 333, 1500, 0, 70], 8, 2, hd, 32, dtype, window, sinks, seed=window % 1000)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd", [8, 16, 24, 32, 40, 72, 80, 96, 112, 120])
def test_other_head_sizes(hd, dtype):
    _paged([50, 300], 6, 2, hd, 16, dtype, seed=hd)


@pytest.mark.parametrize("dtype,hd", TYPES)
def test_many_sequences(dtype, hd):
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 400, (700,), generator=g).tolist()
    _paged(lengths, 4, 1, hd, 16, dtype, seed=5)


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_a_long_cache(dtype, hd):
    _paged([20000, 1], 4, 1, hd, 64, dtype, seed=8)
    _paged([33000], 8, 2, hd, 64, dtype, seed=9, scale=0.5)


def test_rows_behind_2_31_elements():
    """A cache of more than 2^31 elements: the pages in use are its last ones."""
    Hkv, hd, page = 8, 128, 64
    n_pages = (1 << 31) // (Hkv * hd * page) + 300
    kc = torch.zeros(n_pages, Hkv, page, hd, device=DEV, dtype=BF)
    vc = torch.zeros_like(kc)
    lengths = [1500, 900]
    table = torch.stack([torch.arange(n_pages - 1, n_pages - 25, -1), torch.arange(n_pages - 101, n_pages - 125, -1)]).int().to(DEV)
    qkv = torch.randn(2, 1500, (32 + 16) * hd, device=DEV).to(BF)
    counts = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    starts = torch.zeros(2, dtype=torch.int32, device=DEV)
    q, k = ops.cache_append(qkv, kc, vc, table, starts, 32, 8, theta=500000.0, counts=counts, return_k=True)
    v = qkv.unflatten(-1, (48, hd))[:, :, 40:]
    last = torch.stack([q[b, n - 1] for b, n in enumerate(lengths)])
    o = ops.paged_attention(last, kc, vc, table, counts)
    check("o", o, _expect(last, [(k[b, :n].cpu(), v[b, :n].cpu()) for b, n in enumerate(lengths)], lengths, None, 0))
    check_device_status()


# --------------------------------------------------------------------------------------------------- append
def _append64(x, starts, Hq, Hkv, hd, theta):
    """Rotated q and k in 64 bits and the bound of their error: the fp32 sine and cosine are off by at most 2^-22, the two
    products and their sum by 2 * 2^-24 of their size.  The angle: here the exponent's rounding is multiplied by the
    logarithm of theta (13.2 at most) in the power, which is rounded, and so is its product with the position, 15.2 * 2^-53 in
    all; in the kernel the power and the product are rounded, 2 * 2^-53.  Together less than 2^-48 of the angle."""
    x = x.cpu().double().unflatten(-1, (Hq + 2 * Hkv, hd))[:, :, :Hq + Hkv]
    if not theta:
        return x, torch.zeros_like(x)
    pos = starts.cpu().double()[:, None] + torch.arange(x.shape[1]).double()
    ang = pos[..., None] * theta ** (torch.arange(hd // 2).double() * (-2.0 / hd))
    cos, sin = ang.cos()[:, :, None], ang.sin()[:, :, None]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    size = (a.abs() + b.abs()) * (2.0 ** -22 + 2.0 ** -23 + 2.0 ** -48 * ang[:, :, None])
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1), torch.cat([size, size], -1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd", [8, 16, 24, 40, 64, 80, 128])
@pytest.mark.parametrize("theta", [None, 10000.0, 500000.0])
def test_append(theta, hd, dtype):
    B, T, Hq, Hkv, page = 3, 37, 4, 2, 16
    g = torch.Generator(device=DEV).manual_seed(hd)
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * hd, device=DEV, generator=g).to(dtype)
    starts, counts = [0, 5, 131000], [37, 20, 0]
    table = torch.full((B, 8300), -1, dtype=torch.int32)
    table[0, :3] = torch.tensor([4, 1, 9])
    table[1, :2] = torch.tensor([0, 7])
    kc, vc = (torch.full((12, Hkv, page, hd), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    st, ct = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in (starts, counts))
    q, k = ops.cache_append(qkv, kc, vc, table.to(DEV), st, Hq, Hkv, theta=theta, counts=ct, return_k=True)
    check_device_status()
    want, size = _append64(qkv, st, Hq, Hkv, hd, theta)
    bound = size + half_step(dtype) * want.abs()
    check("q", q, (want[:, :, :Hq], bound[:, :, :Hq]))
    check("k", k, (want[:, :, Hq:], bound[:, :, Hq:]))
    kref, vref = torch.full_like(kc, 7.0), torch.full_like(vc, 7.0)
    v = qkv.unflatten(-1, (Hq + 2 * Hkv, hd))[:, :, Hq + Hkv:]
    for b in range(B):
        for t in range(counts[b]):
            pos = starts[b] + t
            kref[table[b, pos // page], :, pos % page] = k[b, t]
            vref[table[b, pos // page], :, pos % page] = v[b, t]
    assert torch.equal(kc, kref) and torch.equal(vc, vref)     # the other rows are as they were


def test_append_far_positions_and_single_tokens():
    """Positions up to 2^31 - 1: the angle is taken in 64 bits."""
    Hq, Hkv, hd, page = 2, 1, 64, 1 << 20
    starts = torch.tensor([0, 1, 131071, 2 ** 24 + 1, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    B = starts.numel()
    table = torch.zeros(B, 2048, dtype=torch.int32, device=DEV)
    table += torch.arange(B, device=DEV, dtype=torch.int32)[:, None]
    kc, vc = (torch.zeros(B, Hkv, page, hd, device=DEV) for _ in range(2))
    qkv = torch.randn(B, 1, (Hq + 2 * Hkv) * hd, device=DEV)
    q, k = ops.cache_append(qkv, kc, vc, table, starts, Hq, Hkv, theta=10000.0, return_k=True)
    check_device_status()
    want, size = _append64(qkv, starts, Hq, Hkv, hd, 10000.0)
    bound = size + half_step(F32) * want.abs()
    check("q", q, (want[:, :, :Hq], bound[:, :, :Hq]))
    check("k", k, (want[:, :, Hq:], bound[:, :, Hq:]))
    for b, p in enumerate(starts.tolist()):
        assert torch.equal(kc[b, 0, p % page], k[b, 0, 0])


@pytest.mark.parametrize("window,sinks", [(8, 0), (8, 3), (100, 2), (1, 0)])
def test_append_keeps_what_a_window_sees(window, sinks):
    """A ring of pages: positions that fall out of the window are not written over those that stay."""
    B, T, Hq, Hkv, hd, page = 2, 90, 2, 1, 64, 4
    ring = (window + page - 1) // page + 1
    sp = (sinks + page - 1) // page
    table = torch.empty(B, 40, dtype=torch.int32)
    for b in range(B):
        for i in range(40):
            table[b, i] = b * (sp + ring) + (i if i < sp else sp + (i - sp) % ring)
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * hd, device=DEV).to(BF)
    kc, vc = (torch.full((B * (sp + ring), Hkv, page, hd), float("nan"), dtype=BF, device=DEV) for _ in range(2))
    starts = torch.tensor([0, 33], dtype=torch.int32, device=DEV)
    counts = torch.tensor([90, 71], dtype=torch.int32, device=DEV)
    q, k = ops.cache_append(qkv, kc, vc, table.to(DEV), starts, Hq, Hkv, counts=counts, window=window, sinks=sinks, return_k=True)
    check_device_status()
    v = qkv.unflatten(-1, (Hq + 2 * Hkv, hd))[:, :, Hq + Hkv:]
    last = torch.stack([q[0, 89], q[1, 70]])
    # the second sequence's sinks were appended before this call: keep to windows that do not need them
    o = ops.paged_attention(last[:1], kc, vc, table[:1].to(DEV), counts[:1], window, sinks)
    check("o", o, _expect(last[:1], [(k[0].cpu(), v[0].cpu())], [90], window, sinks))
    o = ops.paged_attention(last[1:], kc, vc, table[1:].to(DEV), counts[1:] + 33, min(window, 71), 0)
    full = [torch.cat([torch.zeros(33, Hkv, hd, dtype=BF), t[1, :71].cpu()]) for t in (k, v)]
    check("o", o, _expect(last[1:], [tuple(full)], [104], min(window, 71), 0))


def test_strided_and_unaligned_inputs():
    Hq, Hkv, hd, page = 4, 2, 64, 16
    qkv = torch.randn(2, 3, 512, device=DEV).to(BF)
    wide = torch.zeros(2, 5, 2 * 512 + 8, device=DEV, dtype=BF)
    wide[:, :3, 8:520] = qkv
    odd = torch.zeros(2 * 3 * 512 + 1, device=DEV, dtype=BF)[1:].view(2, 3, 512)
    odd.copy_(qkv)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([2, 7], dtype=torch.int32, device=DEV)
    seen = []
    for x in (qkv, wide[:, :3, 8:520], odd, qkv.transpose(1, 2).contiguous().transpose(1, 2)):
        kc, vc = (torch.zeros(2, Hkv, page, hd, device=DEV, dtype=BF) for _ in range(2))
        q = ops.cache_append(x, kc, vc, table, starts, Hq, Hkv, theta=1e4)
        lengths = starts + 3
        for qq in (q[:, 2], q[:, 2].transpose(1, 2).contiguous().transpose(1, 2)):
            seen.append((q, kc, vc, ops.paged_attention(qq, kc, vc, table, lengths)))
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))
    check_device_status()


def test_pages_outside_the_cache_are_reported_and_not_followed():
    Hq, Hkv, hd, page = 2, 1, 64, 4
    kc, vc, table, rows = _cache([12, 12], Hkv, hd, page, BF, slack=0)
    q = torch.randn(2, Hq, hd, device=DEV).to(BF)
    lengths = torch.tensor([12, 12], dtype=torch.int32, device=DEV)
    good = ops.paged_attention(q, kc, vc, table, lengths)
    check_device_status()
    for bad in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[1, 1] = bad
        o = ops.paged_attention(q, kc, vc, broken, lengths)
        with pytest.raises(RuntimeError, match="status 4"):
            check_device_status()
        assert torch.equal(o[0], good[0])
        before = kc.clone(), vc.clone()
        ops.cache_append(torch.randn(2, 1, 4 * hd, device=DEV).to(BF), kc, vc, broken,
                         torch.tensor([3, 5], dtype=torch.int32, device=DEV), Hq, Hkv,
                         counts=torch.tensor([0, 1], dtype=torch.int32, device=DEV))
        with pytest.raises(RuntimeError, match="status 4"):
            check_device_status()
        assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(before, (kc, vc)))
    for n in (-1, 13, 2 ** 31 - 1):
        o = ops.paged_attention(q, kc, vc, table, torch.tensor([12, n], dtype=torch.int32, device=DEV))
        with pytest.raises(RuntimeError, match="status 4"):
            check_device_status()
        assert torch.equal(o[0], good[0])
    for start in (-1, 12, 2 ** 31 - 1):
        ops.cache_append(torch.randn(2, 2, 4 * hd, device=DEV).to(BF), kc, vc, table,
                         torch.tensor([0, start], dtype=torch.int32, device=DEV), Hq, Hkv, theta=1e4)
        with pytest.raises(RuntimeError, match="status 4"):
            check_device_status()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_caches_without_pages_and_tables_without_entries(dtype):
    """Nothing can be held: positions are reported, sequences of length 0 are served."""
    q = torch.ones(2, 2, 64, device=DEV, dtype=dtype)
    zero, some = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 0], [0, 3]))
    for n_pages, width in ((0, 2), (4, 0), (0, 0)):
        kc, vc = (torch.zeros(n_pages, 1, 4, 64, device=DEV, dtype=dtype) for _ in range(2))
        table = torch.zeros(2, width, dtype=torch.int32, device=DEV)
        assert not ops.paged_attention(q, kc, vc, table, zero).any()
        check_device_status()
        assert not ops.paged_attention(q, kc, vc, table, some).any()
        with pytest.raises(RuntimeError, match="status 4"):
            check_device_status()
        ops.cache_append(torch.ones(2, 1, 4 * 64, device=DEV, dtype=dtype), kc, vc, table, zero, 2, 1)
        with pytest.raises(RuntimeError, match="status 4"):
            check_device_status()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_empty_batches(dtype):
    kc, vc = (torch.zeros(4, 1, 4, 64, device=DEV, dtype=dtype) for _ in range(2))
    table, none = torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ops.paged_attention(torch.zeros(0, 2, 64, device=DEV, dtype=dtype), kc, vc, table, none).shape == (0, 2, 64)
    for B, T in ((0, 3), (1, 0)):
        q, k = ops.cache_append(torch.zeros(B, T, 4 * 64, device=DEV, dtype=dtype), kc, vc, table.new_zeros(B, 3), none.new_zeros(B), 2,
                                1, theta=1e4, return_k=True)
        assert q.shape == (B, T, 2, 64) and k.shape == (B, T, 1, 64)
    check_device_status()


def test_infinite_and_undefined_rows_that_nobody_sees():
    for fill in (float("nan"), float("inf"), torch.finfo(BF).min):
        kc, vc, table, rows = _cache([130, 5], 2, 64, 16, BF, fill=fill, seed=2)
        q = torch.randn(2, 8, 64, device=DEV).to(BF)
        lengths = torch.tensor([130, 5], dtype=torch.int32, device=DEV)
        o = ops.paged_attention(q, kc, vc, table, lengths)
        check("o", o, _expect(q, rows, [130, 5], None, 0))
        kc2, vc2 = kc.clone(), vc.clone()
        kc2[table[0, 1].long()], vc2[table[0, 1].long()] = fill, fill       # positions 16..31, outside the window
        o = ops.paged_attention(q, kc2, vc2, table, lengths, 40, 3)
        check("o", o, _expect(q, rows, [130, 5], 40, 3))


def test_scores_of_minus_infinity():
    """A key row with an infinite element: its score is -inf for the queries of the other sign, and it takes no part."""
    kc, vc, table, rows = _cache([40], 1, 64, 16, F32, fill=0.0)
    q = torch.rand(1, 2, 64, device=DEV) + 0.5
    kc[table[0, 0].long(), 0, 0, 3] = -math.inf
    lengths = torch.tensor([40], dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, kc, vc, table, lengths)
    k, v = rows[0]
    check("o", o, _expect(q, [(k[1:], v[1:])], [39], None, 0))


def test_refusals():
    kc, vc, table, _ = _cache([12, 12], 2, 64, 4, BF)
    n = torch.tensor([12, 12], dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 4, 64, device=DEV, dtype=BF)
    qkv = torch.zeros(2, 1, 8 * 64, device=DEV, dtype=BF)
    for args in ((q.half(), kc.half(), vc.half(), table, n), (q.float(), kc, vc, table, n), (q, kc, vc[:1], table, n),
                 (q, kc.transpose(1, 2), vc.transpose(1, 2), table, n), (q, kc, vc, table.long(), n), (q, kc, vc, table, n.long()),
                 (q, kc, vc, table[:1], n), (q, kc, vc, table, n[:1]), (q, kc, vc, table.cpu(), n), (q[:, :3], kc, vc, table, n),
                 (q[..., :32], kc, vc, table, n), (q[0], kc, vc, table, n), (q, kc, vc, table, n, 0), (q, kc, vc, table, n, 4, -1)):
        with pytest.raises(RuntimeError, match="titb200 paged_attention"):
            ops.paged_attention(*args)
    for args, kw in (((qkv, kc, vc, table, n, 4, 1), {}), ((qkv, kc, vc, table, n, 3, 2), {}), ((qkv[0], kc, vc, table, n, 4, 2), {}),
                     ((qkv, kc, vc, table, n.float(), 4, 2), {}), ((qkv, kc, vc, table, n, 4, 2), {"theta": -1.0}),
                     ((qkv, kc, vc, table, n, 4, 2), {"theta": 0.0}), ((qkv, kc, vc, table, n, 4, 2), {"theta": math.inf}),
                     ((qkv, kc, vc, table, n, 4, 2), {"counts": n.cpu()}), ((qkv, kc, vc, table, n, 4, 2), {"window": 0}),
                     ((qkv, kc.float(), vc.float(), table, n, 4, 2), {})):
        with pytest.raises(RuntimeError, match="titb200 cache_append"):
            ops.cache_append(*args, **kw)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.paged_attention(q.requires_grad_(), kc, vc, table, n)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.cache_append(qkv.requires_grad_(), kc, vc, table, n, 4, 2)


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_captured_and_replayed_with_other_lengths(dtype, hd):
    """Two graphs of different sizes, replayed in turn on two streams, with lengths, tables and queries changed in between."""
    runs, keep = [], []
    for seed, lens in ((1, [700, 3]), (2, [1500, 40, 9, 100])):
        kc, vc, table, rows = _cache(lens, 2, hd, 16, dtype, seed=seed)
        q = torch.randn(len(lens), 8, hd, device=DEV).to(dtype)
        n = torch.tensor(lens, dtype=torch.int32, device=DEV)
        ops.paged_attention(q, kc, vc, table, n)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = ops.paged_attention(q, kc, vc, table, n)
        runs.append((graph, o, q, n, rows, lens))
        keep.append((kc, vc, table))          # a graph does not keep its inputs
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for shrink in (0, 1, 2):
        torch.cuda.synchronize()
        for graph, o, q, n, rows, lens in runs:
            q.normal_()
            n.copy_(torch.tensor([max(0, x - shrink * 50) for x in lens], dtype=torch.int32))
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for graph, o, q, n, rows, lens in runs:
            now = n.tolist()
            check("o", o, _expect(q, [(k[:m], v[:m]) for (k, v), m in zip(rows, now)], now, None, 0))


def test_a_write_counts_as_one():
    """Autograd refuses a cache that it has kept and that tokens were appended to; in inference mode there is nothing to count."""
    kc, vc = (torch.zeros(2, 2, 16, 64, device=DEV) for _ in range(2))
    table, lengths = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([[0, 1]], [3]))
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = (kc * w).sum()
    ops.cache_append(torch.zeros(1, 1, 8 * 64, device=DEV), kc, vc, table, lengths, 4, 2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        qkv = torch.randn(1, 1, 8 * 64, device=DEV)
        a, b = torch.zeros_like(kc), torch.zeros_like(vc)
        out = ops.cache_append(qkv, a, b, table, lengths, 4, 2, theta=1e4)
        got = ops.paged_attention(out[:, 0], a, b, table, lengths + 1, window=1)
        assert torch.equal(got[0], qkv[0, 0, 6 * 64:].view(2, 64).repeat_interleave(2, 0))
        q = torch.randn(1, 5, 2, 64, device=DEV)
        assert torch.equal(ops.window_attention(q, q, q, 1), q)


def test_results_do_not_change_from_run_to_run():
    kc, vc, table, _ = _cache([5000, 100, 7, 900], 2, 128, 64, BF, fill=0.0)
    q = torch.randn(4, 8, 128, device=DEV).to(BF)
    n = torch.tensor([5000, 100, 7, 900], dtype=torch.int32, device=DEV)
    first = ops.paged_attention(q, kc, vc, table, n)
    for _ in range(20):
        assert torch.equal(first, ops.paged_attention(q, kc, vc, table, n))


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_prompt_then_tokens_is_attention_over_the_whole_sequence(window, sinks, dtype, hd):
    """The run as a user makes it: a prompt's attention over itself and its append, then one token at a time over the cache,
    against the same rows of one attention over the whole sequence."""
    B, T, new, Hq, Hkv, page = 2, 90, 12, 4, 2, 16
    g = torch.Generator(device=DEV).manual_seed(6)
    qkv = torch.randn(B, T + new, (Hq + 2 * Hkv) * hd, device=DEV, generator=g).to(dtype)
    width = (T + new + page - 1) // page
    table = torch.randperm(B * width, device=DEV, generator=g).int().view(B, width)
    kc, vc = (torch.full((B * width, Hkv, page, hd), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
    starts = torch.zeros(B, dtype=torch.int32, device=DEV)
    heads = qkv.unflatten(-1, (Hq + 2 * Hkv, hd))
    kw = dict(theta=10000.0, window=window, sinks=sinks)
    qs, ks, outs = [], [], []
    q, k = ops.cache_append(qkv[:, :T], kc, vc, table, starts, Hq, Hkv, return_k=True, **kw)
    outs.append(ops.window_attention(q, k, heads[:, :T, Hq + Hkv:], window, sinks))
    qs.append(q), ks.append(k)
    for t in range(T, T + new):
        q, k = ops.cache_append(qkv[:, t:t + 1], kc, vc, table, starts + t, Hq, Hkv, return_k=True, **kw)
        outs.append(ops.paged_attention(q[:, 0], kc, vc, table, starts + t + 1, window, sinks)[:, None])
        qs.append(q), ks.append(k)
    i = torch.arange(T + new)
    ahead = i[:, None] - i[None]
    mask = (ahead >= 0) & ((ahead < (window or 10 ** 9)) | (i[None] < sinks))
    want = attention64(torch.cat(qs, 1), torch.cat(ks, 1), heads[:, :, Hq + Hkv:], None, mask)
    check("o", torch.cat(outs, 1), want["o"])
    check_device_status()
