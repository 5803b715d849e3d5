"""The paged cache's operators on the CPU: values, bad pages and lengths, refusals."""
import pytest
import torch

from tinyinfinitrain_b200 import ops

from _attention_bounds import attention64, check


def _filled(lengths, Hkv=2, hd=16, page=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lengths]
    order = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    kc, vc = (torch.full((sum(need) + 2, Hkv, page, hd), float("nan")) for _ in range(2))
    rows, at = [], 0
    for b, n in enumerate(lengths):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        k, v = torch.randn(n, Hkv, hd, generator=g), torch.randn(n, Hkv, hd, generator=g)
        pos = torch.arange(n)
        kc[table[b, pos // page].long(), :, pos % page] = k
        vc[table[b, pos // page].long(), :, pos % page] = v
        rows.append((k, v))
    return kc, vc, table, rows


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (5, 2), (100, 3)])
def test_paged_attention(window, sinks):
    lengths = [1, 0, 9, 23]
    kc, vc, table, rows = _filled(lengths)
    q = torch.randn(4, 6, 16)
    o = ops.paged_attention(q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32), window, sinks)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not o[b].any()
            continue
        p = torch.arange(n)
        seen = (p >= n - (window or n)) | (p < sinks)
        k, v = (t[seen][None] for t in rows[b])
        want = attention64(q[b][None, None], k, v, None, torch.ones(1, int(seen.sum()), dtype=torch.bool))["o"]
        check("o", o[b][None, None], want)


def test_append_then_attend_is_attention_over_the_sequence():
    B, T, Hq, Hkv, hd, page = 2, 11, 4, 2, 16, 4
    qkv = torch.randn(B, T, (Hq + 2 * Hkv) * hd)
    table = torch.randperm(6).int().view(2, 3)
    kc, vc = torch.zeros(6, Hkv, page, hd), torch.zeros(6, Hkv, page, hd)
    starts = torch.zeros(B, dtype=torch.int32)
    q, k = ops.cache_append(qkv[:, :7], kc, vc, table, starts, Hq, Hkv, theta=1e4, return_k=True)
    rot = ops.rope_qkv(qkv, Hq + Hkv, hd, 0, 1e4)
    assert torch.allclose(q.flatten(2), rot[:, :7, :Hq * hd], atol=1e-5)
    full = ops.causal_attention_qkv(rot, Hq, Hkv)
    for t in range(7, T):
        q = ops.cache_append(qkv[:, t:t + 1], kc, vc, table, starts + t, Hq, Hkv, theta=1e4)
        o = ops.paged_attention(q[:, 0], kc, vc, table, starts + t + 1)
        assert torch.allclose(o, full[:, t], atol=1e-5)


def test_counts_leave_the_other_rows_alone():
    qkv = torch.randn(2, 5, 4 * 8)
    kc, vc = torch.full((4, 1, 4, 8), 3.0), torch.full((4, 1, 4, 8), 3.0)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32)
    ops.cache_append(qkv, kc, vc, table, torch.tensor([1, 6], dtype=torch.int32), 2, 1,
                     counts=torch.tensor([4, 0], dtype=torch.int32))
    k = qkv.view(2, 5, 4, 8)[:, :, 2]
    assert torch.equal(kc[2, 0, 1:], k[0, :3]) and torch.equal(kc[0, 0, 0], k[0, 3])
    assert (kc[2, 0, 0] == 3).all() and (kc[0, 0, 1:] == 3).all() and (kc[[1, 3]] == 3).all()


def test_append_into_a_ring():
    """Six positions of ring, a window of four: eleven tokens at once leave the last four and the first one."""
    qkv = torch.randn(1, 11, 3 * 8)
    kc, vc = torch.zeros(4, 1, 2, 8), torch.zeros(4, 1, 2, 8)
    table = torch.tensor([[0, 1, 2, 3, 1, 2]], dtype=torch.int32)
    n = torch.tensor([11], dtype=torch.int32)
    ops.cache_append(qkv, kc, vc, table, torch.zeros(1, dtype=torch.int32), 1, 1, window=4, sinks=1)
    k = qkv.view(11, 3, 8)[:, 1]
    assert torch.equal(kc[0, 0, 0], k[0]) and not kc[0, 0, 1].any()
    assert torch.equal(torch.stack([kc[3, 0, 1], kc[1, 0, 0], kc[1, 0, 1], kc[2, 0, 0]]), k[7:])
    q = torch.randn(1, 1, 8)
    o = ops.paged_attention(q, kc, vc, table, n, 4, 1)
    keep = torch.tensor([0, 7, 8, 9, 10])
    s = (q[0] @ k[keep].t() / 8 ** 0.5).softmax(-1)
    assert torch.allclose(o[0], s @ qkv.view(11, 3, 8)[keep, 2], atol=1e-6)


@pytest.mark.parametrize("bad", [-1, 8, 2 ** 31 - 1])
def test_bad_pages(bad):
    kc, vc, table, _ = _filled([12, 12])
    table[1, 1] = bad
    n = torch.tensor([12, 12], dtype=torch.int32)
    with pytest.raises(IndexError, match="sequence 1"):
        ops.paged_attention(torch.randn(2, 2, 16), kc, vc, table, n)
    ops.paged_attention(torch.randn(2, 2, 16), kc, vc, table, n, 4)        # the window does not reach that page
    with pytest.raises(IndexError, match="sequence 1"):
        ops.cache_append(torch.randn(2, 1, 6 * 16), kc, vc, table, torch.tensor([3, 5], dtype=torch.int32), 2, 2)


def test_bad_positions():
    kc, vc, table, _ = _filled([12, 12])
    for n in (-1, 13):
        with pytest.raises(IndexError):
            ops.paged_attention(torch.randn(2, 2, 16), kc, vc, table, torch.tensor([12, n], dtype=torch.int32))
    for start in (-1, 12):
        with pytest.raises(IndexError):
            ops.cache_append(torch.randn(2, 1, 6 * 16), kc, vc, table, torch.tensor([0, start], dtype=torch.int32), 2, 2)


def test_refusals():
    kc, vc, table, _ = _filled([12, 12])
    n = torch.tensor([12, 12], dtype=torch.int32)
    q = torch.zeros(2, 4, 16)
    qkv = torch.zeros(2, 1, 8 * 16)
    for args in ((q.half(), kc.half(), vc.half(), table, n), (q.bfloat16(), kc, vc, table, n), (q, kc, vc[:1], table, n),
                 (q, kc.transpose(1, 2), vc.transpose(1, 2), table, n), (q, kc, vc, table.long(), n), (q, kc, vc, table, n.long()),
                 (q, kc, vc, table[:1], n), (q, kc, vc, table, n[:1]), (q[:, :3], kc, vc, table, n), (q[..., :8], kc, vc, table, n),
                 (q[0], kc, vc, table, n), (q, kc, vc, table, n, 0), (q, kc, vc, table, n, 4, -1)):
        with pytest.raises(RuntimeError, match="titb200 paged_attention"):
            ops.paged_attention(*args)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="scale"):
            ops.paged_attention(q, kc, vc, table, n, scale=scale)
    for args, kw in (((qkv, kc, vc, table, n, 4, 1), {}), ((qkv, kc, vc, table, n, 3, 2), {}), ((qkv[0], kc, vc, table, n, 4, 2), {}),
                     ((qkv, kc, vc, table, n.float(), 4, 2), {}), ((qkv, kc, vc, table, n, 4, 2), {"theta": -1.0}),
                     ((qkv, kc, vc, table, n, 4, 2), {"theta": 0.0}), ((qkv, kc, vc, table, n, 4, 2), {"theta": float("inf")}),
                     ((qkv, kc, vc, table, n, 4, 2), {"counts": n[:1]}), ((qkv, kc, vc, table, n, 4, 2), {"window": 0}),
                     ((qkv, kc.double(), vc.double(), table, n, 4, 2), {})):
        with pytest.raises(RuntimeError, match="titb200 cache_append"):
            ops.cache_append(*args, **kw)
    with pytest.raises(RuntimeError, match="share memory"):
        ops.cache_append(qkv, kc, kc, table, n, 4, 2)
    both = torch.zeros(3 * kc.shape[0], *kc.shape[1:])
    with pytest.raises(RuntimeError, match="share memory"):
        ops.cache_append(qkv, both[:kc.shape[0]], both[1:1 + kc.shape[0]], table, n, 4, 2)
    for scale in (1e-60, 1e60):     # zero and infinity in 32 bits
        with pytest.raises(RuntimeError, match="scale"):
            ops.paged_attention(q, kc, vc, table, n, scale=scale)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.paged_attention(q.requires_grad_(), kc, vc, table, n)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.cache_append(qkv.requires_grad_(), kc, vc, table, n, 4, 2)
