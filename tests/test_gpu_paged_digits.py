"""Attention over the paged cache in bf16: as exact as its output's rounding, and infinities that a query sees."""
import pytest
import torch

from tinyinfinitrain_b200 import ops
from tinyinfinitrain_b200._lib import C

from _attention_digits import check_digits, output64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _cache(lengths, Hkv, hd, page, dtype, g):
    """A cache filled with normal numbers, and its keys and values by sequence and position, [B, longest, Hkv, hd]."""
    width = (max(lengths) + page - 1) // page
    table = torch.randperm(len(lengths) * width, generator=g, device=DEV).int().view(len(lengths), width)
    kc, vc = (torch.randn(table.numel(), Hkv, page, hd, generator=g, device=DEV).to(dtype) for _ in range(2))
    rows = [c[table.long()].transpose(2, 3).reshape(len(lengths), width * page, Hkv, hd) for c in (kc, vc)]
    return kc, vc, table, rows


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (25, 25), (32, 2), (34, 2)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 3)])
def test_the_output_is_off_by_its_rounding(window, sinks, hd, Hq, Hkv):
    g = torch.Generator(device=DEV).manual_seed(hd + Hq)
    lengths = [1, 2, 33, 64, 100, 129, 250, 300, 333, 401, 512, 600, 777, 900, 1000, 1024, 1500, 1999, 2048, 3000] * (2 if Hq > 8 else 4)
    kc, vc, table, (k, v) = _cache(lengths, Hkv, hd, 16, BF, g)
    q = (2 * torch.randn(len(lengths), Hq, hd, generator=g, device=DEV)).to(BF)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, kc, vc, table, n, window, sinks)
    p = torch.arange(k.shape[1], device=DEV)
    values, bounds = [], []
    for b, m in enumerate(lengths):
        seen = (p < m) & ((p >= m - (window or m)) | (p < sinks))
        value, bound = output64(q[b][None, None], k[b, seen][None], v[b, seen][None], torch.ones(1, int(seen.sum()), dtype=torch.bool))
        values.append(value[0, 0]), bounds.append(bound[0, 0])
    check_digits("o", o, torch.stack(values), torch.stack(bounds))
    assert C.status_read(True) == 0


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (32, 2)])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64), (BF, 40)])
def test_infinities_that_a_query_sees(dtype, hd, Hq, Hkv):
    """An infinite value is an infinite sum of its sign in its column, one of either sign or an undefined one NaN; the other columns
    are what they are without it."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    lengths = [700, 90]
    kc, vc, table, (k, v) = _cache(lengths, Hkv, hd, 16, dtype, g)
    q = torch.randn(2, Hq, hd, generator=g, device=DEV).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    plain = ops.paged_attention(q, kc, vc, table, n)

    def put(b, pos, d, x):
        vc[table[b, pos // 16].long(), :, pos % 16, d] = x

    inf, nan = float("inf"), float("nan")
    for b, pos, d, x in ((0, 5, 1, inf), (0, 400, 2, -inf), (0, 100, 3, inf), (0, 650, 3, -inf), (0, 699, 4, nan), (1, 0, 5, -inf)):
        put(b, pos, d, x)
    o = ops.paged_attention(q, kc, vc, table, n)
    assert (o[0, :, 1] == inf).all() and (o[0, :, 2] == -inf).all() and torch.isnan(o[0, :, 3:5]).all() and (o[1, :, 5] == -inf).all()
    keep0, keep1 = [0] + list(range(5, hd)), list(range(5)) + list(range(6, hd))
    assert torch.equal(o[0][:, keep0], plain[0][:, keep0]) and torch.equal(o[1][:, keep1], plain[1][:, keep1])
