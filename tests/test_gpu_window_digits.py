"""Window attention in bf16: the output is off by its rounding, and so, beside the roundings of P and dS, are the gradients."""
import pytest
import torch

from tinyinfinitrain_b200 import ops
from tinyinfinitrain_b200._lib import C

from _attention_bounds import visible
from _attention_digits import check_digits, gradients64, output64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("T,window,sinks", [(300, 100, 0), (300, 2, 0), (517, 300, 4), (700, 64, 130), (260, 260, 0), (150, 1, 3)])
@pytest.mark.parametrize("hd,Hq,Hkv", [(64, 8, 2), (128, 6, 3), (64, 5, 5), (40, 6, 2)])
def test_digits(hd, Hq, Hkv, T, window, sinks):
    g = torch.Generator(device=DEV).manual_seed(T + hd)
    q, k, v, do = (torch.randn(2, T, h, hd, device=DEV, generator=g) for h in (Hq, Hkv, Hkv, Hq))
    q, k, v, do = (2 * q).to(BF), k.to(BF), v.to(BF), do.to(BF)
    mask = visible(T, window, sinks)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = ops.window_attention(*leaves, window, sinks)
    grads = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)))
    with torch.no_grad():
        assert torch.equal(o, ops.window_attention(q, k, v, window, sinks))
    check_digits("o", o.detach(), *output64(q, k, v, mask))
    for name, (value, bound) in gradients64(q, k, v, do, mask).items():
        worst = ((grads[name].double() - value).abs() / bound.clamp_min(1e-300)).max().item()
        assert worst <= 1.0, f"{name}: off by {worst:.2f} times its bound"
    assert C.status_read(True) == 0
