"""Window attention on the GPU: each row's output is its own, and stays with it on its way out of the kernel."""
import pytest
import torch

from tinyinfinitrain_b200 import ops
from tinyinfinitrain_b200._lib import C

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("training", [False, True])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (F32, 64)])
def test_a_row_that_sees_itself_only_is_its_value(dtype, hd, training):
    """Window 1: the probability is 1 but for the rounding of its exponent, 2^-24 of a score of 60 at most, and what is kept of
    it is off by 2^-17.  Both are far below half a step of the value, which is a number of the output's type: it comes back bit
    for bit, from every row of every tile, whichever lanes move it.  fp32, where no such slack is, comes within two steps of the
    exponent's error, 2^-17."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    for T in (1, 33, 517, 1024):
        for _ in range(8):
            q, k, v = (torch.randn(3, T, 6, hd, device=DEV, generator=g).to(dtype) for _ in range(3))
            v.requires_grad_(training)
            o = ops.window_attention(q, k, v, 1)
            if dtype == BF:
                assert torch.equal(o, v)
            else:
                assert ((o - v).abs() <= 2.0 ** -17 * v.abs()).all()
            if training:
                # dV = P^T dO: P is 1 after its rounding to bf16, and dO a number of the type
                do = torch.randn(o.shape, device=DEV, generator=g).to(dtype)
                dv = torch.autograd.grad(o, v, do)[0]
                assert ((dv.double() - do.double()).abs() <= 2.0 ** -17 * do.double().abs()).all()
    torch.cuda.synchronize()
    assert C.status_read(True) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_query_heads(dtype):
    """Nobody sees the keys: their gradients are zeros, as on the CPU."""
    for device in ("cpu", DEV):
        q = torch.zeros(2, 50, 0, 64, device=device, dtype=dtype, requires_grad=True)
        k, v = (torch.ones(2, 50, 2, 64, device=device, dtype=dtype, requires_grad=True) for _ in range(2))
        if device == DEV:       # memory that the gradients may be given holds something
            del_me = [torch.full((2, 50, 2, 64), 7.0, device=device, dtype=dtype) for _ in range(4)]
            del del_me
        o = ops.window_attention(q, k, v, 5)
        assert o.shape == q.shape
        for grad in torch.autograd.grad(o, (q, k, v), torch.zeros_like(o)):
            assert not grad.any()
