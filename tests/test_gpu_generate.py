"""Models over a paged cache and with a bounded context on the GPU."""
import pytest
import torch

import tinyinfinitrain_b200 as tit
from tinyinfinitrain_b200.models import GPT2, LLaMA3, GPT2Config, LLaMA3Config
from tinyinfinitrain_b200.parallel.health import check_device_status
from tinyinfinitrain_b200.utils import DecodeStep, TrainStep, generate

pytestmark = pytest.mark.gpu
DEV = "cuda"
WINDOWS = [(0, 0), (20, 0), (20, 2)]


def _models(window, sinks, dtype, hd=64):
    kw = dict(block_size=256, n_layer=2, n_head=4, n_embd=4 * hd, attention_window=window, attention_sinks=sinks)
    yield GPT2(GPT2Config(vocab_size=1000, **kw), device=DEV, dtype=dtype)
    yield LLaMA3(LLaMA3Config(vocab_size=1024, n_kv_head=2, ffn_dim=256, **kw), device=DEV, dtype=dtype)


def _close(a, b, dtype):
    """Logits of the same tokens through differently ordered sums.  A layer's hidden state is rounded about ten times on its
    way; with two layers some 20 roundings of half a step each, of values of the size of the logits' root mean square times
    the width's square root at most: 64 half steps of the largest logit bound them."""
    u = torch.finfo(dtype).eps / 2
    scale = b.float().abs().max().item()
    return (a.float() - b.float()).abs().max().item() <= 64 * max(u, 2.0 ** -20) * scale


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 16)])
def test_cached_logits_are_those_of_the_whole_sequence(window, sinks, dtype, hd):
    torch.manual_seed(0)
    idx = torch.randint(0, 1000, (3, 80), device=DEV)
    lens = [40, 1, 23]
    for model in _models(window, sinks, dtype, hd):
        with torch.no_grad():
            full = [model(idx[b:b + 1])[0] for b in range(3)]
        cache = model.new_cache(3, page_size=16)
        logits = model(idx[:, :40], cache=cache, counts=torch.tensor(lens, dtype=torch.int32, device=DEV))
        step = DecodeStep(model, cache)
        for t in range(30):
            for b in range(3):
                assert _close(logits[b], full[b][lens[b] + t - 1], dtype), (t, b)
            logits = step(torch.stack([idx[b, lens[b] + t] for b in range(3)]))
        assert cache.lengths.tolist() == [70, 31, 53]
        check_device_status()


def test_captured_steps_are_the_eager_ones():
    for model in _models(20, 2, torch.bfloat16):
        prompts = [[5, 6, 7], [1], list(range(90))]
        a = generate(model, prompts, 40, page_size=16)
        b = generate(model, prompts, 40, page_size=16, use_graph=False)
        assert a == b and all(len(x) == 40 for x in a)
        check_device_status()


def test_two_caches_decoded_in_turn():
    """Two captured steps of one model over caches of their own, replayed alternately, and one of them reused after reset()."""
    model = next(iter(_models(0, 0, torch.bfloat16)))
    alone = [generate(model, p, 12) for p in ([[3, 4, 5]], [[8] * 70, [9]])]
    caches = [model.new_cache(1), model.new_cache(2)]
    steps = [DecodeStep(model, c) for c in caches]
    first = [model(torch.tensor([[3, 4, 5]], device=DEV), cache=caches[0]).argmax(-1),
             model(torch.tensor([[8] * 70, [9] * 70], device=DEV), cache=caches[1],
                   counts=torch.tensor([70, 1], dtype=torch.int32, device=DEV)).argmax(-1)]
    toks, got = list(first), [[f.tolist()] for f in first]
    for _ in range(11):
        for i in (0, 1):
            toks[i] = steps[i](toks[i]).argmax(-1)
            got[i].append(toks[i].tolist())
    for i in (0, 1):
        assert [list(x) for x in zip(*got[i])] == alone[i]
    caches[0].reset()
    tok = model(torch.tensor([[3, 4, 5]], device=DEV), cache=caches[0]).argmax(-1)
    again = [tok.tolist()]
    for _ in range(11):
        tok = steps[0](tok).argmax(-1)
        again.append(tok.tolist())
    assert [list(x) for x in zip(*again)] == alone[0]
    check_device_status()


def test_a_sequence_that_outgrows_its_pages_is_reported():
    model = next(iter(_models(0, 0, torch.bfloat16)))
    cache = model.new_cache(1, 32, page_size=16)
    model(torch.zeros(1, 32, dtype=torch.int64, device=DEV), cache=cache)
    check_device_status()
    model(torch.zeros(1, 1, dtype=torch.int64, device=DEV), cache=cache)
    with pytest.raises(RuntimeError, match="status 4"):
        check_device_status()


@pytest.mark.parametrize("window,sinks", [(20, 0), (50, 3)])
def test_a_captured_training_step_with_a_window(window, sinks):
    """The whole step in a CUDA graph."""
    for model in _models(window, sinks, torch.bfloat16):
        opt = tit.optim.MixedPrecisionAdam(model.parameters(), lr=1e-3)
        before = opt.flat.param.clone()
        step = TrainStep(model, opt, 2, 200, DEV, use_graph=True)
        g = torch.Generator().manual_seed(0)
        x = torch.randint(0, 1000, (2, 200), generator=g).pin_memory()
        y = torch.roll(x, -1, 1).pin_memory()
        step.prepare()
        for _ in range(3):
            loss = float(step(x, y))
            assert loss == loss
        assert not torch.equal(before, opt.flat.param)
        check_device_status()
