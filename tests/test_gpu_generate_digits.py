"""Logits of bf16 models over a paged cache against an fp32 model of the same weights on the CPU, run over whole sequences."""
import dataclasses

import pytest
import torch

from tinyinfinitrain_b200.models import GPT2, LLaMA3, GPT2Config, LLaMA3Config
from tinyinfinitrain_b200.parallel.health import check_device_status
from tinyinfinitrain_b200.utils import DecodeStep

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
LENGTHS, STEPS = [40, 1, 23], 30


def _model(family, window, sinks, hd):
    kw = dict(block_size=256, n_layer=2, n_head=4, n_embd=4 * hd, attention_window=window, attention_sinks=sinks)
    if family == "gpt2":
        model = GPT2(GPT2Config(vocab_size=1000, **kw), device=DEV, dtype=BF)
    else:
        model = LLaMA3(LLaMA3Config(vocab_size=1024, n_kv_head=2, ffn_dim=256, **kw), device=DEV, dtype=BF)
    with torch.no_grad():       # scores of a few units, and attention that the logits depend on
        for name, p in model.named_parameters():
            if name.endswith("c_attn.weight"):
                p.mul_(5)
            elif name.endswith("attn.c_proj.weight"):
                p.mul_(10)
    return model


def _fp32(model, **changes):
    other = type(model)(dataclasses.replace(model.config, **changes))
    other.load_state_dict({n: t.float().cpu() for n, t in model.state_dict().items()})
    return other


def _rows(full):
    """Of each sequence's logits those that the cached run returns."""
    return torch.stack([full[b][LENGTHS[b] - 1:LENGTHS[b] - 1 + STEPS] for b in range(3)]).double().cpu()


@torch.no_grad()
def _whole(model, idx):
    return _rows([model(idx[b:b + 1].to(model.lm_head.weight.device))[0] for b in range(3)])


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 0), (20, 2)])
@pytest.mark.parametrize("family,hd", [("gpt2", 64), ("llama3", 64), ("llama3", 128)])
def test_cached_logits_are_as_exact_as_those_of_whole_sequences(family, hd, window, sinks):
    """Both runs round the same quantities the same number of times.  Over 90 rows of 1000 logits the norms of what that adds up to
    differ by a few percent; half as much again is far outside.  The limit is a limit only if a run that sees a key too few or too
    many is beyond it, which the fp32 model with such a window shows."""
    idx = torch.randint(0, 1000, (3, 80), generator=torch.Generator().manual_seed(0))
    model = _model(family, window, sinks, hd)
    want = _whole(_fp32(model), idx)
    plain = (_whole(model, idx) - want).norm()
    limit = 1.5 * plain
    for wrong in ([window - 1, window + 1] if window else [60]):
        assert (_whole(_fp32(model, attention_window=wrong), idx) - want).norm() > 2 * limit, wrong
    cache = model.new_cache(3, page_size=16)
    dev = idx.to(DEV)
    logits = model(dev[:, :40], cache=cache, counts=torch.tensor(LENGTHS, dtype=torch.int32, device=DEV))
    step, got = DecodeStep(model, cache), []
    for t in range(STEPS):
        got.append(logits.double().cpu())
        logits = step(torch.stack([dev[b, LENGTHS[b] + t] for b in range(3)]))
    err = (torch.stack(got, 1) - want).norm()
    assert err <= limit, (err.item(), plain.item(), want.norm().item())
    check_device_status()
