"""Generation at the edges of a model's context and of its arguments, on the CPU."""
import pytest
import torch

from tinyinfinitrain_b200.models import GPT2, LLaMA3, GPT2Config, LLaMA3Config
from tinyinfinitrain_b200.utils import generate


def _models():
    kw = dict(block_size=24, n_layer=1, n_head=2, n_embd=32)
    yield GPT2(GPT2Config(vocab_size=61, **kw)).eval()
    yield LLaMA3(LLaMA3Config(vocab_size=61, n_kv_head=1, ffn_dim=32, **kw)).eval()


@pytest.mark.parametrize("length,new", [(24, 1), (23, 2), (1, 24), (10, 15)])
def test_tokens_up_to_the_end_of_the_context(length, new):
    """The last token is not fed back: with it the sequence is a position longer than the context."""
    for model in _models():
        prompt = [(7 * i + 3) % 61 for i in range(length)]
        seq = list(prompt)
        with torch.no_grad():
            for _ in range(new):
                seq.append(int(model(torch.tensor([seq]))[0, -1].argmax()))
        for page in (4, 16, 64):
            assert generate(model, [prompt], new, page_size=page) == [seq[length:]]


def test_tokens_behind_the_context():
    gpt2 = next(iter(_models()))
    with pytest.raises(ValueError, match="block size"):
        generate(gpt2, [[1] * 24], 2)


def test_caches_of_no_size():
    """No positions is not the default number of them."""
    for model in _models():
        for args in ((1, 0), (1, -3), (0, 8), (1, 8, 0), (1, None, -1)):
            with pytest.raises(ValueError, match="must be positive"):
                model.new_cache(*args)
        assert model.new_cache(1).max_len == model.new_cache(1, None).max_len == 24 and model.new_cache(1, 5).max_len == 5
