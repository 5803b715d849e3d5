"""DecodeStep's arguments, without a GPU."""
import pytest
import torch

from tinyinfinitrain_b200.models import LLaMA3, LLaMA3Config
from tinyinfinitrain_b200.utils import DecodeStep


def _step(batch=3):
    model = LLaMA3(LLaMA3Config(block_size=24, vocab_size=61, n_layer=1, n_head=2, n_kv_head=1, n_embd=32, ffn_dim=32)).eval()
    return DecodeStep(model, model.new_cache(batch))


@pytest.mark.parametrize("shape", [(1,), (2,), (4,), (6,), (1, 1), ()])
def test_another_number_of_tokens_than_sequences(shape):
    """One token was taken for all sequences."""
    step = _step()
    with pytest.raises(ValueError, match="3 sequences"):
        step(torch.zeros(shape, dtype=torch.int64))
    assert step.cache.lengths.tolist() == [0, 0, 0]


def test_logits_or_probabilities_in_place_of_tokens():
    with pytest.raises(ValueError, match="integers"):
        _step()(torch.zeros(3))


def test_tokens_in_any_layout():
    want = _step()(torch.tensor([5, 6, 7]))
    for tokens in (torch.tensor([[5], [6], [7]]), torch.tensor([5, 6, 7], dtype=torch.int32), torch.tensor([[5, 0], [6, 0], [7, 0]])[:, 0],
                   torch.tensor([[5, 6, 7], [0, 0, 0]]).t()[:, :1]):
        assert torch.equal(_step()(tokens), want)
