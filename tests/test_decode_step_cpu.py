"""DecodeStep's arguments, and on which device and stream it captures, without a GPU."""
import contextlib

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


def test_the_capture_is_on_the_caches_device(monkeypatch):
    """Kernels are launched on the model's device; a capture on another one holds nothing, and its replay does nothing."""
    step, log, current = _step(), [], ["cuda:0"]

    class Stream:
        def __init__(self, device=None):
            self.device = str(device) if device is not None else current[0]

        def wait_stream(self, other):
            log.append(("wait", self.device))

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], str(d)
        yield
        current[0] = before

    @contextlib.contextmanager
    def graph(g, stream=None):
        log.append(("graph", current[0], getattr(stream, "device", "the class's default")))
        yield

    for name, fake in dict(Stream=Stream, CUDAGraph=object, graph=graph, device=device, stream=lambda s: contextlib.nullcontext(),
                           current_stream=lambda d=None: Stream(d), synchronize=lambda d=None: None).items():
        monkeypatch.setattr(torch.cuda, name, fake)
    step.cache.lengths = step.cache.lengths.clone()
    monkeypatch.setattr(step, "device", torch.device("cuda:1"), raising=False)
    step._capture()
    assert [x for x in log if x[0] == "graph"] == [("graph", "cuda:1", "cuda:1")] and current == ["cuda:0"]
