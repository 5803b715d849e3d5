"""Generation on the GPU looks at the kernels' status before it returns text."""
import pytest
import torch

from tinyinfinitrain_b200 import data
from tinyinfinitrain_b200._lib import C
from tinyinfinitrain_b200.models import GPT2, GPT2Config
from tinyinfinitrain_b200.parallel.health import check_device_status
from tinyinfinitrain_b200.utils import generate

pytestmark = pytest.mark.gpu


def _model(monkeypatch, pages):
    """A model whose caches are smaller than asked for, so that sequences outgrow them."""
    model = GPT2(GPT2Config(block_size=64, vocab_size=50257, n_layer=1, n_head=2, n_embd=32), device="cuda", dtype=torch.bfloat16)
    whole = model.new_cache
    if pages:
        monkeypatch.setattr(model, "new_cache", lambda batch, max_len=None, page_size=16: whole(batch, pages * 16, 16), raising=False)
    return model


@pytest.mark.parametrize("use_graph", [True, False])
def test_generate(monkeypatch, use_graph):
    check_device_status()
    with pytest.raises(RuntimeError, match="status 4"):
        generate(_model(monkeypatch, 1), [[1, 2, 3]], 20, use_graph=use_graph)
    assert len(generate(_model(monkeypatch, 0), [[1, 2, 3]], 20, use_graph=use_graph)[0]) == 20


def test_generate_text(monkeypatch, tmp_path):
    path = str(tmp_path / "tok.bin")
    C.write_tokenizer(path, [f"<{i}>".encode() for i in range(50300)], 20240328, 50256)
    tk = data.Tokenizer(path)
    check_device_status()
    with pytest.raises(RuntimeError, match="status 4"):
        tk.GenerateText(_model(monkeypatch, 1), 1, 64, 40, "cuda", use_cache=True)
    assert tk.GenerateText(_model(monkeypatch, 0), 1, 64, 40, "cuda", use_cache=True).startswith("The meaning of life is")
