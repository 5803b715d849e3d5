"""Models over a paged cache and with a bounded context, on the CPU: the same logits as a run over the whole sequence."""
import pytest
import torch

from tinyinfinitrain_b200 import data, nn
from tinyinfinitrain_b200._lib import C
from tinyinfinitrain_b200.cli import train_main
from tinyinfinitrain_b200.models import GPT2, LLaMA3, GPT2Config, LLaMA3Config
from tinyinfinitrain_b200.utils import DecodeStep, generate

WINDOWS = [(0, 0), (5, 0), (5, 2), (40, 1)]


def _models(window, sinks):
    kw = dict(block_size=48, n_layer=2, n_head=4, n_embd=64, attention_window=window, attention_sinks=sinks)
    yield GPT2(GPT2Config(vocab_size=97, **kw)).eval()
    yield LLaMA3(LLaMA3Config(vocab_size=97, n_kv_head=2, ffn_dim=96, **kw)).eval()


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("page", [1, 4, 16])
def test_cached_logits_are_those_of_the_whole_sequence(window, sinks, page):
    torch.manual_seed(0)
    idx = torch.randint(0, 97, (3, 30))
    lens = torch.tensor([11, 1, 7], dtype=torch.int32)
    for model in _models(window, sinks):
        with torch.no_grad():
            full = [model(idx[b:b + 1])[0] for b in range(3)]
            cache = model.new_cache(3, page_size=page)
            logits = model(idx[:, :11], cache=cache, counts=lens)
            for t in range(15):
                for b in range(3):
                    assert torch.allclose(logits[b], full[b][int(lens[b]) + t - 1], atol=2e-5), (t, b)
                nxt = torch.stack([idx[b, int(lens[b]) + t] for b in range(3)])
                logits = model(nxt[:, None], cache=cache)
        assert cache.lengths.tolist() == [26, 16, 22]


def test_a_window_holds_a_ring_of_pages():
    cfg = LLaMA3Config(block_size=4096, vocab_size=50, n_layer=1, n_head=2, n_kv_head=1, n_embd=16, ffn_dim=16, attention_window=10,
                       attention_sinks=3)
    cache = LLaMA3(cfg).new_cache(2, page_size=4)
    assert cache.k.shape[1] == 2 * (1 + 4) and cache.page_table.shape == (2, 1024)
    assert cache.page_table[0, :7].tolist() == [0, 1, 2, 3, 4, 1, 2] and int(cache.page_table[1].min()) == 5


def test_an_idle_sequence_stays_as_it_is():
    model = next(iter(_models(0, 0)))
    cache = model.new_cache(2, page_size=4)
    model(torch.randint(0, 97, (2, 5)), cache=cache, counts=torch.tensor([5, 3], dtype=torch.int32))
    held = cache.k[:, cache.page_table[1].long()].clone()
    model(torch.randint(0, 97, (2, 1)), cache=cache, counts=torch.tensor([1, 0], dtype=torch.int32))
    assert cache.lengths.tolist() == [6, 3] and torch.equal(held, cache.k[:, cache.page_table[1].long()])


def test_counts_outside_the_tokens_at_hand():
    for model in _models(0, 0):
        idx = torch.randint(0, 97, (2, 5))
        caches = [model.new_cache(2, page_size=4) for _ in range(2)]
        a, b = (model(idx, cache=c, counts=torch.tensor(n, dtype=torch.int32)) for c, n in zip(caches, ([9, -4], [5, 0])))
        assert torch.equal(a, b) and caches[0].lengths.tolist() == [5, 0]


def test_training_with_a_window_differs_and_runs():
    torch.manual_seed(1)
    idx = torch.randint(0, 97, (2, 20))
    for plain, bounded in zip(_models(0, 0), _models(5, 1)):
        a, b = plain(idx), bounded(idx)
        assert torch.allclose(a[:, :5], b[:, :5], atol=1e-6) and not torch.allclose(a[:, 12:], b[:, 12:], atol=1e-3)
        _, loss = bounded(idx, idx)
        loss.backward()
        assert all(torch.isfinite(p.grad).all() and p.grad.any() for p in bounded.parameters())


def test_generate_and_decode_step():
    for model in _models(6, 1):
        prompts = [[5, 6, 7], [1], [9, 8, 7, 6, 5, 4]]
        got = generate(model, prompts, 6, page_size=4)
        for p, new in zip(prompts, got):
            seq = list(p)
            for _ in range(6):
                seq.append(int(model(torch.tensor([seq]))[0, -1].argmax()))
            assert seq[len(p):] == new
        assert generate(model, prompts, 0) == [[], [], []]
        cache = model.new_cache(2)
        assert DecodeStep(model, cache)(torch.tensor([3, 4])).shape == (2, 97)
        with pytest.raises(ValueError):
            generate(model, [[]], 3)


def test_generate_text_over_a_cache(tmp_path):
    table = [f"<{i}>".encode() for i in range(50300)]
    path = str(tmp_path / "tok.bin")
    C.write_tokenizer(path, table, 20240328, 50256)
    tk = data.Tokenizer(path)
    model = GPT2(GPT2Config(block_size=32, vocab_size=50257, n_layer=1, n_head=2, n_embd=16))
    assert tk.GenerateText(model, 2, 32, 14, "cpu", use_cache=True) == tk.GenerateText(model, 2, 32, 14, "cpu")


def test_command_line_switches(tmp_path, capsys):
    table = [f"<{i}>".encode() for i in range(50300)]
    path = str(tmp_path / "tok.bin")
    C.write_tokenizer(path, table, 20240328, 50256)
    argv = ["--device", "cpu", "--dtype", "float32", "--synthetic", "--num_iteration", "1", "--batch_size", "1",
            "--sequence_length", "16", "--n_layer", "1", "--n_embd", "16", "--n_head", "2", "--tokenizer_bin", path,
            "--freq_generate_txt", "1", "--text_length", "8", "--attention_window", "4", "--attention_sinks", "1"]
    assert train_main("gpt2", argv) == 0
    plain = capsys.readouterr().out
    assert train_main("gpt2", argv + ["--kv_cache"]) == 0
    cached = capsys.readouterr().out
    text = lambda out: [line for line in out.splitlines() if line.startswith("The meaning")]
    assert text(plain) and text(plain) == text(cached)
    with pytest.raises(SystemExit):
        train_main("gpt2", argv[:-4] + ["--attention_sinks", "2"])


def test_refusals():
    model = next(iter(_models(0, 0)))
    cache = model.new_cache(2, 8, page_size=4)
    with pytest.raises(ValueError, match="batch"):
        model(torch.zeros(3, 1, dtype=torch.int64), cache=cache)
    with pytest.raises(ValueError, match="positions"):
        model(torch.zeros(2, 9, dtype=torch.int64), cache=cache)
    with pytest.raises(ValueError, match="int32"):
        model(torch.zeros(2, 2, dtype=torch.int64), cache=cache, counts=torch.tensor([1, 2]))
    model(torch.zeros(2, 3, dtype=torch.int64), cache=cache)
    with pytest.raises(ValueError, match="empty cache"):
        model(torch.zeros(2, 2, dtype=torch.int64), cache=cache)
    for _ in range(5):
        model(torch.zeros(2, 1, dtype=torch.int64), cache=cache)
    with pytest.raises(IndexError):
        model(torch.zeros(2, 1, dtype=torch.int64), cache=cache)
    cache.reset()
    model(torch.zeros(2, 3, dtype=torch.int64), cache=cache)
    with pytest.raises(ValueError, match="block size"):
        model.new_cache(1, 49)
    for bad in (dict(batch=0), dict(window=0), dict(sinks=-1)):
        with pytest.raises(ValueError):
            nn.PagedKVCache(**{**dict(n_layer=1, batch=1, max_len=4, n_kv_head=1, head_dim=8), **bad})
