"""A bounded context in the tensor-parallel models: 2 CPU ranks (gloo) against the single-process model."""
import os
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _worker(rank, world, port, q, which):
    sys.path.insert(0, ROOT)
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from tinyinfinitrain_b200.models import GPT2, GPT2Config, LLaMA3, LLaMA3Config
        from tinyinfinitrain_b200.models.tp_models import TPTransformer
        from tinyinfinitrain_b200.parallel import mesh as pm
        from tinyinfinitrain_b200.parallel.tp import TPComm

        comm = TPComm(pm.init_mesh(tp=world, pp=1).tp_group)
        kw = dict(block_size=32, n_layer=2, n_head=4, attention_window=5, attention_sinks=2)
        if which == "gpt2":
            cfg, cls = GPT2Config(vocab_size=250, n_embd=32, **kw), GPT2
        else:
            cfg, cls = LLaMA3Config(vocab_size=256, n_kv_head=2, n_embd=64, ffn_dim=96, **kw), LLaMA3
        full, tp = cls(cfg), TPTransformer(cfg, comm)
        tp.load_full_state_dict(full.StateDict())
        idx = torch.randint(0, cfg.vocab_size, (2, 16), generator=torch.Generator().manual_seed(7))
        tgt = torch.roll(idx, -1, 1)
        _, bounded = full(idx, tgt)
        full.config.attention_window = 0
        _, unbounded = full(idx, tgt)
        q.put((rank, float(bounded), float(unbounded), float(tp(idx, tgt))))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("which,port", [("gpt2", 29761), ("llama3", 29762)])
def test_window_in_tensor_parallel_models(which, port):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ps = [ctx.Process(target=_worker, args=(r, 2, port, q, which)) for r in range(2)]
    for p in ps:
        p.start()
    try:
        results = [q.get(timeout=300) for _ in ps]
    finally:
        for p in ps:
            p.join(60)
            if p.is_alive():
                p.terminate()
    for _, bounded, unbounded, tp in results:
        # fp32 sums of some 300 terms in another order, of a loss of 5.5: 300 * 2^-24 * 5.5 = 1e-4; the window changes it by 3.5e-4
        assert abs(tp - bounded) < 1e-4 and abs(bounded - unbounded) > 2e-4, results
