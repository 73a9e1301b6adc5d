"""The example of continuous batching against the resident model: requests of unequal length that enter, wait, share pages and
leave get the logits and tokens that each gets alone from a cache of its own."""
import importlib.util
import os
import sys

import numpy as np
import pytest
import torch

from ferrum_gpu_b200 import CudaLlama, QKind, _ffi
from ferrum_gpu_b200.hostmodel import LlamaConfig, random_llama, random_tokens

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
    m = sys.modules["paged_serving"] = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _cfg(neox=True, heads=4, kv=2, hd=64):
    return LlamaConfig(vocab=301, ctx=160, dim=128, heads=heads, kv_heads=kv, head_dim=hd, layers=3, hidden=256, rope_dim=hd,
                       rope_type=_ffi.FC_ROPE_NEOX if neox else _ffi.FC_ROPE_NORM)


@pytest.mark.parametrize("neox,heads,kv,hd,page", [(True, 4, 2, 64, 16), (False, 8, 1, 32, 8), (True, 2, 2, 128, 64)])
def test_steps_give_the_resident_models_logits(dev, example, neox, heads, kv, hd, page):
    cfg = _cfg(neox, heads, kv, hd)
    host = random_llama(cfg, seed=5, std=0.1, gain_jitter=0.1)
    paged = example.PagedLlama(dev, host, QKind.Q8_0, pages=6 * -(-cfg.ctx // page), page=page, requests=5, max_len=cfg.ctx)
    alone = CudaLlama(dev, host, QKind.Q8_0, max_streams=3)
    texts = [random_tokens(i, n, cfg.vocab).tolist() for i, n in enumerate((1, 37, 100))]
    places = [4, 0, 2]
    want = [alone.prefill(np.array(t, dtype=np.int32), stream=i) for i, t in enumerate(texts)]
    logits, out, step = paged.step(places, texts, top=4)
    for turn in range(4):
        dev.sync()
        assert int(step.status) == 0
        got = logits.cpu().numpy()
        for i in range(3):
            # two f32 paths of the same weights that sum in other orders: the bound that this repository holds its models to
            assert np.abs(got[i] - want[i]).max() < 2e-5 * max(1.0, np.abs(want[i]).max()), (turn, i)
            x = want[i].astype(np.float64)
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            assert np.abs(out.top_logprob[i].cpu().numpy() - lp[out.top_index[i].cpu().numpy()]).max() < 1e-4
        picks = [int(w.argmax()) for w in want]
        want = [alone.feed(t, stream=i) for i, t in enumerate(picks)]
        logits, out, step = paged.step(places, [[t] for t in picks], top=4)


def test_requests_that_wait_share_and_leave(dev, example):
    cfg = _cfg()
    host = random_llama(cfg, seed=6, std=0.15)
    paged = example.PagedLlama(dev, host, QKind.Q4_0, pages=14, page=16, requests=3, max_len=cfg.ctx)
    rng = np.random.default_rng(3)
    requests = [example.Request(random_tokens(20 + i, int(rng.integers(1, 90)), cfg.vocab).tolist(), int(rng.integers(1, 30))) for i in range(9)]
    example.serve(paged, requests)
    assert int(paged.cache.n_free) == 14 and sorted(paged.cache.free.tolist()) == list(range(14))
    alone = CudaLlama(dev, host, QKind.Q4_0, max_streams=1)
    for r in requests:
        alone.reset(0)
        x = alone.prefill(np.array(r.prompt, dtype=np.int32))
        for i, t in enumerate(r.tokens):
            best = np.sort(x)[::-1]
            if best[0] - best[1] > 1e-4 * max(1.0, np.abs(x).max()):  # (closer ones are decided by rounding)
                assert t == int(x.argmax())
            if i + 1 < len(r.tokens):
                x = alone.feed(t)
        assert len(r.tokens) == r.want == len(r.notes)


def test_the_example_runs(example, capsys):
    example.main()
    assert "pages free again" in capsys.readouterr().out
