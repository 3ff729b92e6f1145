"""Greedy decoding with weights and caches of 4 bits in models without a router, whose choices a rounding cannot turn over.

A position's logits are off by 2 TOL of their rms in the median (tests/test_four_bits_models_gpu.py): a token that another one leads by 8 TOL in the oracle, four
times that, is not chosen."""
import numpy as np
import pytest

from oracle import bubotar_oracle as bo
from oracle import sonalorn_oracle as so
from tests import _bubotar as tb
from tests import _sonalorn as ts
from tests.test_four_bits_models_gpu import TOL, attention_heavy, make_engine, rng, rounded, rounded_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


def without_router():
    return ts.config(83, 128, [ts.layer("attention", ts.attention(4, 1, 64, 64, 0.2, (0.4, 50)), ts.dense(72)),
                               ts.layer("attention", ts.attention(16, 4, 128, 64, 0.1), ts.dense(200))], max_positions=500)


@pytest.mark.parametrize("t", [ts, tb])
def test_recorded_steps_of_the_scheduler(lm, t, monkeypatch):
    cfg = without_router() if t is ts else attention_heavy(tb)
    W = t.weights(cfg, 71)
    W["head"] = t.bf16_values(W["head"] * 2)
    mod = so if t is ts else bo
    monkeypatch.setattr(mod, "attention", rounded_cache(mod.attention))
    oracle = mod.Model(cfg, rounded(W))
    g = rng(72)
    e = make_engine(lm, t, cfg, W, weight_bits=4, cache_bits=4, portion=70, step_rows=80)
    prompts = [g.integers(0, cfg["vocab"], n).tolist() for n in (1, 33, 5, 18, 64, 150)]
    got = e.generate(prompts, 12)
    assert got == e.generate(prompts, 12)
    for x, y in zip(prompts, got):
        logits = oracle.forward(x + y[:-1], oracle.start())[len(x) - 1:]
        lead = logits.max(-1) - logits[np.arange(len(y)), y]
        assert (lead < 8 * TOL * np.sqrt((logits ** 2).mean())).all(), len(x)
    e.close()
