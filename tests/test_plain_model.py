"""The 64-bit model of the quantised cache's tests against the oracle, and how far its
logits move with a cache type and with the roundings of f32 steps."""
import copy

import numpy as np
import pytest

from plain_model import PlainModel


def model(lrs, orc, hd):
    cfg = lrs.LlamaConfig(512, 1024, 512 // hd, 2 if hd == 128 else 4, 3, 2000, 1e-6, 1e6, 32768, hd, hd == 64)
    sm = lrs.SynthModel(cfg, 5, lrs.LoadQuantization.Q4KM)
    return cfg, sm, PlainModel(lrs, orc, sm, cfg)


@pytest.mark.parametrize("hd", [64, 128])
def test_plain_model_is_the_oracles(lrs, orc, hd):
    """Three layers of dots of at most 1,024 f32 terms: 7 * 3 + 1 products of 2^-24 * sqrt(1024)
    of their size, 4e-5 of logits below 2; the bar is 1e-4."""
    cfg, sm, plain = model(lrs, orc, hd)
    prompt = lrs.prompt_tokens(5, 90, cfg.vocab_size)
    ref = orc.OracleModel(sm.desc(), 128).benchmark_tokens(prompt, 2, keep_logits=True)
    assert np.abs(plain.logits(prompt, lrs.KvType.F32)[-1] - ref["logits"][0]).max() < 1e-4


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv", ["BF16", "Q8_0"])
def test_a_cache_type_moves_the_logits_more_than_roundings(lrs, orc, kv, hd):
    """What the GPU test of the models rests on: products that are off by 1e-5 of their size,
    which flips single codes, move the logits by less than a third of what the type does."""
    cfg, sm, plain = model(lrs, orc, hd)
    prompt = lrs.prompt_tokens(5, 150, cfg.vocab_size)
    exact, held = (plain.logits(prompt, lrs.KvType[t])[-1] for t in ("F32", kv))
    rng = np.random.default_rng(0)
    off = copy.copy(plain)
    off.layers = [{k: w * (1 + 1e-5 * rng.standard_normal(w.shape)) if w.ndim == 2 else w for k, w in layer.items()}
                  for layer in plain.layers]
    moved = np.abs(off.logits(prompt, lrs.KvType[kv])[-1] - held).max()
    assert 0 < 3 * moved < np.abs(held - exact).max()
