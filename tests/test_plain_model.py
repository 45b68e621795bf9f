"""The 64-bit model of the quantised cache's tests against the oracle, and how far its
logits move with a cache type and with the roundings of f32 steps."""
import copy

import numpy as np
import pytest

from plain_model import PlainModel
from test_x_split import split_b1, split_batched


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


def test_what_the_split_of_x_does_to_the_logits(lrs, orc):
    """The single-token dots see x in int8 pairs, off by up to 2^-16 of the largest of eight
    (test_x_split): each logit is off by a sum of hundreds of such roundings, rms 1.6e-5 and
    8e-5 at most over the 150,000 here.  4e-4, 25 times the rms, is the bar of f32 caches'
    logits in the tests of the models.  The batched dots' split is 300 times finer."""
    cfg = lrs.LlamaConfig(512, 1024, 8, 4, 2, 2048, 1e-6, 1e6, 4096, 64, False)
    plain = PlainModel(lrs, orc, lrs.SynthModel(cfg, 11, lrs.LoadQuantization.Q4KM), cfg)
    prompt = lrs.prompt_tokens(11, 74, cfg.vocab_size)
    exact, single, batched = (plain.logits(prompt, lrs.KvType.F32, split) for split in (None, split_b1, split_batched))
    assert 2e-5 < np.abs(single - exact).max() < 1e-4
    assert np.sqrt(((single - exact) ** 2).mean()) < 2e-5
    assert np.abs(batched - exact).max() < 1e-6
