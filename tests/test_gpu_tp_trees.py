"""Trees verified and accepted by tensor-parallel models, over f32 and q8_0 caches: every
rank makes the calls, each on its own GPU and with its own KV heads, and gets the whole
model's tokens.  world 1 is the same worker without shards."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

from plain_model import PlainModel

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPE = [512, 1024, 8, 4, 2, 2048, 1e-6, 1e6, 4096, 64, False]
TOKENS, PARENTS, CTX = [11, 500, 1200, 7, 9, 1999, 3], [-1, 0, 0, 1, 1, 2, -1], 70

WORKER = r"""
import importlib.util, json, os, sys
root, rank, world, tp_id, out = sys.argv[1], int(sys.argv[2]), int(sys.argv[3]), bytes.fromhex(sys.argv[4]), sys.argv[5]
shape, kv, p2p, tokens, parents, ctx = json.loads(sys.argv[6])
pkg = os.path.join(root, "llama.rs_b200")
spec = importlib.util.spec_from_file_location("llamars_b200", os.path.join(pkg, "__init__.py"),
                                              submodule_search_locations=[pkg])
lrs = importlib.util.module_from_spec(spec); sys.modules["llamars_b200"] = lrs; spec.loader.exec_module(lrs)
cfg = lrs.LlamaConfig(*shape)
sm = lrs.SynthModel(cfg, 11, lrs.LoadQuantization.Q4KM)
be = lrs.CudaBackend(rank)
m = lrs.CudaQwen2Model(be, sm.desc(), max_seq_len=256, max_sequences=2, kv_dtype=lrs.KvType[kv],
                       tp_rank=rank, tp_world=world, tp_id=tp_id, tp_p2p=p2p)
prompt = lrs.prompt_tokens(11, ctx, cfg.vocab_size)
m.prefill(prompt, want_logits=False)
res = {"argmax": m.verify_tree(tokens, parents, ctx).tolist()}
m.accept_tree([0, 2, 5], ctx)
logits, best = m.forward_token(42, ctx + 3)
res["logits"], res["best"] = logits.tolist(), int(best)
res["tokens"] = m.decode_greedy([best], [ctx + 4], 6)[:, 0].tolist()
json.dump(res, open(out, "w"))
"""


@pytest.mark.parametrize("kv", ["F32", "Q8_0"])
@pytest.mark.parametrize("world,allreduce", [(1, "nccl"), (2, "nccl"), (2, "p2p")])
def test_trees_of_tensor_parallel_models(lrs, orc, tmp_path, world, allreduce, kv):
    import torch
    if torch.cuda.device_count() < world:
        pytest.skip(f"needs {world} GPUs")
    tp_id = lrs.tp_unique_id().hex() if world > 1 else ""
    procs, outs = [], []
    for r in range(world):
        outs.append(str(tmp_path / f"rank{r}.json"))
        procs.append(subprocess.Popen([sys.executable, "-c", WORKER, ROOT, str(r), str(world), tp_id, outs[-1],
                                       json.dumps([SHAPE, kv, allreduce == "p2p", TOKENS, PARENTS, CTX])],
                                      env={**os.environ, "NCCL_NVLS_ENABLE": "0"}))
    try:
        codes = [p.wait(timeout=600) for p in procs]
    finally:
        for p in procs:
            if p.poll() is None:
                p.kill()
    assert codes == [0] * world
    res = [json.load(open(o)) for o in outs]
    assert all(r == res[0] for r in res)
    cfg = lrs.LlamaConfig(*SHAPE)
    sm = lrs.SynthModel(cfg, 11, lrs.LoadQuantization.Q4KM)
    plain = PlainModel(lrs, orc, sm, cfg)
    prompt = [int(t) for t in lrs.prompt_tokens(11, CTX, cfg.vocab_size)]

    def near(tokens):  # the logits, and how far off a cache of the type may be (test_plain_model)
        exact, held = (plain.logits(tokens, lrs.KvType[t])[-1] for t in ("F32", kv))
        return held, max(4e-4, np.abs(held - exact).max() / 3)
    paths = []
    for i, p in enumerate(PARENTS):
        paths.append((paths[p] if p >= 0 else []) + [TOKENS[i]])
        want, tol = near(prompt + paths[i])
        assert want.max() - want[res[0]["argmax"][i]] <= 2 * tol, i
    want, tol = near(prompt + [TOKENS[0], TOKENS[2], TOKENS[5], 42])
    assert np.abs(np.array(res[0]["logits"]) - want).max() < tol
    fed = prompt + [TOKENS[0], TOKENS[2], TOKENS[5], 42, res[0]["best"]]
    for t in res[0]["tokens"]:
        want, tol = near(fed)
        assert want.max() - want[t] <= 2 * tol
        fed.append(t)
