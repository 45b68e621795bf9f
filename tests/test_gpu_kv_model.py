"""The models over the paged cache's operators on a B200: decoding with a q8_0
KV cache, and drafted trees verified and accepted with every cache type."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LOGIT_TOL = 2e-2  # the bar of the f32 cache's logits against the oracle


def _model(lrs, backend, kv, hd=64, seqs=3, seed=5, max_seq=512, **kw):
    cfg = lrs.LlamaConfig(512, 1024, 512 // hd, 2 if hd == 128 else 4, 3, 2000, 1e-6, 1e6, 32768, hd, hd == 64)
    sm = lrs.SynthModel(cfg, seed, lrs.LoadQuantization.Q4KM)
    return cfg, sm, lrs.CudaQwen2Model(backend, sm.desc(), max_seq_len=max_seq, max_sequences=seqs,
                                       kv_dtype=lrs.KvType[kv], **kw)


def _near_best(logits, token, tol):
    """The token is the argmax, or within what two runs of the arithmetic may differ by."""
    return float(logits.max() - logits[token]) <= tol


@pytest.mark.parametrize("hd", [64, 128])
def test_q8_0_cache_follows_the_f32_cache(lrs, backend, hd):
    """Prompt logits and greedy tokens of a q8_0 cache against the f32 cache's.
    A q8_0 value is off by at most amax / 254 of its block, rms 0.6% of the
    values' deviation, five times bf16's 0.11%; bf16's bar is 5e-2."""
    cfg, _, f32 = _model(lrs, backend, "F32", hd)
    _, _, q8 = _model(lrs, backend, "Q8_0", hd)
    prompt = lrs.prompt_tokens(5, 150, cfg.vocab_size)
    (la, aa), (lb, ab) = f32.prefill(prompt), q8.prefill(prompt)
    off = float(np.abs(la - lb).max())
    print(f"q8_0 prompt logits off by {off:.2e}")
    assert 0.0 < off < 0.25
    assert _near_best(la, ab, 2 * off)
    tokens = f32.decode_greedy([aa], [150], 40)[:, 0]
    feed, fed = int(aa), []
    for i in range(40):  # teacher-forced: the f32 cache's tokens
        lg, am = q8.forward_token(feed, 150 + i)
        fed.append(am)
        want, _ = f32.forward_token(feed, 150 + i)
        off = float(np.abs(want - lg).max())
        assert off < 0.25 and _near_best(want, am, 2 * off)
        feed = int(tokens[i])


def test_q8_0_steps_agree(lrs, backend):
    """Prompt chunks, single tokens, captured and plain steps, a batch of
    sequences: one cache content, so the tokens agree (to near-ties)."""
    cfg, sm, a = _model(lrs, backend, "Q8_0", 128)
    b = lrs.CudaQwen2Model(backend, sm.desc(), max_seq_len=512, max_sequences=3, kv_dtype=lrs.KvType.Q8_0,
                           use_graph=False)
    prompts = [lrs.prompt_tokens(5, n, cfg.vocab_size, i) for i, n in enumerate((70, 64, 3))]
    firsts = []
    for s, p in enumerate(prompts):
        la, fa = a.prefill(p, seq=s)
        for i, t in enumerate(p[:-1]):
            assert b.forward_token(int(t), i, lrs.LogitsMode.SKIP, seq=s) is None
        lb, fb = b.forward_token(int(p[-1]), len(p) - 1, seq=s)
        # the batched and the single-token products differ by their roundings, which
        # move single codes of the cache: one step of a block in a few rows
        assert np.abs(la - lb).max() < LOGIT_TOL
        assert _near_best(la, fb, LOGIT_TOL)
        firsts.append(fa)
    lens = [len(p) for p in prompts]
    whole = a.decode_greedy(firsts, lens, 30)
    assert a.step_kernels() > 0
    again = a.decode_greedy(firsts, lens, 30)  # the same positions once more: the graph replayed
    assert np.array_equal(whole, again)
    plain = lrs.CudaQwen2Model(backend, sm.desc(), max_seq_len=512, max_sequences=3, kv_dtype=lrs.KvType.Q8_0,
                               use_graph=False)
    for s, p in enumerate(prompts):
        plain.prefill(p, seq=s, want_logits=False)
    assert np.array_equal(plain.decode_greedy(firsts, lens, 30), whole)


def test_q8_0_model_options(lrs, backend):
    """The persistent step does not read q8_0 caches: the option changes nothing."""
    cfg, sm, a = _model(lrs, backend, "Q8_0", 64)
    _, _, b = _model(lrs, backend, "Q8_0", 64, persistent_decode=True)
    prompt = lrs.prompt_tokens(5, 20, cfg.vocab_size)
    for m in (a, b):
        m.prefill(prompt, want_logits=False)
    assert np.array_equal(a.decode_greedy([7], [20], 10), b.decode_greedy([7], [20], 10))
    # and its measurement hook counts the attention
    *_, attn = a.profile_step([7], [30])
    assert attn > 0.0


def _paths(parents):
    paths = []
    for i, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else []) + [i])
    return paths


@pytest.mark.parametrize("kv", ["F32", "BF16", "Q8_0"])
@pytest.mark.parametrize("hd", [64, 128])
def test_verify_tree(lrs, backend, kv, hd):
    """Each node's greedy token is the one that the path to it gives token by token."""
    cfg, _, m = _model(lrs, backend, kv, hd)
    rng = np.random.default_rng(3)
    for ctx, n in ((0, 5), (63, 9), (130, 17)):
        prompt = lrs.prompt_tokens(5, max(ctx, 1), cfg.vocab_size)[:ctx]
        parents = [-1] + [int(rng.integers(-1 if i == 3 else 0, i)) for i in range(1, n)]
        tokens = [int(t) for t in rng.integers(0, cfg.vocab_size, n)]
        if ctx:
            m.prefill(prompt, seq=0, want_logits=False)
        got = m.verify_tree(tokens, parents, ctx, seq=0)
        for i, path in enumerate(_paths(parents)):
            m.reset(1)
            logits, _ = m.prefill(list(prompt) + [tokens[j] for j in path], seq=1)
            # (q8_0: as in test_q8_0_steps_agree)
            assert _near_best(logits, int(got[i]), LOGIT_TOL), (ctx, i)
        again = m.verify_tree(tokens, parents, ctx, seq=0)
        assert np.array_equal(got, again)


@pytest.mark.parametrize("kv", ["F32", "BF16", "Q8_0"])
def test_speculative_greedy_decode(lrs, backend, kv):
    """Drafts that are partly right, verified and accepted round after round, give
    greedy decoding's tokens (to near-ties), on a slot beside another one's."""
    cfg, _, m = _model(lrs, backend, kv, 64)
    rng = np.random.default_rng(11)
    prompt = lrs.prompt_tokens(9, 60, cfg.vocab_size)
    m.prefill(prompt, seq=2, want_logits=False)
    _, first = m.prefill(prompt, seq=0)
    greedy = [int(first)] + [int(t) for t in m.decode_greedy([first], [60], 50, seqs=[2])[:, 0]]
    pos, out, nxt, rounds = 60, [], int(first), 0
    while len(out) < 40:
        # a chain of the true continuation that goes wrong somewhere, and side branches
        tokens, parents, at = [nxt], [-1], 0
        for k in range(int(rng.integers(0, 6))):
            right = greedy[len(out) + k + 1]
            tokens += [int(rng.integers(0, cfg.vocab_size)), right if rng.random() < 0.8 else 3]
            parents += [at, at]
            at = len(tokens) - 1
        argmax = m.verify_tree(tokens, parents, pos, seq=0)
        path, nxt = lrs.greedy_path(tokens, parents, argmax)
        m.accept_tree(path, pos, seq=0)
        out += [tokens[j] for j in path]
        pos += len(path)
        rounds += 1
    assert rounds < len(out)  # drafts were accepted
    diff = [i for i, (a, b) in enumerate(zip(out, greedy)) if a != b]
    if diff:  # only where the two arithmetics may choose differently
        i = diff[0]
        logits, _ = m.prefill(list(prompt) + greedy[:i], seq=1)
        assert _near_best(logits, out[i], LOGIT_TOL) and _near_best(logits, greedy[i], LOGIT_TOL)
    # what was kept serves plain decoding as well
    tail = m.decode_greedy([nxt], [pos], 5, seqs=[0])[:, 0]
    m.reset(1)
    logits, _ = m.prefill(list(prompt) + out + [nxt], seq=1)
    assert _near_best(logits, int(tail[0]), LOGIT_TOL)


def test_bad_trees_are_refused(lrs, backend):
    cfg, _, m = _model(lrs, backend, "F32", 64, max_seq=128)
    m.prefill([1, 2, 3], want_logits=False)
    v = cfg.vocab_size
    for call, code in ((lambda: m.verify_tree([1], [0], 3), 1), (lambda: m.verify_tree([], [], 3), 1),
                       (lambda: m.verify_tree([v], [-1], 3), 1), (lambda: m.verify_tree([1], [-1], 3, seq=9), 1),
                       (lambda: m.verify_tree([1, 2], [-1, 0], 127), 1), (lambda: m.verify_tree([1] * 65, [-1] * 65, 3), 1),
                       (lambda: m.accept_tree([1, 1], 3), 1), (lambda: m.accept_tree([64], 3), 1),
                       (lambda: m.accept_tree([0], 3, seq=7), 1), (lambda: m.accept_tree([0, 63], 3), 1),
                       (lambda: m.accept_tree([0], 64), 1)):
        with pytest.raises(lrs.LrsError) as e:
            call()
        assert e.value.code == code
    m.accept_tree([], 3)
    m.verify_tree([5, 6], [-1, 0], 126)  # the last positions
