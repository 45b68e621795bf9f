"""Models over the paged cache's operators on a B200: what a call may depend on."""
import numpy as np
import pytest

from test_gpu_kv_model import _model, _near_best
from test_plain_model import model as plain_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
def test_a_prompt_does_not_depend_on_the_room(lrs, backend, hd):
    """The form of the attention goes by the positions in use, not by those that the slot
    has room for: the same bits at any max_seq_len, by prompt chunks and token by token."""
    prompt = lrs.prompt_tokens(5, 1088, 2000)  # whole chunks; the CTAs' parts differ between the forms
    got = []
    for room in (1152, 2048, 16384):
        _, _, m = _model(lrs, backend, "Q8_0", hd, seqs=1, max_seq=room)
        logits, _ = m.prefill(prompt)
        got.append([logits] + [m.forward_token(7 + i, 1088 + i)[0] for i in range(3)])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("kv", ["F32", "Q8_0"])
def test_only_paths_of_the_verified_tree_are_accepted(lrs, backend, kv):
    """A node past the tree, a node that its predecessor is not the parent of, another
    start or slot, a tree already accepted or written over: refused, nothing moved."""
    cfg, _, m = _model(lrs, backend, kv, 64)
    prompt = lrs.prompt_tokens(5, 9, cfg.vocab_size)
    tokens, parents = [5, 6, 7, 8, 9], [-1, 0, 0, 1, -1]

    def refused(nodes, start=9, seq=0):
        with pytest.raises(lrs.LrsError, match="tree") as e:
            m.accept_tree(nodes, start, seq=seq)
        assert e.value.code == 1

    m.prefill(prompt, want_logits=False)
    refused([0])  # nothing is verified yet
    want = m.verify_tree(tokens, parents, 9)
    for nodes in ([0, 5], [5], [63], [0, 3], [1], [1, 3], [0, 1, 2], [0, 0], [1, 0], [0, 4], [2 ** 32 - 1]):
        refused(nodes)
    for start, seq in ((8, 0), (10, 0), (9, 1)):
        refused([0], start, seq)
    m.accept_tree([], 9)
    m.accept_tree([0, 1, 3], 9)  # the refused calls have not touched it
    refused([0, 1])
    # the kept rows are those of the tokens one after another
    logits, _ = m.forward_token(11, 12)
    m.prefill(list(prompt) + [5, 6, 8], seq=1, want_logits=False)
    other, _ = m.forward_token(11, 12, seq=1)
    assert np.abs(logits - other).max() < 2e-2
    # whatever writes the slot's positions ends its tree; calls on other slots do not
    for call in (lambda: m.prefill([1, 2], 9), lambda: m.forward_token(3, 9), lambda: m.decode_greedy([3], [9], 2),
                 lambda: m.forward_sample(3, 9, lrs.Sampler(), [1], 0.5), lambda: m.reset(0),
                 lambda: m.profile_step([3], [9])):
        m.prefill(prompt, want_logits=False)
        m.verify_tree(tokens, parents, 9)
        call()
        refused([0])
    m.prefill(prompt, want_logits=False)
    assert np.array_equal(m.verify_tree(tokens, parents, 9), want)
    m.forward_token(3, 15, seq=1)
    m.verify_tree([4, 4], [-1, -1], 20, seq=1)
    m.accept_tree([4], 9)
    m.accept_tree([1], 20, seq=1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv", ["BF16", "Q8_0"])
def test_logits_are_the_cache_types(lrs, orc, backend, kv, hd):
    """Prompt chunks and single tokens over a cache type against a 64-bit model whose rows
    are held in it: within a third of what the type itself does to the logits, which the
    f32 cache's are off by."""
    cfg, sm, plain = plain_case(lrs, orc, hd)
    tokens = [int(t) for t in lrs.prompt_tokens(5, 150, cfg.vocab_size)]
    exact, held = (plain.logits(tokens, lrs.KvType[t]) for t in ("F32", kv))
    m = lrs.CudaQwen2Model(backend, sm.desc(), max_seq_len=512, max_sequences=2, kv_dtype=lrs.KvType[kv])
    for n in (64, 130, 150):
        got, _ = m.prefill(tokens[:n])
        effect = np.abs(held[n - 1] - exact[n - 1]).max()
        assert np.abs(got - held[n - 1]).max() < effect / 3 < np.abs(got - exact[n - 1]).max()
    for i, t in enumerate(tokens):
        got, _ = m.forward_token(t, i, seq=1)
        if i >= 20:  # (of few rows the effect is small)
            effect = np.abs(held[i] - exact[i]).max()
            assert np.abs(got - held[i]).max() < effect / 3, i


@pytest.mark.parametrize("kv", ["F32", "BF16", "Q8_0"])
def test_verified_nodes_are_the_64_bit_models(lrs, orc, backend, kv):
    """Each node's token is the best of the path to it, or as near as the logits may be off:
    for f32 1e-4 (test_plain_model), else a third of what the type does, on either side."""
    cfg, sm, plain = plain_case(lrs, orc, 64)
    rng = np.random.default_rng(8)
    m = lrs.CudaQwen2Model(backend, sm.desc(), max_seq_len=512, max_sequences=1, kv_dtype=lrs.KvType[kv])
    for ctx, n in ((3, 6), (120, 20), (200, 9)):
        prompt = [int(t) for t in lrs.prompt_tokens(5, ctx, cfg.vocab_size)]
        parents = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
        tokens = [int(t) for t in rng.integers(0, cfg.vocab_size, n)]
        m.prefill(prompt, want_logits=False)
        got = m.verify_tree(tokens, parents, ctx)
        paths = []
        for i, p in enumerate(parents):
            paths.append((paths[p] if p >= 0 else []) + [tokens[i]])
            exact, held = (plain.logits(prompt + paths[i], lrs.KvType[t])[-1] for t in ("F32", kv))
            tol = max(1e-4, np.abs(held - exact).max() / 3)
            assert held.max() - held[got[i]] <= 2 * tol, (ctx, i)


def test_a_persistent_step_continues_an_accepted_tree(lrs, backend):
    """Decoding in one kernel a step, before and after trees verified by several."""
    cfg, _, m = _model(lrs, backend, "F32", 64, persistent_decode=True)
    _, _, plain = _model(lrs, backend, "F32", 64)
    prompt = lrs.prompt_tokens(5, 60, cfg.vocab_size)
    got = []
    for x in (m, plain):
        x.prefill(prompt, want_logits=False)
        a = x.decode_greedy([7], [60], 4)[:, 0]
        tree = [int(a[-1]), 5, 9, 5]
        x.verify_tree(tree, [-1, 0, 0, 2], 64)
        x.accept_tree([0, 2, 3], 64)
        logits, _ = x.forward_token(11, 67)
        got.append((a, logits, x.decode_greedy([12], [68], 4)[:, 0]))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][2], got[1][2])
    assert np.abs(got[0][1] - got[1][1]).max() < 4e-4


@pytest.mark.parametrize("kv", ["F32", "Q8_0"])
def test_the_last_positions_of_a_slot(lrs, orc, backend, kv):
    """A full tree that ends at the context's end; a chunk of one token behind one of 64."""
    cfg, sm, plain = plain_case(lrs, orc, 64)
    m = lrs.CudaQwen2Model(backend, sm.desc(), max_seq_len=129, max_sequences=1, kv_dtype=lrs.KvType[kv])
    tokens = [int(t) for t in lrs.prompt_tokens(5, 129, cfg.vocab_size)]

    def tol(n):
        exact, held = (plain.logits(tokens[:n], lrs.KvType[t]) for t in ("F32", kv))
        return held, max(4e-4, np.abs(held[-1] - exact[-1]).max() / 3)
    held, bar = tol(129)
    for n in (65, 129):
        assert np.abs(m.prefill(tokens[:n])[0] - held[n - 1]).max() < bar
    m.prefill(tokens[:65], want_logits=False)
    got = m.verify_tree(tokens[65:], list(range(-1, 63)), 65)
    for i in range(64):
        assert held[65 + i].max() - held[65 + i][got[i]] <= 2 * bar
    m.accept_tree(list(range(64)), 65)
    with pytest.raises(lrs.LrsError, match="exceeds"):
        m.verify_tree([1, 2], [-1, 0], 128)


def test_a_batch_of_more_sequences_than_a_chunk(lrs, backend):
    """q8_0 decode steps of 70 sequences of ragged lengths, each as it decodes alone."""
    cfg, _, m = _model(lrs, backend, "Q8_0", 64, seqs=70, max_seq=256)
    lens = [3 + 2 * i for i in range(70)]
    first = []
    for i, n in enumerate(lens):
        first.append(int(m.prefill(lrs.prompt_tokens(40 + i, n, cfg.vocab_size), seq=i)[1]))
    got = m.decode_greedy(first, lens, 6)
    for i in (0, 1, 33, 63, 64, 69):
        logits, _ = m.forward_token(first[i], lens[i], seq=i)
        assert _near_best(logits, int(got[0, i]), 1e-3)


def test_refused_calls_leave_the_verified_tree(lrs, backend):
    """A batch that is refused for another item has written nothing."""
    cfg, _, m = _model(lrs, backend, "F32", 64)
    m.prefill(lrs.prompt_tokens(5, 9, cfg.vocab_size), want_logits=False)
    m.verify_tree([5, 6], [-1, 0], 9)
    for call in (lambda: m.decode_greedy([3, 3], [9, 9], 2, [0, 99]), lambda: m.decode_greedy([3, 3], [9, 600], 2, [0, 1]),
                 lambda: m.decode_greedy([3, 3], [9, 9], 2, [0, 0]), lambda: m.profile_step([3, 3], [9, 9], [0, 99]),
                 lambda: m.prefill([cfg.vocab_size], 9), lambda: m.verify_tree([5], [0], 9)):
        with pytest.raises(lrs.LrsError):
            call()
    m.accept_tree([0, 1], 9)
