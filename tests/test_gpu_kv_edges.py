"""Edges of the paged cache's operators on a B200: units of one tile, values that
are not finite, what is reported where."""
import numpy as np
import pytest

import kv_plain
import kv_terms
from test_gpu_kv import DTYPES, Cache, Trees, dev, sync_ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,nodes", [(4, 3), (7, 4), (7, 9)])
def test_units_of_one_tile(lrs, backend, dtype, group, nodes):
    """Units whose only tile sets every row's maximum, several a CTA and softmax
    groups with and without rows: right, and the same bits each time."""
    import torch
    s = [(13 * i % 115, 1 + i % nodes) for i in range(150)]
    cache = Cache(lrs, dtype, 4, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, group)
    trees.run(backend)
    sync_ok(backend)
    first = trees.out.clone()
    trees.check()
    for _ in range(30):
        trees.out.fill_(-5.0)
        trees.run(backend)
        sync_ok(backend)
        assert torch.equal(first, trees.out)


# ------------------------------------------------- values that are not finite --
BITS = {"nan": {"F32": 0x7fc00000, "BF16": 0x7fc0, "Q8_0": 0x7e00}, "inf": {"F32": 0x7f800000, "BF16": 0x7f80, "Q8_0": 0x7c00},
        "-inf": {"F32": 0xff800000, "BF16": 0xff80, "Q8_0": 0xfc00}}


def poison(cache, dtype, which, slot, pos, head, col, what):
    """One value of the cache (of q8_0: the scale of its block) becomes NaN or infinite."""
    import torch
    hd, bits = cache.hd, BITS[what][dtype]
    tile = cache.pool[which][int(cache.pages[slot, pos // 64]), head]
    r, signed = pos % 64, bits - (1 << 32 if dtype == "F32" else 1 << 16) if bits >> (31 if dtype == "F32" else 15) else bits
    if dtype == "Q8_0":
        at = 64 * hd + 2 * (col // 32 * 64 + r if which else r * (hd // 32) + col // 32)
        tile[at:at + 2].view(torch.int16).fill_(signed)
    else:
        tile.view(torch.int16 if dtype == "BF16" else torch.int32)[r * hd + col] = signed


def check_rows(trees, bad, part=()):
    """Rows (tree, node, head) of `bad` hold no finite value, those of `part` some that are
    not; all others are within their bounds."""
    got = trees.out.cpu().numpy()[:trees.rows * trees.out_ld].reshape(trees.rows, trees.nh, -1)
    for t, (ctx, n) in enumerate(trees.sizes):
        k, v = (trees.cache.rows_of(trees.slots[t], ctx + n, i) for i in range(2))
        q = np.nan_to_num(trees.q(t), nan=0.0, posinf=0.0, neginf=0.0)
        want, err = kv_plain.attention(q, k, v, ctx, trees.masks[t], trees.scale)
        for i in range(n):
            for h in range(trees.nh):
                row = got[trees.start[t] + i, h]
                if (t, i, h) in bad:
                    assert not np.isfinite(row).any(), (t, i, h)
                elif (t, i, h) in part:
                    assert not np.isfinite(row).all(), (t, i, h)
                else:
                    assert (np.abs(row - want[i, h]) <= err[i, h]).all(), (t, i, h)


@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("ctx", [0, 70, 4000])  # a unit of one tile, a unit shared by CTAs
@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_that_are_not_finite(lrs, backend, dtype, ctx, what):
    s = [(ctx, 3), (5, 2)]
    cache = Cache(lrs, dtype, 2, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 3)
    node, head, value = 1, 4, {"nan": np.nan, "inf": np.inf, "-inf": -np.inf}[what]
    trees.qbuf[node * trees.q_ld + head * 128 + 17] = value
    trees.d["q"].copy_(dev(trees.qbuf))
    trees.run(backend)
    sync_ok(backend)
    check_rows(trees, {(0, node, head)})


@pytest.mark.parametrize("pos", [0, 129, 3967, 3968])  # the last is the one position of the last tile, a node
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dtype", DTYPES)
def test_cached_values_that_are_not_finite(lrs, backend, dtype, which, pos):
    """A NaN that a row attends to shows, wherever the split of a long context puts it."""
    s = [(3968, 1)]
    cache = Cache(lrs, dtype, 2, 128, [3969])
    trees = Trees(lrs, backend, cache, s, 3)
    poison(cache, dtype, which, 0, pos, 1, 40, "nan")
    trees.run(backend)
    sync_ok(backend)
    rows = {(0, 0, h) for h in (3, 4, 5)}
    check_rows(trees, rows if which == 0 else (), rows)


@pytest.mark.parametrize("ctx", [0, 100, 4000])
def test_scores_of_minus_infinity(lrs, backend, ctx):
    """bf16 K of -inf against a q whose three terms are positive: the weight is zero, and
    NaN is the result where no other score is left."""
    n = 3
    cache = Cache(lrs, "BF16", 1, 64, [ctx + n])
    trees = Trees(lrs, backend, cache, [(ctx, n)], 2, masks="chain")
    trees.qbuf[:] = 0.0
    trees.qbuf[0::64] = 1.0 + 2.0 ** -9 + 2.0 ** -18  # column 0 of every row, three terms of one sign
    trees.scale = float(np.float32(np.log(2.0)))
    assert np.float32(trees.scale) * np.float32(1.44269504088896) == 1.0
    trees.d["q"].copy_(dev(trees.qbuf))
    for p in range(ctx + n):
        if p != ctx + 1:  # node 1 keeps its score
            poison(cache, "BF16", 0, 0, p, 0, 0, "-inf")
    trees.run(backend)
    sync_ok(backend)
    got = trees.out.cpu().numpy()[:n * 128].reshape(n, 2, 64)
    assert np.isnan(got[0]).all()
    v = cache.rows_of(0, ctx + n, 1)[0, ctx + 1]
    # one weight over itself: three sums that may truncate (2^-23), an inverse and a product (2^-24)
    assert (np.abs(got[1:] - v) <= 2.0 ** -21 * np.abs(v)).all()


# ------------------------------------------------------- what is reported where --
@pytest.mark.parametrize("stream", ["legacy", "backend", "side"])
def test_skipped_entries_are_not_the_models(lrs, backend, stream):
    """A row that kv_store skips fails neither a matvec nor a model's call, which would
    withhold its result, and is still there for the next synchronize."""
    import torch
    cfg = lrs.LlamaConfig(512, 1024, 8, 4, 2, 2000, 1e-6, 1e6, 32768, 64, True)
    sm = lrs.SynthModel(cfg, 5, lrs.LoadQuantization.Q4KM)
    m = lrs.CudaQwen2Model(backend, sm.desc(), max_seq_len=256, max_sequences=2)
    prompt = lrs.prompt_tokens(5, 70, cfg.vocab_size)
    w = lrs.QuantTensor.quantize(np.ones(64 * 32, np.float32), 64, 32, lrs.QuantType.Q8_0)
    calls = [lambda: backend.matvec_batched(w, np.ones((1, 32), np.float32)).tolist(),
             lambda: m.prefill(prompt)[1], lambda: m.forward_token(3, 70)[1],
             lambda: m.decode_greedy([3], [70], 4).tolist(), lambda: m.verify_tree([3, 4], [-1, 0], 74).tolist(),
             lambda: m.accept_tree([0, 1], 74), lambda: m.forward_sample(3, 76, lrs.Sampler(), [1], 0.5)]
    want = [call() for call in calls]
    cache = Cache(lrs, "Q8_0", 2, 64, [70])
    d_seq, d_pos, dx = dev([9], np.int32), dev([3], np.int32), dev(np.ones((2, 64), np.float32))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def skip():
        at = {"legacy": 0, "backend": None, "side": side.cuda_stream}[stream]
        backend.kv_store(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), 1, dx.data_ptr(), dx.data_ptr(), stream=at)
        torch.cuda.synchronize()

    for call, expect in zip(calls, want):
        skip()
        assert call() == expect
        with pytest.raises(lrs.LrsError, match="out of range") as e:
            backend.synchronize()
        assert e.value.code == 1
        backend.synchronize()  # once


# ---------------------------------------------------------- products of terms --
@pytest.mark.parametrize("hd,at,group,room", [(64, 0, 1, 0), (64, 35, 1, 0), (128, 40, 1, 0), (128, 97, 1, 0),
                                              # rows and room that take units of 32 and of 64 rows
                                              (64, 35, 20, 600), (128, 40, 20, 600), (64, 0, 60, 300), (128, 97, 60, 300)])
@pytest.mark.parametrize("before", [0, 100, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_each_product_of_terms_counts(lrs, backend, dtype, before, hd, at, group, room):
    """Outputs that rest on one product each, to half of what losing it does.  What else
    moves them: the sums of products 2^20 times the result at most, with 2^-23 of the
    largest (an eighth of the result), and for the third term of P, 14 units of 2^-22
    where the exponents' and exponentials' roundings make 3.4."""
    import torch
    cases = kv_terms.cases(dtype, hd, at)
    for (part, a, b), case in cases.items():
        q, k, v = kv_terms.padded(case, before, (at + 10) % hd)
        n = len(k)
        cache = Cache(lrs, dtype, 1, hd, [n], extra=room)
        for which, rows in enumerate((k, v)):
            for p in range(n):
                cache.rows[which][cache.pages[0, p // 64], 0, p % 64] = rows[p]
            cache.value[which] = kv_plain.held(lrs, cache.dtype, cache.rows[which])
            cache.pool[which].copy_(dev(kv_plain.pack(lrs, cache.dtype, cache.rows[which], bool(which))))
        trees = Trees(lrs, backend, cache, [(n - 1, 1)], group, max_len=max(n, room * 64))
        trees.scale = kv_terms.SCALE
        trees.qbuf[:hd * group] = np.tile(q, group)
        trees.d["q"].copy_(dev(trees.qbuf))
        torch.cuda.synchronize()
        trees.run(backend)
        sync_ok(backend)
        got = trees.out.cpu().numpy()[:hd * group].reshape(group, hd)
        kk, vv = (cache.rows_of(0, n, i) for i in range(2))
        want, _ = kv_plain.attention(q.reshape(1, 1, hd), kk, vv, n - 1, [1], kv_terms.SCALE)
        lost = kv_terms.emulate(dtype, q, kk[0], vv[0], *(((a, b),) if i == part else () for i in (0, 1)))
        assert (np.abs(got - want.reshape(hd)) <= np.abs(lost - want.reshape(hd)) / 2).all(), (part, a, b)


# ------------------------------------------------------- the ends of the types --
@pytest.mark.parametrize("value", [3.4028234663852886e38, -3.4028234663852886e38, 3.3961775e38])
@pytest.mark.parametrize("ctx", [61, 2000])
@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_the_largest_values_in_masked_places(lrs, backend, dtype, ctx, value):
    """The type's largest K and V at a node reach only the rows that attend to it; K's
    with a query that is zero there is a score of zero."""
    n, bad = 8, 5
    cache = Cache(lrs, dtype, 2, 128, [ctx + n])
    trees = Trees(lrs, backend, cache, [(ctx, n)], 3, seed=4)
    for i in range(6, 8):
        trees.masks[0][i] = 1 << i | 1 << 2
    trees.d["mask"][:n].copy_(dev(np.array(trees.masks[0], np.uint64)))
    trees.qbuf[77::128] = 0.0
    trees.d["q"].copy_(dev(trees.qbuf))
    p = ctx + bad
    bf16_max = float(np.sign(value) * 3.3895313892515355e38)
    for which, col in ((0, 77), (1, 40)):
        at = cache.pages[0, p // 64], slice(None), p % 64, col
        cache.rows[which][at] = value if dtype == "F32" else bf16_max
        cache.value[which] = kv_plain.held(lrs, cache.dtype, cache.rows[which])
        outside = ~np.broadcast_to(cache.inside[:, None], cache.rows[which].shape[:3])
        t = kv_plain.pack(lrs, cache.dtype, cache.rows[which], bool(which))
        cache.pool[which].copy_(dev(np.where(cache.marks(outside, bool(which)), 0xff, t).astype(np.uint8)))
    trees.run(backend)
    sync_ok(backend)
    got = trees.out.cpu().numpy()[:n * trees.out_ld].reshape(n, 6, 128)
    k, v = (cache.rows_of(0, ctx + n, i) for i in range(2))
    seen = [i for i in range(n) if trees.masks[0][i] >> bad & 1]
    assert seen and len(seen) < n
    for rows, cols in ((sorted(set(range(n)) - set(seen)), range(128)), (seen, [c for c in range(128) if c != 40])):
        vv = v[..., list(cols)]
        want, err = kv_plain.attention(trees.q(0), k, vv, ctx, trees.masks[0], trees.scale)
        for i in rows:
            assert (np.abs(got[i][:, list(cols)] - want[i]) <= err[i]).all(), i


# --------------------------------------------------- calls that the header allows --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx", [0, 90, 1000])
def test_masks_of_any_nodes(lrs, backend, dtype, ctx):
    """A mask may name any nodes of the tree, later ones too, and leave out the node itself."""
    rng = np.random.default_rng(ctx)
    s = [(ctx, 64), (ctx // 2, 17)]
    cache = Cache(lrs, dtype, 1, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 5)
    trees.masks = [[int(m) & (1 << n) - 1 for m in rng.integers(0, 2 ** 64, n, dtype=np.uint64)] for _, n in s]
    trees.masks[0][3] = 1 << 63
    trees.d["mask"][:81].copy_(dev(np.array([m for t in trees.masks for m in t], np.uint64)))
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_trees_that_share_a_slot(lrs, backend, dtype):
    """Several trees on one slot, from different committed lengths, overlapping."""
    s = [(700, 3), (100, 5), (700, 3), (698, 5)]
    cache = Cache(lrs, dtype, 2, 128, [703])
    cache.pages = np.repeat(cache.pages, 4, axis=0)  # (the class gives each tree a slot)
    trees = Trees(lrs, backend, cache, s, 3)
    trees.d["seq"].fill_(0)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-30, -3.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(lrs, backend, dtype, scale):
    s = [(300, 4), (0, 3)]
    cache = Cache(lrs, dtype, 1, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 4)
    trees.scale = scale
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_widest_rows(lrs, backend, dtype):
    """64 nodes of 64 query heads a KV head: 64 units of 64 rows each."""
    s = [(130, 64), (1, 33)]
    cache = Cache(lrs, dtype, 1, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 64)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_calls_under_way(lrs, backend, dtype):
    """Calls of two host threads on streams of their own, a workspace each."""
    import threading

    import torch
    s = [(900, 9), (30, 4), (400, 20)]
    cache = Cache(lrs, dtype, 2, 64, [c + n for c, n in reversed(s)])
    both = [Trees(lrs, backend, cache, s, 7, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()

    def work(i):
        for _ in range(20):
            both[i].run(backend, stream=streams[i].cuda_stream)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    sync_ok(backend)
    for t in both:
        t.check()


def test_one_of_two_threads_reports_a_skipped_entry(lrs, backend):
    """Two threads that synchronize at once: an entry skipped before is reported by one."""
    import threading

    import torch
    cache = Cache(lrs, "F32", 1, 64, [64])
    d_seq, d_pos, dx = dev([9], np.int32), dev([3], np.int32), dev(np.ones(64, np.float32))
    torch.cuda.synchronize()
    for _ in range(300):
        backend.kv_store(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), 1, dx.data_ptr(), dx.data_ptr(), stream=0)
        torch.cuda.synchronize()
        codes, gate = [], threading.Barrier(2)

        def report():
            gate.wait()
            try:
                backend.synchronize()
            except lrs.LrsError as e:
                codes.append(e.code)
        threads = [threading.Thread(target=report) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert codes == [1]
