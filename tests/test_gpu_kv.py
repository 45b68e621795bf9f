"""The paged KV cache's operators on a B200 against their plain forms: writing
and reading back in every type, attention of token trees, accepting a path."""
import numpy as np
import pytest

import kv_plain
from kv_plain import PAGE

pytestmark = pytest.mark.gpu

DTYPES = ["F32", "BF16", "Q8_0"]
LEGACY = 0  # the default stream, which torch's work here runs on


def dev(x, dtype=None):
    import torch
    x = np.ascontiguousarray(x if dtype is None else np.asarray(x).astype(dtype))
    return torch.from_numpy(x.view(np.int64) if x.dtype == np.uint64 else x).cuda()


class Cache:
    """A cache of random rows on the device and its values in 64 bits.  What lies
    outside the slots' first `lens` positions is bytes 0xff: NaN values and
    scales."""

    def __init__(self, lrs, dtype, heads, hd, lens, seed=1, spare=3, scale=1.0, extra=0):
        import torch
        rng = np.random.default_rng(seed)
        self.dtype, self.heads, self.hd = lrs.KvType[dtype], heads, hd
        lens = list(lens)
        width = max(-(-max(n, 1) // PAGE) for n in lens) + extra
        n_pages = len(lens) * width + spare
        self.pages = rng.permutation(n_pages)[:len(lens) * width].reshape(len(lens), width).astype(np.int32)
        k, v = (rng.standard_normal((2, n_pages, heads, PAGE, hd)) * scale).astype(np.float32)
        k[..., hd // 3] += 5.0
        self.rows = [k, v]
        tiles = [kv_plain.pack(lrs, self.dtype, x, bool(i)) for i, x in enumerate(self.rows)]
        inside = np.zeros((n_pages, PAGE), bool)
        for s, n in enumerate(lens):
            for p in range(n):
                inside[self.pages[s, p // PAGE], p % PAGE] = True
        outside = ~np.broadcast_to(inside[:, None], (n_pages, heads, PAGE))
        self.tiles = [np.where(self.marks(outside, bool(i)), 0xff, t).astype(np.uint8) for i, t in enumerate(tiles)]
        self.inside, self.lens = inside, lens
        self.pool = [torch.from_numpy(t).cuda() for t in self.tiles]
        self.d_pages = dev(self.pages)
        self.c = lrs.KvCache(self.pool[0].data_ptr(), self.pool[1].data_ptr(), self.d_pages.data_ptr(),
                             n_pages, len(lens), width, heads, hd, int(self.dtype))
        self.value = [kv_plain.held(lrs, self.dtype, x) for x in self.rows]

    def marks(self, rows, is_v):
        """[pages, heads, bytes]: the bytes of a tile that belong to marked rows."""
        p, h, _ = rows.shape
        if self.dtype != 2:
            return np.repeat(rows, self.hd * (4 if self.dtype == 0 else 2), axis=2)
        hd = self.hd
        per = np.broadcast_to(rows[:, :, :, None], (p, h, PAGE, hd))
        sc = np.broadcast_to(rows[:, :, :, None], (p, h, PAGE, hd // 32))
        if is_v:
            codes, sc = per.reshape(p, h, PAGE // 4, 4, hd).transpose(0, 1, 2, 4, 3), sc.transpose(0, 1, 3, 2)
        else:
            codes = per.reshape(p, h, PAGE, hd // 16, 16).transpose(0, 1, 3, 2, 4)
        return np.concatenate([codes.reshape(p, h, -1), np.repeat(sc.reshape(p, h, -1), 2, axis=2)], axis=2)

    def rows_of(self, slot, n, which):
        """Values [heads, n, hd] of a slot's first n positions."""
        x = self.value[which][self.pages[slot]]  # [width, heads, 64, hd]
        return x.transpose(1, 0, 2, 3).reshape(self.heads, -1, self.hd)[:, :n]

    def bytes_now(self):
        import torch
        torch.cuda.synchronize()
        return [p.cpu().numpy() for p in self.pool]


def sync_ok(backend):
    import torch
    torch.cuda.synchronize()
    backend.synchronize()


# ------------------------------------------------------------ write and read --
def rows_case(rng, n, slots, width, kind):
    """(seq, pos) of n distinct positions."""
    if kind == "run":  # one slot after another, from an odd position
        per = -(-n // slots)
        seq = np.repeat(np.arange(slots), per)[:n]
        return seq, (np.arange(n) % per) + min(5, width * PAGE - per)
    cells = rng.permutation(slots * width * PAGE)[:n]
    if kind == "step":  # one row a slot
        return np.arange(n) % slots, np.full(n, 37) + np.arange(n) // slots
    return cells // (width * PAGE), cells % (width * PAGE)


@pytest.mark.parametrize("hd,heads", [(64, 2), (128, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,slots,width,kind", [(1, 1, 1, "run"), (3, 1, 2, "run"), (64, 64, 2, "step"), (130, 2, 2, "run"),
                                                (191, 3, 1, "mixed"), (4000, 4, 17, "run"), (2500, 2, 20, "mixed")])
def test_store_then_load(lrs, backend, dtype, hd, heads, n, slots, width, kind):
    """The stored bytes are the host encoders', nothing else changes, and the
    rows read back are the held values, bit for bit."""
    import torch
    rng = np.random.default_rng(n)
    cache = Cache(lrs, dtype, heads, hd, [0] * slots, extra=width - 1)
    seq, pos = rows_case(rng, n, slots, width, kind)
    k, v = (rng.standard_normal((2, n, heads, hd)) * 3).astype(np.float32)
    k[0, 0, :32] = 0.0                                   # a block of zeros
    v[-1, -1, 32:64] = 1e-30                             # scale 0 in f16
    v[0, 0, 0] = 30000.0
    d_seq, d_pos, dk, dv = dev(seq, np.int32), dev(pos, np.int32), dev(k), dev(v)
    backend.kv_store(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), n, dk.data_ptr(), dv.data_ptr(), stream=LEGACY)
    out = [torch.full((n, heads, hd), 7.0, device="cuda") for _ in range(2)]
    backend.kv_load(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr(), stream=LEGACY)
    sync_ok(backend)
    page = cache.pages[seq, pos // PAGE]
    for i, x in enumerate((k, v)):
        full = np.zeros(cache.rows[0].shape, np.float32)
        full[page, :, pos % PAGE] = x
        written = np.zeros(full.shape[:3], bool)
        written[page, :, pos % PAGE] = True
        want = np.where(cache.marks(written, bool(i)), kv_plain.pack(lrs, cache.dtype, full, bool(i)), cache.tiles[i])
        assert np.array_equal(cache.bytes_now()[i], want)
        assert np.array_equal(out[i].cpu().numpy(), kv_plain.held(lrs, cache.dtype, x).astype(np.float32))


def test_store_rounds_ties_as_the_host_encoder(lrs, backend):
    """Products that are exact ties, of either sign, and their neighbours."""
    rng = np.random.default_rng(2)
    n, heads, hd = 40, 2, 64
    x = (rng.integers(-126, 127, (2, n, heads, hd)) + rng.choice([0.5, -0.5, 0.0, 0.49999997], (2, n, heads, hd)))
    x = np.clip(x, -127, 127)
    x[..., ::32] = 127.0                                 # d = 1
    x *= 2.0 ** rng.integers(-90, 8, (2, n, 1, 1))       # exact powers of two keep the ties
    x = x.astype(np.float32)
    cache = Cache(lrs, "Q8_0", heads, hd, [0])
    d_seq, d_pos, dk, dv = dev(np.zeros(n, np.int32)), dev(np.arange(n) + 3, np.int32), dev(x[0]), dev(x[1])
    backend.kv_store(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), n, dk.data_ptr(), dv.data_ptr(), stream=LEGACY)
    sync_ok(backend)
    pos = np.arange(n) + 3
    for i in range(2):
        full = np.zeros(cache.rows[0].shape, np.float32)
        full[cache.pages[0, 0], :, pos] = x[i]
        written = np.zeros(full.shape[:3], bool)
        written[cache.pages[0, 0], :, pos] = True
        want = np.where(cache.marks(written, bool(i)), kv_plain.pack(lrs, cache.dtype, full, bool(i)), cache.tiles[i])
        assert np.array_equal(cache.bytes_now()[i], want)


def test_store_clamps_what_q8_0_cannot_hold(lrs, backend):
    import torch
    cache = Cache(lrs, "Q8_0", 1, 64, [0])
    x = np.zeros((2, 1, 64), np.float32)
    x[0, 0, :6] = [np.inf, -np.inf, np.nan, 1e30, -7e4, 512.0]
    x[1, 0, 40:43] = [np.nan, 2.0, -1.0]
    d_seq, d_pos, dx = dev([0, 0], np.int32), dev([3, 4], np.int32), dev(x)
    backend.kv_store(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), 2, dx.data_ptr(), dx.data_ptr(), stream=LEGACY)
    out = torch.zeros(2, 2, 64, device="cuda")
    backend.kv_load(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), 2, out[0].data_ptr(), out[1].data_ptr(), stream=LEGACY)
    sync_ok(backend)
    got = out.cpu().numpy()
    want = kv_plain.held(lrs, cache.dtype, x).reshape(2, 64).astype(np.float32)
    assert np.isfinite(got).all() and want[0, 0] == 65024.0 and want[0, 1] == -65024.0 and want[0, 2] == 0.0
    assert np.array_equal(got[0], want) and np.array_equal(got[1], want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift,ld", [(1, 261), (0, 260), (3, 0), (2, 1024)])
def test_store_and_load_strides(lrs, backend, dtype, shift, ld):
    """Rows at any float address and stride; what lies between them stays."""
    import torch
    heads, hd, n = 2, 128, 9
    rng = np.random.default_rng(ld)
    step = ld or heads * hd
    cache = Cache(lrs, dtype, heads, hd, [0, 0])
    buf = rng.standard_normal((2, n * step + 8)).astype(np.float32)
    seq, pos = np.arange(n) % 2, np.arange(n) // 2 + 11
    d_seq, d_pos, db = dev(seq, np.int32), dev(pos, np.int32), dev(buf)
    at = [db[i].data_ptr() + 4 * shift for i in range(2)]
    backend.kv_store(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), n, at[0], at[1], ld=ld, stream=LEGACY)
    out = torch.full((2, n * step + 8), -3.0, device="cuda")
    to = [out[i].data_ptr() + 4 * shift for i in range(2)]
    backend.kv_load(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), n, to[0], to[1], ld=ld, stream=LEGACY)
    sync_ok(backend)
    got = out.cpu().numpy()
    for i in range(2):
        want = np.full(n * step + 8, -3.0, np.float32)
        for r in range(n):
            row = slice(shift + r * step, shift + r * step + heads * hd)
            want[row] = kv_plain.held(lrs, cache.dtype, buf[i, row].reshape(heads, hd)).ravel()
        assert np.array_equal(got[i], want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_out_of_range_are_skipped(lrs, backend, dtype):
    """Bad slots, positions and pages touch nothing and are reported once."""
    import torch
    cache = Cache(lrs, dtype, 2, 64, [70, 70])
    table = cache.pages.copy()
    table[1, 1] = cache.c.n_pages  # slot 1 has no second page
    cache.d_pages.copy_(dev(table))
    seq = np.array([0, 5, -1, 0, 0, 1, 1], np.int32)
    pos = np.array([7, 3, 3, 128, -2, 66, 9], np.int32)
    ok = np.array([1, 0, 0, 0, 0, 0, 1], bool)
    rng = np.random.default_rng(0)
    x = rng.standard_normal((7, 2, 64)).astype(np.float32)
    d_seq, d_pos, dx = dev(seq), dev(pos), dev(x)
    backend.kv_store(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), 7, dx.data_ptr(), dx.data_ptr(), stream=LEGACY)
    torch.cuda.synchronize()
    with pytest.raises(lrs.LrsError, match="out of range") as e:
        backend.synchronize()
    assert e.value.code == 1
    backend.synchronize()  # reported once
    out = torch.full((2, 7, 2, 64), 9.0, device="cuda")
    backend.kv_load(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), 7, out[0].data_ptr(), out[1].data_ptr(), stream=LEGACY)
    torch.cuda.synchronize()
    with pytest.raises(lrs.LrsError, match="out of range"):
        backend.synchronize()
    want = np.where(ok[:, None, None], kv_plain.held(lrs, cache.dtype, x), 9.0).astype(np.float32)
    for i in range(2):
        assert np.array_equal(out[i].cpu().numpy(), want)
        full = np.zeros(cache.rows[0].shape, np.float32)
        written = np.zeros(full.shape[:3], bool)
        for r in np.nonzero(ok)[0]:
            full[cache.pages[seq[r], 0], :, pos[r]] = x[r]
            written[cache.pages[seq[r], 0], :, pos[r]] = True
        want_b = np.where(cache.marks(written, bool(i)), kv_plain.pack(lrs, cache.dtype, full, bool(i)), cache.tiles[i])
        assert np.array_equal(cache.bytes_now()[i], want_b)


def test_load_one_of_the_two(lrs, backend):
    import torch
    cache = Cache(lrs, "Q8_0", 2, 128, [50])
    d_seq, d_pos = dev(np.zeros(50, np.int32)), dev(np.arange(50), np.int32)
    out = torch.zeros(50, 2, 128, device="cuda")
    for i in range(2):
        at = [out.data_ptr() if j == i else None for j in range(2)]
        backend.kv_load(cache.c, d_seq.data_ptr(), d_pos.data_ptr(), 50, *at, stream=LEGACY)
        sync_ok(backend)
        assert np.array_equal(out.cpu().numpy(), cache.rows_of(0, 50, i).transpose(1, 0, 2).astype(np.float32))


# -------------------------------------------------------------- attention ----
class Trees:
    """Trees of the given (committed, nodes) over a cache's slots in reverse order."""

    def __init__(self, lrs, backend, cache, sizes, group, seed=2, masks="tree", max_nodes=None, max_len=None,
                 spare_rows=2, q_ld=0, out_ld=0, shift=0):
        import torch
        rng = np.random.default_rng(seed)
        self.cache, self.sizes, self.group = cache, sizes, group
        self.slots = np.arange(len(sizes))[::-1].copy()
        self.nh = cache.heads * group
        n = sum(s[1] for s in sizes)
        self.n, self.rows = n, n + spare_rows
        self.masks = [kv_plain.random_tree(rng, t) if masks != "chain" else [(2 << i) - 1 for i in range(t)]
                      for _, t in sizes]
        width = self.nh * cache.hd
        self.q_ld, self.out_ld, self.shift = q_ld or width, out_ld or width, shift
        self.qbuf = rng.standard_normal(self.rows * self.q_ld + 8).astype(np.float32)
        self.start = np.concatenate([[0], np.cumsum([s[1] for s in sizes])])
        flat = np.array([m for tree in self.masks for m in tree] + [~0 & (2 ** 64 - 1)] * spare_rows, np.uint64)
        self.d = dict(seq=dev(self.slots, np.int32), ctx=dev([s[0] for s in sizes], np.int32),
                      start=dev(self.start, np.int32), mask=dev(flat), q=dev(self.qbuf))
        self.out = torch.full((self.rows * self.out_ld + 8,), -5.0, device="cuda")
        self.b = lrs.TreeBatch(self.d["seq"].data_ptr(), self.d["ctx"].data_ptr(), self.d["start"].data_ptr(),
                               None if masks == "chain" else self.d["mask"].data_ptr(), len(sizes), self.rows,
                               max_nodes or max(1, max(s[1] for s in sizes)),
                               max_len or max(1, max(s[0] + s[1] for s in sizes)))
        size = backend.tree_attention_workspace(cache.c, self.b, self.nh)
        self.space = torch.full((max(size, 16),), 0xff, dtype=torch.uint8, device="cuda")
        self.scale = cache.hd ** -0.5

    def q(self, tree):
        rows = range(self.start[tree], self.start[tree + 1])
        return np.array([self.qbuf[self.shift + r * self.q_ld:][:self.nh * self.cache.hd] for r in rows],
                        np.float32).reshape(-1, self.nh, self.cache.hd)

    def run(self, backend, stream=LEGACY):
        backend.tree_attention(self.cache.c, self.b, self.d["q"].data_ptr() + 4 * self.shift,
                               self.out.data_ptr() + 4 * self.shift, self.nh, scale=self.scale,
                               q_ld=self.q_ld, out_ld=self.out_ld, d_workspace=self.space.data_ptr(),
                               workspace_bytes=self.space.numel(), stream=stream)

    def check(self, skip=()):
        """Every row within its bound, the whole within 2^-16 of its norm, and
        nothing written between or behind the rows."""
        got = self.out.cpu().numpy().copy()
        width = self.nh * self.cache.hd
        num = den = 0.0
        for t, (ctx, n) in enumerate(self.sizes):
            if t in skip or n == 0:
                continue
            k, v = (self.cache.rows_of(self.slots[t], ctx + n, i) for i in range(2))
            want, err = kv_plain.attention(self.q(t), k, v, ctx, self.masks[t], self.scale)
            for i in range(n):
                at = self.shift + (self.start[t] + i) * self.out_ld
                row = got[at:at + width].reshape(self.nh, -1).astype(np.float64)
                off = np.abs(row - want[i])
                assert (off <= err[i]).all(), (t, i, float((off / np.maximum(err[i], 1e-300)).max()))
                num += float((off ** 2).sum())
                den += float((want[i] ** 2).sum())
                got[at:at + width] = -5.0
        assert num <= 2.0 ** -32 * den
        if not skip:
            assert (got == -5.0).all()


SIZES = {
    "one": [(0, 1)],
    "short": [(100, 5)],
    "decode": [(5, 1), (63, 1), (64, 1), (65, 1), (127, 1), (128, 1), (300, 1)],
    "ragged": [(0, 3), (1, 9), (61, 8), (127, 2), (130, 7), (255, 5), (500, 1)],
    "empty": [(70, 0), (10, 4), (0, 0), (0, 2), (200, 0)],
    "full": [(129, 64), (0, 64), (64, 63)],
    "many": [(i * 7 % 90, 1 + i % 5) for i in range(40)],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,group,hd", [(2, 7, 64), (2, 6, 128), (4, 7, 128), (1, 1, 64), (3, 8, 128)])
@pytest.mark.parametrize("sizes", list(SIZES))
def test_tree_attention(lrs, backend, dtype, heads, group, hd, sizes):
    s = SIZES[sizes]
    cache = Cache(lrs, dtype, heads, hd, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, group)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,nodes", [(16, 9), (64, 3), (9, 33), (5, 64)])
def test_tree_attention_wide_groups(lrs, backend, dtype, group, nodes):
    s = [(77, nodes), (3, nodes - 1)]
    cache = Cache(lrs, dtype, 1, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, group)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype,ctx,nodes,group", [("Q8_0", 20011, 3, 7), ("BF16", 9000, 16, 2), ("F32", 5003, 5, 4),
                                                   ("Q8_0", 3001, 64, 7)])
def test_tree_attention_long(lrs, backend, dtype, ctx, nodes, group):
    s = [(ctx, nodes), (17, 1)]
    cache = Cache(lrs, dtype, 2, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, group)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_chains_without_masks(lrs, backend, dtype):
    s = [(0, 64), (37, 30), (64, 1)]
    cache = Cache(lrs, dtype, 2, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 3, masks="chain")
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_ld,out_ld,shift", [(1025, 900, 1), (2048, 1028, 0), (900, 901, 3)])
def test_tree_attention_strides(lrs, backend, dtype, q_ld, out_ld, shift):
    s = [(40, 6), (130, 3)]
    cache = Cache(lrs, dtype, 1, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 7, q_ld=q_ld, out_ld=out_ld, shift=shift)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_attend_to_nothing(lrs, backend, dtype):
    """Mask 0 without committed positions gives zeros; bits past the tree's
    nodes count for nothing."""
    s = [(0, 5), (90, 4)]
    cache = Cache(lrs, dtype, 2, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 5)
    trees.masks[0][1] = trees.masks[0][4] = 0
    flat = [m for t in trees.masks for m in t]
    flat[0] |= 1 << 63 | 1 << 17  # no such nodes
    flat[4] = 1 << 40
    trees.d["mask"][:9].copy_(dev(np.array(flat, np.uint64)))
    trees.run(backend)
    sync_ok(backend)
    trees.check()
    assert (trees.out.cpu().numpy().reshape(-1)[128 * 10:128 * 20] == 0).all()


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_values_do_not_leak(lrs, backend, dtype, which, what):
    """A node whose K or V is not finite reaches only the nodes that attend to it."""
    import torch
    s = [(61, 8), (10, 2)]
    cache = Cache(lrs, dtype, 2, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 7, seed=4)
    bad, p = 5, 61 + 5
    for i in range(6, 8):  # nodes 6 and 7 do not descend from node 5; 7 is on 6
        trees.masks[0][i] = trees.masks[0][i - 1] & ~(1 << bad) if i == 7 else trees.masks[0][4] | 1 << 4
        trees.masks[0][i] |= 1 << i
    trees.d["mask"][:10].copy_(dev(np.array([m for t in trees.masks for m in t], np.uint64)))
    page, r = int(cache.pages[1, p // PAGE]), p % PAGE
    tile = cache.pool[which][page, 1]
    bits = {"nan": 0x7e00, "inf": 0x7c00} if dtype == "Q8_0" else {"nan": 0x7fc0, "inf": 0x7f80}
    if dtype == "Q8_0":  # a scale
        at = 64 * 128 + 2 * (64 + r if which else r * 4 + 1)
        tile[at:at + 2].view(torch.int16).fill_(bits[what])
    elif dtype == "BF16":
        tile.view(torch.int16)[r * 128 + 33] = bits[what]
    else:
        tile.view(torch.int32)[r * 128 + 33] = bits[what] << 16
    torch.cuda.synchronize()
    trees.run(backend)
    sync_ok(backend)
    got = trees.out.cpu().numpy()[:trees.rows * trees.out_ld].reshape(-1, trees.nh, 128)
    for i in range(8):
        if trees.masks[0][i] >> bad & 1:
            # K infinite: its score is +-inf (or NaN), and -inf is a weight of 0
            if which == 1 or what == "nan":
                assert not np.isfinite(got[i, 7:]).all()
            trees.out[i * trees.out_ld:(i + 1) * trees.out_ld] = 0.0
        else:
            assert np.isfinite(got[i]).all()
        assert np.isfinite(got[i, :7]).all()  # the other KV head
    # the rows that do not attend to it are exact: compare them on a batch without the node
    attends = [i for i in range(8) if trees.masks[0][i] >> bad & 1]
    k, v = (cache.rows_of(1, 69, i) for i in range(2))
    want, err = kv_plain.attention(trees.q(0), k, v, 61, trees.masks[0], trees.scale)
    for i in set(range(8)) - set(attends):
        assert (np.abs(got[i] - want[i]) <= err[i]).all()
    assert bad in attends and len(attends) < 8


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(lrs, backend, dtype):
    """Scores of several hundred, and rising along the context: the running
    maximum moves many times.  The bound grows with them as the arithmetic says."""
    s = [(700, 4), (256, 2)]
    cache = Cache(lrs, dtype, 1, 64, [c + n for c, n in reversed(s)])
    for p in range(700):  # K grows with the position
        cache.rows[0][cache.pages[1, p // PAGE], :, p % PAGE] *= p / 100.0
    cache.value[0] = kv_plain.held(lrs, cache.dtype, cache.rows[0])
    outside = ~np.broadcast_to(cache.inside[:, None], cache.rows[0].shape[:3])
    t = kv_plain.pack(lrs, cache.dtype, cache.rows[0], False)
    cache.pool[0].copy_(dev(np.where(cache.marks(outside, False), 0xff, t).astype(np.uint8)))
    trees = Trees(lrs, backend, cache, s, 4)
    trees.scale = 2.0
    trees.run(backend)
    sync_ok(backend)
    got = trees.out.cpu().numpy()
    for t, (ctx, n) in enumerate(s):
        k, v = (cache.rows_of(trees.slots[t], ctx + n, i) for i in range(2))
        want, err = kv_plain.attention(trees.q(t), k, v, ctx, trees.masks[t], 2.0)
        row = got[trees.start[t] * 256:trees.start[t + 1] * 256].reshape(n, 4, 64)
        assert (np.abs(row - want) <= err).all()


def test_values_over_many_magnitudes(lrs, backend):
    """V of 1e-6 to 1e4 and q of 1e-12 to 1e12, scale and sign negative."""
    for dtype in DTYPES:
        s = [(150, 6)]
        cache = Cache(lrs, dtype, 1, 128, [156])
        cache.rows[1][...] *= np.float32(10.0) ** np.linspace(-6, 4, 128, dtype=np.float32)
        cache.value[1] = kv_plain.held(lrs, cache.dtype, cache.rows[1])
        outside = ~np.broadcast_to(cache.inside[:, None], cache.rows[1].shape[:3])
        t = kv_plain.pack(lrs, cache.dtype, cache.rows[1], True)
        cache.pool[1].copy_(dev(np.where(cache.marks(outside, True), 0xff, t).astype(np.uint8)))
        for mag, scale in ((1e-12, -1e11), (1e12, 1e-13), (1.0, 0.0)):
            trees = Trees(lrs, backend, cache, s, 2)
            trees.qbuf *= np.float32(mag)
            trees.d["q"].copy_(dev(trees.qbuf))
            trees.scale = float(np.float32(scale))
            trees.run(backend)
            sync_ok(backend)
            k, v = (cache.rows_of(0, 156, i) for i in range(2))
            got = trees.out.cpu().numpy()[:6 * 256].reshape(6, 2, 128)
            for d in range(0, 128, 8):  # each column against its own magnitude
                want, err = kv_plain.attention(trees.q(0), k, v, 150, trees.masks[0], trees.scale)
                _, e = kv_plain.attention(trees.q(0), k, v[:, :, d:d + 8], 150, trees.masks[0], trees.scale)
                assert (np.abs(got - want)[:, :, d:d + 8] <= e).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_trees_are_skipped(lrs, backend, dtype):
    """Lengths above max_len, a bad slot or page, node counts above max_nodes:
    reported, and the other trees are right."""
    import torch
    s = [(30, 3), (100, 2), (20, 2), (60, 6), (64, 1)]
    cache = Cache(lrs, dtype, 2, 64, [c + n for c, n in reversed(s)])
    for breaks in range(4):
        trees = Trees(lrs, backend, cache, s, 3, max_nodes=6, max_len=102)
        if breaks == 0:
            trees.d["ctx"][1] = 2 ** 30
        elif breaks == 1:
            trees.d["seq"][1] = 77
        elif breaks == 2:
            table = cache.pages.copy()
            table[trees.slots[1], 1] = -1
            cache.d_pages.copy_(dev(table))
        else:
            trees.d["ctx"][1] = -3
        trees.run(backend)
        torch.cuda.synchronize()
        with pytest.raises(lrs.LrsError, match="out of range"):
            backend.synchronize()
        cache.d_pages.copy_(dev(cache.pages))
        trees.check(skip=(1,))


def test_nothing_to_do(lrs, backend):
    """All trees empty: no row is written."""
    cache = Cache(lrs, "Q8_0", 2, 64, [10, 10])
    trees = Trees(lrs, backend, cache, [(5, 0), (9, 0)], 2)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_streams_and_graph_replays(lrs, backend, dtype):
    """On a side stream and the backend's own; captured once, replayed with
    other lengths, masks, slots and rows, bit-equal to plain calls."""
    import torch
    s = [(100, 8), (300, 3), (7, 1)]
    cache = Cache(lrs, dtype, 2, 128, [400, 400, 400])
    trees = Trees(lrs, backend, cache, s, 7, max_nodes=16, max_len=400, spare_rows=20)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    trees.run(backend, stream=side.cuda_stream)
    sync_ok(backend)
    trees.check()
    first = trees.out.clone()
    trees.out.fill_(-5.0)
    torch.cuda.synchronize()
    trees.run(backend, stream=None)
    sync_ok(backend)
    assert torch.equal(first, trees.out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        trees.run(backend, stream=side.cuda_stream)
    for sizes in ([(0, 16), (399, 1), (200, 5)], [(64, 1), (64, 2), (128, 16)], s):
        again = Trees(lrs, backend, cache, sizes, 7, seed=9, max_nodes=16, max_len=400, spare_rows=0)
        n = again.n
        trees.d["ctx"].copy_(again.d["ctx"])
        trees.d["start"].copy_(again.d["start"])
        trees.d["mask"][:n].copy_(again.d["mask"][:n])
        trees.d["q"][:n * trees.q_ld].copy_(again.d["q"][:n * trees.q_ld])
        trees.out.fill_(-5.0)
        torch.cuda.synchronize()
        graph.replay()
        again.run(backend)
        sync_ok(backend)
        again.check()
        assert torch.equal(trees.out[:n * trees.out_ld], again.out[:n * trees.out_ld])
        assert (trees.out[n * trees.out_ld:] == -5.0).all()
    del graph


def test_two_graphs_at_once(lrs, backend):
    """Two captured calls with a workspace each run on two streams together."""
    import torch
    caches = [Cache(lrs, "Q8_0", 2, 128, [900, 900], seed=i) for i in range(2)]
    trees = [Trees(lrs, backend, c, [(800 + i, 9), (650, 12)], 7, seed=i) for i, c in enumerate(caches)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for t, st in zip(trees, streams):
        t.run(backend, stream=st.cuda_stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            t.run(backend, stream=st.cuda_stream)
        graphs.append(g)
    for t in trees:
        t.out.fill_(-5.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    sync_ok(backend)
    for t in trees:
        t.check()
    graphs.clear()


def test_results_repeat(lrs, backend):
    """The same call twice gives the same bits."""
    import torch
    s = [(1500, 9), (40, 20), (700, 1)]
    cache = Cache(lrs, "BF16", 2, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 7)
    trees.run(backend)
    sync_ok(backend)
    first = trees.out.clone()
    for _ in range(5):
        trees.space.random_(0, 256)
        trees.run(backend)
        sync_ok(backend)
        assert torch.equal(first, trees.out)


def test_pools_past_4_gb(lrs, backend):
    """Pages whose byte offsets pass 2^32: written, read, attended to and moved."""
    import torch
    heads, hd, pages = 1, 128, 140000
    pool = [torch.empty(pages * PAGE * hd, device="cuda") for _ in range(2)]  # 4.6 GB each
    table = np.array([[pages - 1, 5, pages - 2]], np.int32)
    d_pages = dev(table)
    c = lrs.KvCache(pool[0].data_ptr(), pool[1].data_ptr(), d_pages.data_ptr(), pages, 1, 3, heads, hd, 0)
    rng = np.random.default_rng(1)
    n = 150
    k, v = rng.standard_normal((2, n, 1, hd)).astype(np.float32)
    d_seq, d_pos, dk, dv = dev(np.zeros(n, np.int32)), dev(np.arange(n), np.int32), dev(k), dev(v)
    backend.kv_store(c, d_seq.data_ptr(), d_pos.data_ptr(), n, dk.data_ptr(), dv.data_ptr(), stream=LEGACY)
    out = torch.zeros(2, n, 1, hd, device="cuda")
    backend.kv_load(c, d_seq.data_ptr(), d_pos.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr(), stream=LEGACY)
    sync_ok(backend)
    assert np.array_equal(out[0].cpu().numpy(), k) and np.array_equal(out[1].cpu().numpy(), v)
    q = rng.standard_normal((2, 4, hd)).astype(np.float32)
    dq, ctx, start = dev(q), dev([148], np.int32), dev([0, 2], np.int32)
    b = lrs.TreeBatch(d_seq.data_ptr(), ctx.data_ptr(), start.data_ptr(), None, 1, 2, 2, 150)
    space = torch.empty(max(16, backend.tree_attention_workspace(c, b, 4)), dtype=torch.uint8, device="cuda")
    o = torch.zeros(2, 4, hd, device="cuda")
    backend.tree_attention(c, b, dq.data_ptr(), o.data_ptr(), 4, d_workspace=space.data_ptr(),
                           workspace_bytes=space.numel(), stream=LEGACY)
    nodes = dev([1], np.int32)
    backend.kv_accept(c, d_seq.data_ptr(), ctx.data_ptr(), dev([0, 1], np.int32).data_ptr(), nodes.data_ptr(), 1, 1,
                      stream=LEGACY)
    backend.kv_load(c, d_seq.data_ptr(), d_pos.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr(), stream=LEGACY)
    sync_ok(backend)
    want, err = kv_plain.attention(q, k.transpose(1, 0, 2).astype(np.float64), v.transpose(1, 0, 2).astype(np.float64),
                                   148, [1, 3], hd ** -0.5)
    assert (np.abs(o.cpu().numpy() - want) <= err).all()
    k[148], v[148] = k[149], v[149]
    assert np.array_equal(out[0].cpu().numpy(), k) and np.array_equal(out[1].cpu().numpy(), v)


# ----------------------------------------------------------------- accept ----
def accepted(cache, ctx, paths, slots):
    """The tiles after the paths' rows moved down."""
    got = []
    for i in range(2):
        t = [x.copy() for x in (cache.tiles[i],)][0]
        rows = np.arange(cache.c.n_pages * cache.heads * PAGE).reshape(-1, cache.heads, PAGE)
        for c, path, s in zip(ctx, paths, slots):
            moved = []
            for node in path:
                m = np.zeros(rows.shape, bool)
                m[cache.pages[s, (c + node) // PAGE], :, (c + node) % PAGE] = True
                mark = cache.marks(m, bool(i))
                moved.append([cache.tiles[i][p, h][mark[p, h]] for p in [cache.pages[s, (c + node) // PAGE]]
                              for h in range(cache.heads)])
            for j, data in enumerate(moved):
                m = np.zeros(rows.shape, bool)
                p = cache.pages[s, (c + j) // PAGE]
                m[p, :, (c + j) % PAGE] = True
                mark = cache.marks(m, bool(i))
                for h in range(cache.heads):
                    t[p, h][mark[p, h]] = data[h]
        got.append(t)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads", [(64, 2), (128, 3)])
def test_accept(lrs, backend, dtype, hd, heads):
    """Paths of every kind, across a page's end, in three caches at once."""
    ctx = [0, 61, 64, 100, 30, 5, 63]
    paths = [[0], [0, 2, 5, 6, 9], [], list(range(64)), list(range(0, 64, 3)), [63], [1, 2, 3, 4, 5, 6, 7, 8, 9, 60]]
    slots = [3, 0, 6, 1, 5, 2, 4]
    lens = [0] * 7
    for c, s in zip(ctx, slots):
        lens[s] = c + 64
    caches = [Cache(lrs, dtype, heads, hd, lens, seed=5) for _ in range(3)]
    for i, c in enumerate(caches):  # one page table, other rows
        other = Cache(lrs, dtype, heads, hd, lens, seed=5, scale=1.0 + i)
        c.tiles = other.tiles
        for a, b in zip(c.pool, other.pool):
            a.copy_(b)
        c.c.pages = caches[0].c.pages
    start = np.concatenate([[0], np.cumsum([len(p) for p in paths])])
    nodes = np.concatenate(paths).astype(np.int32)
    d = [dev(slots, np.int32), dev(ctx, np.int32), dev(start, np.int32), dev(nodes)]
    backend.kv_accept([c.c for c in caches], *(x.data_ptr() for x in d), 7, len(nodes), stream=LEGACY)
    sync_ok(backend)
    for c in caches:
        for got, want in zip(c.bytes_now(), accepted(c, ctx, paths, slots)):
            assert np.array_equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_paths_are_skipped(lrs, backend, dtype):
    import torch
    ctx, slots = [10, 20, 30, 50, 0, 120, 12], [0, 1, 2, 3, 4, 5, 99]
    paths = [[0, 3, 2], [1, 1], [64], [-1, 4], [2, 4], [3, 20], [1]]  # slot 5 has two pages only
    cache = Cache(lrs, dtype, 2, 64, [128] * 6)
    start = np.concatenate([[0], np.cumsum([len(p) for p in paths])])
    nodes = np.concatenate(paths).astype(np.int32)
    d = [dev(slots, np.int32), dev(ctx, np.int32), dev(start, np.int32), dev(nodes)]
    backend.kv_accept(cache.c, *(x.data_ptr() for x in d), 7, len(nodes), stream=LEGACY)
    torch.cuda.synchronize()
    with pytest.raises(lrs.LrsError, match="out of range"):
        backend.synchronize()
    for got, want in zip(cache.bytes_now(), accepted(cache, [0], [[2, 4]], [4])):
        assert np.array_equal(got, want)


def test_starts_at_the_ends_of_int32_are_skipped(lrs, backend):
    """Node ranges whose ends' difference passes 32 bits: no tree, nothing read."""
    import torch
    cache = Cache(lrs, "BF16", 2, 64, [100, 100])
    top, low = 2 ** 31 - 1, -2 ** 31
    for start in ([top - 10, low + 20], [0, top], [low, low + 8], [top, top - 3], [-5, 3], [3, 99]):
        d = [dev([0], np.int32), dev([20], np.int32), dev(start, np.int32), dev([0, 1, 2, 3, 4, 5, 6, 8], np.int32)]
        backend.kv_accept(cache.c, *(x.data_ptr() for x in d), 1, 8, stream=LEGACY)
        torch.cuda.synchronize()
        with pytest.raises(lrs.LrsError, match="out of range"):
            backend.synchronize()
        for got, want in zip(cache.bytes_now(), cache.tiles):
            assert np.array_equal(got, want)
        trees = Trees(lrs, backend, cache, [(20, 5), (30, 3)], 3, max_nodes=64, max_len=100)
        trees.d["start"].copy_(dev(start + [start[1]], np.int32))
        trees.run(backend)
        torch.cuda.synchronize()
        with pytest.raises(lrs.LrsError, match="out of range"):
            backend.synchronize()
        assert bool((trees.out == -5.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_batch(lrs, backend, dtype):
    """Trees without nodes may hold anything; the others are right and nothing is reported."""
    s = [(0, 0), (70, 3), (9, 0), (130, 1), (0, 0)]
    cache = Cache(lrs, dtype, 2, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 3, max_nodes=3, max_len=140)
    for i, (slot, ctx) in zip((0, 2, 4), ((-1, -7), (99, 2 ** 31 - 1), (0, 141))):
        trees.d["seq"][i], trees.d["ctx"][i] = slot, ctx
    trees.run(backend)
    sync_ok(backend)
    trees.check()
    d = [dev([-1, 3, 99], np.int32), dev([-5, 60, 2 ** 31 - 1], np.int32), dev([0, 0, 1, 1], np.int32), dev([2], np.int32)]
    backend.kv_accept(cache.c, *(x.data_ptr() for x in d), 3, 1, stream=LEGACY)
    sync_ok(backend)
    for got, want in zip(cache.bytes_now(), accepted(cache, [60], [[2]], [3])):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_len", [200, 3000, 40000])
def test_rows_by_the_batchs_bounds(lrs, backend, dtype, max_len):
    """The same trees under bounds that choose units of 16 and of 64 rows."""
    s = [(150, 9), (90, 30), (3, 5)]
    cache = Cache(lrs, dtype, 2, 64, [c + n for c, n in reversed(s)], extra=640)
    trees = Trees(lrs, backend, cache, s, 7, max_len=max_len)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


@pytest.mark.parametrize("dtype", ["BF16", "Q8_0"])
def test_more_trees_than_threads(lrs, backend, dtype):
    s = [(i * 7 % 60, i % 3) for i in range(2500)]
    cache = Cache(lrs, dtype, 1, 64, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 4)
    trees.run(backend)
    sync_ok(backend)
    trees.check()


def test_workspace_of_a_smaller_batch_is_no_larger(lrs, backend):
    rng = np.random.default_rng(11)
    cache = lrs.KvCache(4096, 8192, 4096, 64, 64, 4096, 2, 64, 2)

    def size(trees, nodes, length, heads):
        return backend.tree_attention_workspace(cache, lrs.TreeBatch(4096, 4096, 4096, None, trees, trees * nodes, nodes,
                                                                     length), 2 * heads)
    for _ in range(4000):
        big = [int(np.exp(rng.uniform(0, np.log(m + 0.99)))) for m in (300, 64, 9000)]
        small = [int(rng.integers(1, b + 1)) for b in big]
        heads = int(rng.integers(1, 9))
        assert size(*small, heads) <= size(*big, heads), (big, small, heads)


@pytest.mark.parametrize("dtype", DTYPES)
def test_out_may_be_q(lrs, backend, dtype):
    s = [(700, 9), (5, 2), (0, 1), (1500, 20)]
    cache = Cache(lrs, dtype, 2, 128, [c + n for c, n in reversed(s)])
    trees = Trees(lrs, backend, cache, s, 7)
    trees.run(backend)
    sync_ok(backend)
    want = trees.out.clone()
    trees.out = trees.d["q"]
    trees.run(backend)
    sync_ok(backend)
    rows = trees.n * trees.out_ld
    assert bool((trees.out[:rows] == want[:rows]).all())


def test_accept_in_more_caches_than_a_launch(lrs, backend):
    base = Cache(lrs, "BF16", 1, 64, [30])
    pools = [[p.clone() for p in base.pool] for _ in range(150)]
    caches = [lrs.KvCache(k.data_ptr(), v.data_ptr(), base.d_pages.data_ptr(), base.c.n_pages, 1, base.c.max_pages, 1,
                          64, 1) for k, v in pools]
    d = [dev([0], np.int32), dev([20], np.int32), dev([0, 2], np.int32), dev([3, 8], np.int32)]
    backend.kv_accept(caches, *(x.data_ptr() for x in d), 1, 2, stream=LEGACY)
    sync_ok(backend)
    want = accepted(base, [20], [[3, 8]], [0])
    for pool in pools:
        for got, w in zip(pool, want):
            assert np.array_equal(got.cpu().numpy(), w)


# --------------------------------------------------------- all of them, as used --
@pytest.mark.parametrize("dtype", DTYPES)
def test_draft_verify_accept(lrs, backend, dtype):
    """Three rounds of a speculative decode over one cache: the draft's rows are
    written behind the committed positions, its nodes attend, a path is kept;
    then the cache holds what writing the kept rows one by one would hold."""
    import torch
    heads, group, hd, slots = 2, 7, 128, 3
    rng = np.random.default_rng(8)
    cache = Cache(lrs, dtype, heads, hd, [0] * slots, extra=2)
    kept = [[np.zeros((0, heads, hd), np.float32)] * 2 for _ in range(slots)]
    ctx = [0] * slots
    space = None
    for rnd, counts in enumerate(([60, 63, 1], [8, 5, 64], [16, 1, 7])):
        n = sum(counts)
        k, v = rng.standard_normal((2, n, heads, hd)).astype(np.float32)
        q = rng.standard_normal((n, heads * group, hd)).astype(np.float32)
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        masks = [kv_plain.random_tree(rng, c) for c in counts]
        seq = np.repeat(np.arange(slots), counts).astype(np.int32)
        pos = np.concatenate([np.arange(c) + ctx[s] for s, c in enumerate(counts)]).astype(np.int32)
        d = [dev(x) for x in (seq, pos, k, v, q, np.arange(slots, dtype=np.int32), np.array(ctx, np.int32), start)]
        d_mask = dev(np.array([m for t in masks for m in t], np.uint64))
        backend.kv_store(cache.c, d[0].data_ptr(), d[1].data_ptr(), n, d[2].data_ptr(), d[3].data_ptr(), stream=LEGACY)
        b = lrs.TreeBatch(d[5].data_ptr(), d[6].data_ptr(), d[7].data_ptr(), d_mask.data_ptr(), slots, n, 64, 192)
        size = backend.tree_attention_workspace(cache.c, b, heads * group)
        space = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        out = torch.zeros(n, heads * group, hd, device="cuda")
        backend.tree_attention(cache.c, b, d[4].data_ptr(), out.data_ptr(), heads * group, d_workspace=space.data_ptr(),
                               workspace_bytes=space.numel(), stream=LEGACY)
        paths = []
        for s, c in enumerate(counts):  # the path to the last node
            paths.append([j for j in range(c) if masks[s][c - 1] >> j & 1])
        pstart = dev(np.concatenate([[0], np.cumsum([len(p) for p in paths])]), np.int32)
        nodes = dev(np.concatenate(paths), np.int32)
        backend.kv_accept(cache.c, d[5].data_ptr(), d[6].data_ptr(), pstart.data_ptr(), nodes.data_ptr(), slots,
                          nodes.numel(), stream=LEGACY)
        sync_ok(backend)
        got = out.cpu().numpy()
        for s, c in enumerate(counts):
            rows = slice(start[s], start[s + 1])
            both = [np.concatenate([kept[s][i], x[rows]]) for i, x in enumerate((k, v))]
            kk, vv = (kv_plain.held(lrs, cache.dtype, x).transpose(1, 0, 2) for x in both)
            want, err = kv_plain.attention(q[rows], kk, vv, ctx[s], masks[s], hd ** -0.5)
            assert (np.abs(got[rows] - want) <= err).all(), (rnd, s)
            kept[s] = [np.concatenate([kept[s][i], x[rows][paths[s]]]) for i, x in enumerate((k, v))]
            ctx[s] += len(paths[s])
        for s in range(slots):
            m = ctx[s]
            d_s, d_p = dev(np.full(m, s, np.int32)), dev(np.arange(m), np.int32)
            back = torch.zeros(2, m, heads, hd, device="cuda")
            backend.kv_load(cache.c, d_s.data_ptr(), d_p.data_ptr(), m, back[0].data_ptr(), back[1].data_ptr(), stream=LEGACY)
            sync_ok(backend)
            for i in range(2):
                want = kv_plain.held(lrs, cache.dtype, kept[s][i]).astype(np.float32)
                assert np.array_equal(back[i].cpu().numpy(), want)
