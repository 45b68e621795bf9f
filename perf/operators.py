"""What the paged KV cache's operators are measured on.

Four operators over the paged cache of a GQA decoder ([page][kv head] tiles of
64 positions, a page table per sequence slot):

* write: rows of K and V go into the cache, in its type (f32, bf16, or q8_0:
  blocks of 32 values with an f16 scale), then come back as the values that the
  cache now holds (``kv_store`` + ``kv_load``);
* read: rows of the cache come back as f32 values (``kv_load``);
* tree: attention of the nodes of drafted token trees over their sequences'
  committed positions and over the nodes' own ancestors (``tree_attention``);
  one node a sequence is a plain decode step, a chain a prompt chunk;
* accept: after a verification, the accepted nodes' rows move down to follow
  the committed positions, in the caches of all layers (``kv_accept``).

``run`` computes them with elementary torch operations, or with ``own`` through
the package's entry points, on the same state.

q8_0 tiles (64 * hd codes, then 64 * hd / 32 f16 scales): K codes are
[hd / 16][64][16] and its scales [64][hd / 32]; V codes are [16][hd][4] (four
positions of a column side by side) and its scales [hd / 32][64].
"""
import functools
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64          # positions a page
TREE_MAX = 64      # nodes a tree
LIMIT = 65024.0    # q8_0 holds values up to 512 * 127
DTYPES = {"f32": 0, "bf16": 1, "q8_0": 2}


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # the K/V rows of one decoded token, 0.5B heads: launch latency
        dict(name="write_1_row", op="write", dtype="q8_0", heads=2, dim=64, seqs=1, rows=1, ctx=127),
        # one decode step of the benchmark's 64 sequences, 7B heads
        dict(name="write_64_rows", op="write", dtype="q8_0", heads=4, dim=128, seqs=64, rows=1, ctx=1100),
        # 64 prompts of 1024 tokens moved into a cache at once
        dict(name="write_64x1024", op="write", dtype="q8_0", heads=4, dim=128, seqs=64, rows=1024, ctx=0),
        # a short prefix of one sequence read back, odd length
        dict(name="read_77_rows", op="read", dtype="q8_0", heads=2, dim=128, seqs=1, rows=77, ctx=33),
        # 64 sequences read back whole (moved to another host or another type)
        dict(name="read_64x1024", op="read", dtype="q8_0", heads=4, dim=128, seqs=64, rows=1024, ctx=0),
        # a small draft on a short chat, 0.5B heads, bf16 cache
        dict(name="tree_1x5_short", op="tree", dtype="bf16", heads=2, group=7, dim=64, seqs=1, nodes=5, ctx=100, ragged=0),
        # a decode step of the benchmark's 64 sequences over a q8_0 cache
        dict(name="tree_64x1_decode", op="tree", dtype="q8_0", heads=4, group=7, dim=128, seqs=64, nodes=1, ctx=1100, ragged=400),
        # drafts of up to 8 nodes for 64 sequences of ragged lengths
        dict(name="tree_64x8_ragged", op="tree", dtype="q8_0", heads=4, group=7, dim=128, seqs=64, nodes=8, ctx=4095, ragged=2000),
        # full trees of 64 nodes on long contexts
        dict(name="tree_4x64_long", op="tree", dtype="q8_0", heads=4, group=7, dim=128, seqs=4, nodes=64, ctx=8191, ragged=1000),
        # the default f32 cache, 1.5B heads
        dict(name="tree_8x13_f32", op="tree", dtype="f32", heads=2, group=6, dim=128, seqs=8, nodes=13, ctx=2049, ragged=500),
        # one sequence's accepted path, one layer
        dict(name="accept_1", op="accept", dtype="f32", heads=2, dim=64, seqs=1, nodes=9, ctx=61, caches=1),
        # 64 sequences, all 28 layers of the 7B shape
        dict(name="accept_64x28", op="accept", dtype="bf16", heads=4, dim=128, seqs=64, nodes=12, ctx=97, caches=28),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["write", "read", "tree", "tree", "tree", "accept"])
    heads, group, dim = rng.choice([(2, 7, 64), (2, 6, 128), (4, 7, 128), (8, 5, 128), (1, 8, 64), (3, 1, 128)])
    dtype = rng.choice(["q8_0", "q8_0", "bf16", "f32"])
    seqs = _log(rng, 1, 64)
    if op in ("write", "read"):
        rows = _log(rng, 1, max(1, 65536 // (seqs * max(1, heads // 4))) if seqs > 8 else 4096)
        return dict(op=op, dtype=dtype, heads=heads, dim=dim, seqs=seqs, rows=rows, ctx=rng.randrange(0, 200))
    if op == "accept":
        return dict(op=op, dtype=dtype, heads=heads, dim=dim, seqs=seqs, nodes=_log(rng, 1, 40), ctx=rng.randrange(0, 150),
                    caches=_log(rng, 1, 28))
    nodes = _log(rng, 1, TREE_MAX)
    # at most the listed cases' positions, and at most their products
    most = min(32000, 260000 // (seqs * max(1, heads // 4)), 2000000 // (seqs * nodes * max(1, heads // 4)))
    ctx = _log(rng, 1, max(1, most)) - 1
    return dict(op=op, dtype=dtype, heads=heads, group=group, dim=dim, seqs=seqs, nodes=nodes, ctx=ctx,
                ragged=rng.choice([0, ctx // 3, ctx]))


def _tree_sizes(case):
    """[(committed positions, nodes)] of each tree: ragged, down to none committed."""
    got = []
    for i in range(case["seqs"]):
        ctx = case["ctx"] - (i * 617) % (case["ragged"] + 1)
        n = case["nodes"] if case["nodes"] == 1 else max(1, case["nodes"] - i % 3)
        got.append((ctx, n))
    return got


def _kept(case):
    """Accepted nodes of each tree, from none to all."""
    return [(i * 5 + 3) % (case["nodes"] + 1) if case["seqs"] > 1 else (case["nodes"] + 1) // 2 for i in range(case["seqs"])]


def _row_bytes(dtype, dim):
    return {"f32": 4 * dim, "bf16": 2 * dim, "q8_0": dim // 32 * 34}[dtype]


def work(case):
    h, d = case["heads"], case["dim"]
    cell = 2 * h * _row_bytes(case["dtype"], d)  # one position's K and V, all heads
    if case["op"] in ("write", "read"):
        n = case["seqs"] * case["rows"]
        floats = 2 * h * d * 4
        if case["op"] == "write":
            return {"bytes": n * (floats + cell + cell + floats), "flops": n * 2 * h * d * 3}
        return {"bytes": n * (cell + floats), "flops": n * 2 * h * d}
    if case["op"] == "accept":
        return {"bytes": 2 * sum(_kept(case)) * cell * case["caches"], "flops": 0}
    g = case["group"]
    sizes = _tree_sizes(case)
    nodes = sum(n for _, n in sizes)
    return {"bytes": sum(c + n for c, n in sizes) * cell + 2 * nodes * h * g * d * 4,
            "flops": sum(4 * n * g * h * d * (c + n) for c, n in sizes)}


# ------------------------------------------------------------------ state ---
def _pool_shape(dtype, pages, heads, dim):
    if dtype == "q8_0":
        return (pages, heads, PAGE * _row_bytes(dtype, dim)), torch.uint8
    return (pages, heads, PAGE, dim), torch.float32 if dtype == "f32" else torch.bfloat16


def _rows(gen, n, heads, dim, k):
    """Rows as a projection leaves them: K has a few channels with a large bias."""
    x = torch.randn(n, heads, dim, device="cuda", generator=gen)
    if k:
        bias = torch.zeros(heads, dim, device="cuda")
        bias[:, dim // 5] = 6.0
        bias[:, dim // 2 + 3] = -4.0
        x = x + bias
    return x


def _filled(dtype, pages, heads, dim, gen, k):
    """A pool of pages full of rows."""
    shape, kind = _pool_shape(dtype, pages, heads, dim)
    x = _rows(gen, pages * PAGE, heads, dim, k).view(pages, PAGE, heads, dim).transpose(1, 2)
    if dtype != "q8_0":
        return x.to(kind).contiguous()
    codes, scale = _encode(x)
    pool = torch.empty(shape, dtype=torch.uint8, device="cuda")
    c, s = _planes(pool, dim, k)
    if k:
        c.copy_(codes.unflatten(3, (dim // 16, 16)).transpose(2, 3))
        s.copy_(scale)
    else:
        c.copy_(codes.unflatten(2, (PAGE // 4, 4)).transpose(3, 4))
        s.copy_(scale.transpose(2, 3))
    return pool


def _page_table(seqs, per_seq, gen):
    """Every slot its pages, in no order; [slots][per_seq + 1] with an unused column."""
    pages = torch.randperm(seqs * per_seq, device="cuda", generator=gen).to(torch.int32).view(seqs, per_seq)
    return torch.cat([pages, torch.zeros(seqs, 1, dtype=torch.int32, device="cuda")], 1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, dtype, h, d, b = case["op"], case["dtype"], case["heads"], case["dim"], case["seqs"]
    st = dict(op=op, dtype=dtype, heads=h, dim=d)
    if op in ("write", "read"):
        last = case["ctx"] + case["rows"]
        per = -(-last // PAGE)
        st["pages"] = _page_table(b, per, gen)
        slots = torch.randperm(b, device="cuda", generator=gen).to(torch.int32)
        st["seq"] = slots.repeat_interleave(case["rows"])
        st["pos"] = torch.arange(case["ctx"], last, device="cuda", dtype=torch.int32).repeat(b)
        n = b * case["rows"]
        shape, kind = _pool_shape(dtype, b * per, h, d)
        if op == "write":
            st["k"], st["v"] = _rows(gen, n, h, d, True), _rows(gen, n, h, d, False)
            st["pool_k"] = torch.zeros(shape, dtype=kind, device="cuda")
            st["pool_v"] = torch.zeros(shape, dtype=kind, device="cuda")
        else:
            st["pool_k"] = _filled(dtype, b * per, h, d, gen, True)
            st["pool_v"] = _filled(dtype, b * per, h, d, gen, False)
        st["out_k"] = torch.empty(n, h, d, device="cuda")
        st["out_v"] = torch.empty(n, h, d, device="cuda")
        return st
    if op == "accept":
        per = -(-(case["ctx"] + case["nodes"]) // PAGE)
        st["pages"] = _page_table(b, per, gen)
        st["seq"] = torch.randperm(b, device="cuda", generator=gen).to(torch.int32)
        st["ctx"] = torch.full((b,), case["ctx"], dtype=torch.int32, device="cuda")
        kept = torch.tensor(_kept(case), device="cuda")
        st["start"] = torch.cat([kept.new_zeros(1), kept.cumsum(0)]).to(torch.int32)
        # each tree's path: `kept` of its nodes, in order
        mark = torch.rand(b, case["nodes"], device="cuda", generator=gen).argsort(1)
        take = torch.where(torch.arange(case["nodes"], device="cuda")[None] < kept[:, None], mark, case["nodes"]).sort(1).values
        st["nodes"] = take[take < case["nodes"]].to(torch.int32)
        c = case["caches"]
        st["pool_k"] = _filled(dtype, c * b * per, h, d, gen, True)
        st["pool_v"] = _filled(dtype, c * b * per, h, d, gen, False)
        st["pool_k"] = st["pool_k"].view(c, b * per, *st["pool_k"].shape[1:])
        st["pool_v"] = st["pool_v"].view(c, b * per, *st["pool_v"].shape[1:])
        return st
    g = case["group"]
    sizes = _tree_sizes(case)
    per = -(-max(c + n for c, n in sizes) // PAGE)
    st["pages"] = _page_table(b, per, gen)
    st["seq"] = torch.randperm(b, device="cuda", generator=gen).to(torch.int32)
    st["ctx"] = torch.tensor([c for c, _ in sizes], dtype=torch.int32, device="cuda")
    counts = torch.tensor([n for _, n in sizes], device="cuda")
    st["start"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    st["max_nodes"], st["max_len"] = max(n for _, n in sizes), max(c + n for c, n in sizes)
    # a random tree: node i hangs on one of the nodes before it
    n = int(counts.sum())
    u = torch.rand(b, st["max_nodes"], device="cuda", generator=gen)
    masks = torch.ones(b, 1, dtype=torch.int64, device="cuda")
    for i in range(1, st["max_nodes"]):
        parent = (u[:, i:i + 1] * i).long().clamp(max=i - 1)
        bit = 1 << i if i < 63 else -(1 << 63)
        masks = torch.cat([masks, masks.gather(1, parent) | bit], 1)
    inside = torch.arange(st["max_nodes"], device="cuda")[None] < counts[:, None]
    st["mask"] = masks[inside].contiguous()
    st["q"] = torch.randn(n, h * g, d, device="cuda", generator=gen)
    st["group"], st["scale"] = g, 1.0 / math.sqrt(d)
    st["out"] = torch.empty(n, h * g, d, device="cuda")
    st["pool_k"] = _filled(dtype, b * per, h, d, gen, True)
    st["pool_v"] = _filled(dtype, b * per, h, d, gen, False)
    return st


# ------------------------------------------------------------ plain forms ---
def _half_away(x):
    t = torch.trunc(x)
    return t + torch.sign(x) * ((x - t).abs() >= 0.5)


def _encode(x):
    """q8_0 blocks of 32: int8 codes and f16 scales, from f32 values."""
    blocks = torch.nan_to_num(x, nan=0.0).clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    d = blocks.abs().amax(-1) / torch.full((), 127.0, device=x.device)
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    codes = _half_away(blocks * inv[..., None]).clamp(-127, 127)
    return codes.to(torch.int8).flatten(-2), d.half()


def _planes(pool, dim, k):
    """Views of a q8_0 pool's codes and scales."""
    lead = pool.dim() - 1
    codes = pool[..., :PAGE * dim].view(torch.int8)
    scale = pool[..., PAGE * dim:].view(torch.float16)
    if k:
        return codes.unflatten(lead, (dim // 16, PAGE, 16)), scale.unflatten(lead, (PAGE, dim // 32))
    return codes.unflatten(lead, (PAGE // 4, dim, 4)), scale.unflatten(lead, (dim // 32, PAGE))


def _put(pool, dtype, page, r, x, k):
    """Rows x [n, heads, dim] to row r of page `page`."""
    if dtype != "q8_0":
        pool[page, :, r] = x.to(pool.dtype)
        return
    codes, scale = _encode(x)
    c, s = _planes(pool, x.shape[-1], k)
    if k:
        c[page, :, :, r] = codes.unflatten(-1, (-1, 16))
        s[page, :, r] = scale
    else:
        c[page, :, r // 4, :, r % 4] = codes
        s[page, :, :, r] = scale


def _get(pool, dtype, dim, page, r, k):
    if dtype != "q8_0":
        return pool[page, :, r].float()
    c, s = _planes(pool, dim, k)
    if k:
        codes, scale = c[page, :, :, r].flatten(-2), s[page, :, r]
    else:
        codes, scale = c[page, :, r // 4, :, r % 4], s[page, :, :, r]
    return (codes.float().unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(-2)


def _whole(pool, dtype, dim, pages, k):
    """f32 values [trees, heads, positions, dim] of the pages [trees, n]."""
    if dtype != "q8_0":
        x = pool[pages].float()
    else:
        c, s = _planes(pool[pages.flatten()], dim, k)
        if k:
            codes, scale = c.transpose(2, 3).flatten(3), s
        else:
            codes, scale = c.transpose(3, 4).flatten(2, 3), s.transpose(2, 3)
        x = (codes.float().unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(-2)
        x = x.unflatten(0, pages.shape)
    return x.transpose(1, 2).flatten(2, 3)


def _tree_plain(st):
    b, t, g, h, d = st["seq"].numel(), st["max_nodes"], st["group"], st["heads"], st["dim"]
    start, ctx = st["start"].long(), st["ctx"].long()
    pages = st["pages"][st["seq"].long(), :-(-st["max_len"] // PAGE)].long()
    k = _whole(st["pool_k"], st["dtype"], d, pages, True)
    v = _whole(st["pool_v"], st["dtype"], d, pages, False)
    length = k.shape[2]
    tree = torch.arange(t, device="cuda")
    inside = tree[None] < (start[1:] - start[:-1])[:, None]
    at = (start[:-1, None] + tree).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][at].view(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d)
    node = torch.arange(length, device="cuda")[None] - ctx[:, None]  # < 0: committed
    bits = (st["mask"][at][:, :, None] >> node.clamp(0, 63)[:, None]) & 1
    seen = (node < 0)[:, None] | ((node < t)[:, None] & (bits == 1))
    seen = seen[:, None, :, None].expand(b, 1, t, g, length).reshape(b, 1, t * g, length)
    s = torch.matmul(q, k.transpose(2, 3)) * st["scale"]
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.view(b, h, t, g, d).permute(0, 2, 1, 3, 4).reshape(b, t, h * g, d)
    return o[inside]


def _cells(st, pos, seq):
    """Page and row of positions of slots."""
    pos = pos.long()
    return st["pages"][seq.long(), pos // PAGE].long(), pos % PAGE


def _accept_plain(st):
    start, ctx, seq = st["start"].long(), st["ctx"].long(), st["seq"].long()
    n = st["nodes"].numel()
    tree = torch.searchsorted(start, torch.arange(n, device="cuda"), right=True) - 1
    j = torch.arange(n, device="cuda") - start[tree]
    ps, rs = _cells(st, ctx[tree] + st["nodes"], seq[tree])
    pd, rd = _cells(st, ctx[tree] + j, seq[tree])
    for pool, k in ((st["pool_k"], True), (st["pool_v"], False)):
        if st["dtype"] != "q8_0":
            pool[:, pd, :, rd] = pool[:, ps, :, rs]
            continue
        c, s = _planes(pool, st["dim"], k)
        if k:
            c[:, pd, :, :, rd] = c[:, ps, :, :, rs]
            s[:, pd, :, rd] = s[:, ps, :, rs]
        else:
            c[:, pd, :, rd // 4, :, rd % 4] = c[:, ps, :, rs // 4, :, rs % 4]
            s[:, pd, :, :, rd] = s[:, ps, :, :, rs]
    return st["pool_k"], st["pool_v"]


# ----------------------------------------------------- the package's calls ---
@functools.lru_cache(None)
def _backend():
    lrs = sys.modules.get("llamars_b200")
    if lrs is None:
        pkg = os.path.join(os.getcwd(), "llama.rs_b200")
        spec = importlib.util.spec_from_file_location("llamars_b200", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        lrs = sys.modules["llamars_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(lrs)
    return lrs, lrs.CudaBackend(torch.cuda.current_device())


def _cache(lrs, st, pool_k, pool_v):
    slots, width = st["pages"].shape
    return lrs.KvCache(pool_k.data_ptr(), pool_v.data_ptr(), st["pages"].data_ptr(), pool_k.shape[0], slots, width,
                       st["heads"], st["dim"], DTYPES[st["dtype"]])


def _run_own(st):
    lrs, be = _backend()
    stream = torch.cuda.current_stream().cuda_stream
    if "caches" not in st:  # the descriptors, and the attention's workspace
        if st["op"] == "accept":
            caches = [_cache(lrs, st, k, v) for k, v in zip(st["pool_k"], st["pool_v"])]
            st["caches"] = (lrs.KvCache * len(caches))(*caches)
        else:
            st["caches"] = [_cache(lrs, st, st["pool_k"], st["pool_v"])]
        if st["op"] == "tree":
            st["trees"] = lrs.TreeBatch(st["seq"].data_ptr(), st["ctx"].data_ptr(), st["start"].data_ptr(), st["mask"].data_ptr(),
                                        st["seq"].numel(), st["q"].shape[0], st["max_nodes"], st["max_len"])
            size = be.tree_attention_workspace(st["caches"][0], st["trees"], st["q"].shape[1])
            st["space"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    cache = st["caches"][0]
    if st["op"] == "tree":
        be.tree_attention(cache, st["trees"], st["q"].data_ptr(), st["out"].data_ptr(), st["q"].shape[1], scale=st["scale"],
                          d_workspace=st["space"].data_ptr(), workspace_bytes=st["space"].numel(), stream=stream)
        return st["out"]
    if st["op"] == "accept":
        be.kv_accept(st["caches"], st["seq"].data_ptr(), st["ctx"].data_ptr(), st["start"].data_ptr(), st["nodes"].data_ptr(),
                     st["seq"].numel(), st["nodes"].numel(), stream=stream)
        return st["pool_k"], st["pool_v"]
    n, seq, pos = st["pos"].numel(), st["seq"].data_ptr(), st["pos"].data_ptr()
    if st["op"] == "write":
        be.kv_store(cache, seq, pos, n, st["k"].data_ptr(), st["v"].data_ptr(), stream=stream)
    be.kv_load(cache, seq, pos, n, st["out_k"].data_ptr(), st["out_v"].data_ptr(), stream=stream)
    return st["out_k"], st["out_v"]


def run(state):
    st = state
    if own:
        return _run_own(st)
    if st["op"] == "tree":
        return _tree_plain(st)
    if st["op"] == "accept":
        return _accept_plain(st)
    page, r = _cells(st, st["pos"], st["seq"])
    if st["op"] == "write":
        _put(st["pool_k"], st["dtype"], page, r, st["k"], True)
        _put(st["pool_v"], st["dtype"], page, r, st["v"], False)
    return _get(st["pool_k"], st["dtype"], st["dim"], page, r, True), _get(st["pool_v"], st["dtype"], st["dim"], page, r, False)


# ------------------------------------------------------------------ 64 bits -
def _exact_rows(pool, dtype, dim, pages, first, last, k):
    """Positions first..last of one sequence from the bytes of its tiles, in 64
    bits: [heads, positions, dim]."""
    pos = torch.arange(first, last, device="cuda")
    page, r = pages[pos // PAGE].long(), pos % PAGE
    heads = pool.shape[1]
    if dtype != "q8_0":
        return torch.stack([pool[page, i, r] for i in range(heads)]).double()
    col = torch.arange(dim, device="cuda")
    if k:
        code_at = (col // 16)[None] * (PAGE * 16) + r[:, None] * 16 + (col % 16)[None]
        scale_at = r[:, None] * (dim // 32) + (col // 32)[None]
    else:
        code_at = (r // 4)[:, None] * (4 * dim) + col[None] * 4 + (r % 4)[:, None]
        scale_at = (col // 32)[None] * PAGE + r[:, None]
    got = []
    for i in range(heads):
        tile = pool[:, i]
        code = tile[page[:, None], code_at].to(torch.int64)
        code = torch.where(code > 127, code - 256, code).double()
        lo = tile[page[:, None], PAGE * dim + 2 * scale_at].to(torch.int32)
        hi = tile[page[:, None], PAGE * dim + 2 * scale_at + 1].to(torch.int32)
        bits = lo | (hi << 8)
        bits = torch.where(bits > 32767, bits - 65536, bits).to(torch.int16)
        got.append(code * bits.view(torch.float16).double())
    return torch.stack(got)


def _exact_written(x, dtype):
    """The value that the cache holds for each f32 value of x, by the format's
    definition: q8_0 rounds amax / 127, its reciprocal and each product to f32
    (a 64-bit result rounded to f32 is the f32 operation's)."""
    y = x.double()
    if dtype == "f32":
        return y
    if dtype == "bf16":
        return y.to(torch.bfloat16).double()
    y = y.clamp(-LIMIT, LIMIT).view(*y.shape[:-1], -1, 32)
    d = (y.abs().max(-1, keepdim=True).values / 127).float().double()
    inv = torch.where(d > 0, 1 / d, d).float().double()
    z = (y * inv).float().double()
    code = torch.floor(z.abs() + 0.5) * torch.sign(z)
    return (code.clamp(-127, 127) * d.half().double()).view(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    dtype, d, h = st["dtype"], st["dim"], st["heads"]
    if case["op"] == "write":
        return _exact_written(st["k"], dtype), _exact_written(st["v"], dtype)
    if case["op"] == "read":
        seqs = st["seq"].view(case["seqs"], case["rows"])[:, 0].tolist()
        both = []
        for pool, k in ((st["pool_k"], True), (st["pool_v"], False)):
            rows = [_exact_rows(pool, dtype, d, st["pages"][s], case["ctx"], case["ctx"] + case["rows"], k) for s in seqs]
            both.append(torch.stack(rows).transpose(1, 2).reshape(-1, h, d))
        return tuple(both)
    if case["op"] == "accept":
        if dtype == "q8_0":
            return None  # bytes that move
        start, nodes, seqs = st["start"].tolist(), st["nodes"].tolist(), st["seq"].tolist()
        pages = st["pages"].cpu().numpy()
        src, dst = [], []
        for i, s in enumerate(seqs):
            for j, node in enumerate(nodes[start[i]:start[i + 1]]):
                a, b = case["ctx"] + node, case["ctx"] + j
                src.append((int(pages[s, a // PAGE]), a % PAGE))
                dst.append((int(pages[s, b // PAGE]), b % PAGE))
        both = []
        for pool in (st["pool_k"], st["pool_v"]):
            out = pool.double()
            for (pa, ra), (pb, rb) in zip(src, dst):
                out[:, pb, :, rb] = pool[:, pa, :, ra].double()
            both.append(out)
        return tuple(both)
    out = torch.empty_like(st["q"], dtype=torch.float64)
    start, seqs = st["start"].tolist(), st["seq"].tolist()
    for i, (ctx, n) in enumerate(_tree_sizes(case)):
        k = _exact_rows(st["pool_k"], dtype, d, st["pages"][seqs[i]], 0, ctx + n, True)
        v = _exact_rows(st["pool_v"], dtype, d, st["pages"][seqs[i]], 0, ctx + n, False)
        masks = np.array([[int(m) >> j & 1 for j in range(n)] for m in st["mask"][start[i]:start[i + 1]].tolist()], dtype=bool)
        seen = torch.ones(n, ctx + n, dtype=torch.bool, device="cuda")
        seen[:, ctx:] = torch.from_numpy(masks).cuda()
        for head in range(h):
            for j in range(case["group"]):
                qh = head * case["group"] + j
                s = st["q"][start[i]:start[i + 1], qh].double() @ k[head].T * st["scale"]
                out[start[i]:start[i + 1], qh] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v[head]
    return out
