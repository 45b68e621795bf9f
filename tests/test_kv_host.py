"""The paged KV cache's operators on the host: their checks of arguments (no
CUDA call is made before them) and the plain forms the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import kv_plain

INVALID, UNSUPPORTED = 1, 2
A = 4096  # an aligned address that no refused call reads


def _cache(lrs, **kw):
    f = dict(k_pool=A, v_pool=A, pages=A, n_pages=8, n_seqs=2, max_pages=4, kv_heads=2,
             head_dim=128, kv_dtype=2)
    f.update(kw)
    return lrs.KvCache(**f)


def _trees(lrs, **kw):
    f = dict(seq=A, ctx=A, start=A, mask=A, n_trees=1, n_nodes=4, max_nodes=4, max_len=100)
    f.update(kw)
    return lrs.TreeBatch(**f)


class _Host:
    """A CudaBackend's methods on a handle that no device stands behind: a
    refused call returns before it touches the backend."""

    def __new__(cls, lrs):
        be = object.__new__(lrs.CudaBackend)
        be._h, be._models, be._cache = None, [], {}
        return be


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype,row", [(0, 4), (1, 2), (2, 34 / 32)])
def test_tile_bytes(lrs, hd, dtype, row):
    assert _cache(lrs, head_dim=hd, kv_dtype=dtype).tile_bytes() == 64 * hd * row


@pytest.mark.parametrize("bad,code", [
    (dict(kv_dtype=3), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
    (dict(n_pages=0), INVALID), (dict(n_seqs=0), INVALID), (dict(max_pages=0), INVALID),
    (dict(kv_heads=0), INVALID), (dict(kv_heads=70000), INVALID), (dict(n_pages=1 << 31), INVALID),
    (dict(max_pages=1 << 26), INVALID), (dict(k_pool=None), INVALID), (dict(v_pool=None), INVALID),
    (dict(pages=None), INVALID), (dict(k_pool=A + 8), INVALID), (dict(v_pool=A + 4), INVALID)], ids=str)
def test_bad_caches_are_refused(lrs, bad, code):
    c, be = _cache(lrs, **bad), _Host(lrs)
    for call in (c.tile_bytes, lambda: be.kv_store(c, A, A, 1, A, A), lambda: be.kv_load(c, A, A, 1, A, A),
                 lambda: be.kv_accept([c], A, A, A, A, 1, 1), lambda: be.tree_attention_workspace(c, _trees(lrs), 4),
                 lambda: be.tree_attention(c, _trees(lrs), A, A, 4, d_workspace=A, workspace_bytes=1 << 30)):
        with pytest.raises(lrs.LrsError) as e:
            call()
        assert e.value.code == code


def test_null_arguments_are_refused(lrs):
    c, be = _cache(lrs), _Host(lrs)
    lib = lrs.library()
    assert lib.lrs_kv_check(None, None) == INVALID
    for call in (lambda: be.kv_store(c, A, A, 1, A, A),  # the null backend
                 lambda: be.kv_load(c, None, A, 1, A, A), lambda: be.kv_accept([c], A, None, A, A, 1, 1),
                 lambda: be.tree_attention(c, _trees(lrs), None, A, 4),
                 lambda: be.tree_attention_workspace(c, _trees(lrs), 4)):
        with pytest.raises(lrs.LrsError) as e:
            call()
        assert e.value.code == INVALID
    assert lib.lrs_tree_attention_workspace(None, C.byref(c), None, 4, None) == INVALID


def test_empty_calls_do_nothing(lrs):
    c, be = _cache(lrs), _Host(lrs)
    be.kv_store(c, None, None, 0, None, None)
    be.kv_load(c, None, None, 0, None, None)
    be.kv_load(c, A, A, 5, None, None)
    be.kv_accept([], A, A, A, A, 1, 1)
    be.kv_accept([c], None, None, None, None, 0, 0)
    be.tree_attention(c, _trees(lrs, n_trees=0), None, None, 4)
    be.tree_attention(c, _trees(lrs, n_nodes=0), None, None, 4)


@pytest.mark.parametrize("ld", [1, 255])
def test_short_row_strides_are_refused(lrs, ld):
    c, be = _cache(lrs), _Host(lrs)
    for call in (lambda: be.kv_store(c, A, A, 1, A, A, ld=ld), lambda: be.kv_load(c, A, A, 1, A, A, ld=ld),
                 lambda: be.tree_attention(c, _trees(lrs), A, A, 4, q_ld=ld),
                 lambda: be.tree_attention(c, _trees(lrs), A, A, 4, out_ld=ld)):
        with pytest.raises(lrs.LrsError, match="stride") as e:
            call()
        assert e.value.code == INVALID


@pytest.mark.parametrize("trees,heads,code", [
    (dict(max_nodes=0), 4, INVALID), (dict(max_nodes=65), 4, INVALID), (dict(max_len=0), 4, INVALID),
    (dict(max_len=257), 4, INVALID), (dict(seq=None), 4, INVALID), (dict(ctx=None), 4, INVALID),
    (dict(start=None), 4, INVALID), (dict(), 3, INVALID), (dict(), 0, INVALID), (dict(), 130, UNSUPPORTED),
    (dict(n_trees=1 << 17), 4, UNSUPPORTED), (dict(n_nodes=1 << 25), 4, UNSUPPORTED)], ids=str)
def test_bad_trees_are_refused(lrs, trees, heads, code):
    c, be = _cache(lrs), _Host(lrs)
    with pytest.raises(lrs.LrsError) as e:
        be.tree_attention(c, _trees(lrs, **trees), A, A, heads, d_workspace=A, workspace_bytes=1 << 30)
    assert e.value.code == code


def test_bad_scale_is_refused(lrs):
    for scale in (float("nan"), float("inf")):
        with pytest.raises(lrs.LrsError, match="scale"):
            _Host(lrs).tree_attention(_cache(lrs), _trees(lrs), A, A, 4, scale=scale)


def test_accept_wants_equal_caches(lrs):
    be = _Host(lrs)
    for other in (dict(pages=2 * A), dict(n_pages=9), dict(n_seqs=3), dict(max_pages=5), dict(kv_heads=1),
                  dict(head_dim=64), dict(kv_dtype=1)):
        with pytest.raises(lrs.LrsError, match="pools only"):
            be.kv_accept([_cache(lrs), _cache(lrs, **other)], A, A, A, A, 1, 1)


def test_accept_wants_distinct_pools(lrs):
    be = _Host(lrs)
    apart = [_cache(lrs, k_pool=A * (2 * i + 2), v_pool=A * (2 * i + 3)) for i in range(3)]
    for bad in (dict(k_pool=apart[0].k_pool), dict(v_pool=apart[1].v_pool),
                             dict(k_pool=apart[0].v_pool), dict(v_pool=apart[1].k_pool)):
        last = _cache(lrs, **{**dict(k_pool=50 * A, v_pool=51 * A), **bad})
        with pytest.raises(lrs.LrsError, match="named twice") as e:
            be.kv_accept(apart + [last], A, A, A, A, 1, 1)
        assert e.value.code == INVALID
    with pytest.raises(lrs.LrsError, match="named twice"):  # one cache's two pools
        be.kv_accept([_cache(lrs)], A, A, A, A, 1, 1)


def test_unaligned_arrays_are_refused(lrs):
    be, B = _Host(lrs), A + 2
    c = _cache(lrs, v_pool=2 * A)
    calls = [lambda i=i: be.kv_store(c, *(B if j == i else A for j in range(2)), 1,
                                     *(B if j == i else A for j in (2, 3))) for i in range(4)]
    calls += [lambda i=i: be.kv_load(c, *(B if j == i else A for j in range(2)), 1,
                                     *(B if j == i else A for j in (2, 3))) for i in range(4)]
    calls += [lambda i=i: be.kv_accept([c], *(B if j == i else A for j in range(4)), 1, 1) for i in range(4)]
    calls += [lambda n=n: be.tree_attention_workspace(c, _trees(lrs, **{n: B}), 4) for n in ("seq", "ctx", "start", "mask")]
    calls += [lambda: be.tree_attention_workspace(c, _trees(lrs, mask=A + 4), 4)]
    calls += [lambda q=q: be.tree_attention(c, _trees(lrs), *q, 4, d_workspace=A, workspace_bytes=1 << 30)
              for q in ((B, A), (A, B))]
    calls += [_cache(lrs, pages=B).tile_bytes]
    be._h = C.c_void_p(A)  # a handle that the refused calls do not read
    try:
        for call in calls:
            with pytest.raises(lrs.LrsError, match="aligned") as e:
                call()
            assert e.value.code == INVALID
    finally:
        be._h = None


def test_lengths_near_int32_are_refused(lrs):
    c = _cache(lrs, max_pages=(2 ** 31 - 1) // 64)
    with pytest.raises(lrs.LrsError) as e:
        _Host(lrs).tree_attention_workspace(c, _trees(lrs, max_len=2 ** 31 - 64), 2)
    assert e.value.code == UNSUPPORTED


def test_default_stream_is_not_the_backends(lrs):
    assert [lrs._cuda_stream(s) for s in (None, 0, 1, 12345)] == [None, 1, 1, 12345]


@pytest.mark.parametrize("hd", [64, 128])
def test_plain_layout_holds_the_values(lrs, hd):
    """The packed tiles, read by the layout's formulas, are the held values."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 3, 64, hd)).astype(np.float32)
    want = kv_plain.held(lrs, lrs.KvType.Q8_0, x)
    for is_v in (False, True):
        t = kv_plain.pack(lrs, lrs.KvType.Q8_0, x, is_v)
        assert t.shape[2] == 64 * hd // 32 * 34
        for p, h, r, c in ((0, 0, 0, 0), (1, 2, 63, hd - 1), (0, 1, 37, 45), (1, 0, 2, 17), (0, 2, 5, 33)):
            code = (r // 4 * hd + c) * 4 + r % 4 if is_v else (c // 16 * 64 + r) * 16 + c % 16
            s = 64 * hd + 2 * (c // 32 * 64 + r if is_v else r * (hd // 32) + c // 32)
            d = t[p, h, s:s + 2].copy().view(np.float16)[0]
            assert float(t[p, h, code].view(np.int8)) * float(d) == want[p, h, r, c]


def test_plain_attention_is_softmax(lrs):
    """The 64-bit form against an independent one: all rows at once, masked."""
    rng = np.random.default_rng(5)
    n, ctx, hd = 6, 11, 64
    q = rng.standard_normal((n, 4, hd)).astype(np.float32)
    k, v = rng.standard_normal((2, 2, ctx + n, hd))
    masks = kv_plain.random_tree(rng, n)
    masks[3] = 0
    out, err = kv_plain.attention(q, k, v, ctx, masks, 0.125)
    seen = np.array([[True] * ctx + [bool(m >> j & 1) for j in range(n)] for m in masks])
    for h in range(4):
        s = np.where(seen, q[:, h].astype(np.float64) @ k[h // 2].T * 0.125, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        assert np.allclose(out[:, h], p / p.sum(1, keepdims=True) @ v[h // 2], atol=1e-13)
    assert (err > 0).all() and err.max() < 1e-2
    empty, _ = kv_plain.attention(q, k, v, 0, [0] * n, 0.125)
    assert (empty == 0).all()


# ----------------------------------------------------------- token trees -----
@pytest.mark.parametrize("parents", [[0], [-2], [-1, 1], [-1, 0, 3], [], [-1] * 65], ids=str)
def test_bad_parents_are_refused(lrs, parents):
    n = len(parents)
    with pytest.raises(lrs.LrsError) as e:
        lrs.greedy_path([1] * n, parents, [1] * n)
    assert e.value.code == INVALID


def test_tree_arguments_of_different_lengths_are_refused(lrs):
    for args in (([1, 2], [-1], [3, 3]), ([1], [-1], [3, 3])):
        with pytest.raises(lrs.LrsError):
            lrs.greedy_path(*args)


@pytest.mark.parametrize("tokens,parents,argmax,path,nxt", [
    ([5], [-1], [9], [0], 9),
    ([5, 9], [-1, 0], [9, 4], [0, 1], 4),
    ([5, 8, 9, 4], [-1, 0, 0, 2], [9, 1, 4, 7], [0, 2, 3], 7),      # the second child
    ([5, 9, 9], [-1, -1, 0], [9, 3, 2], [0, 2], 2),                 # node 1 does not follow node 0
    ([5, 9, 3, 9], [-1, 0, 1, 0], [9, 3, 6, 1], [0, 1, 2], 6),      # of two equal children the first
    ([5, 6], [-1, 0], [9, 3], [0], 9),
    (list(range(64)), list(range(-1, 63)), list(range(1, 65)), list(range(64)), 64)])
def test_greedy_path(lrs, tokens, parents, argmax, path, nxt):
    assert lrs.greedy_path(tokens, parents, argmax) == (path, nxt)
