"""Refusals of the paged cache's operators on the host that keep a launch from
reaching past its arrays."""
import numpy as np
import pytest

import kv_plain
import kv_terms

from test_kv_host import A, INVALID, _cache, _Host, _trees


@pytest.mark.parametrize("ld", [-1, -256, 2 ** 63, 2 ** 62, 2 ** 46])
def test_strides_past_the_address_space_are_refused(lrs, ld):
    c, be = _cache(lrs), _Host(lrs)
    for call in (lambda: be.kv_store(c, A, A, 2, A, A, ld=ld), lambda: be.kv_load(c, A, A, 2, A, A, ld=ld),
                 lambda: be.tree_attention(c, _trees(lrs), A, A, 4, q_ld=ld),
                 lambda: be.tree_attention(c, _trees(lrs), A, A, 4, out_ld=ld)):
        with pytest.raises(lrs.LrsError, match="address space") as e:
            call()
        assert e.value.code == INVALID


def test_wide_strides_are_taken(lrs):
    """Up to the address space: the calls get as far as the null backend."""
    c, be = _cache(lrs), _Host(lrs)
    for call in (lambda: be.kv_store(c, A, A, 2, A, A, ld=2 ** 44), lambda: be.tree_attention(c, _trees(lrs), A, 2 * A, 4, q_ld=2 ** 43)):
        with pytest.raises(lrs.LrsError, match="null argument"):
            call()


@pytest.mark.parametrize("q_ld,out_ld", [(0, 1024), (1024, 0), (600, 601)])
def test_out_that_is_q_has_its_stride(lrs, q_ld, out_ld):
    with pytest.raises(lrs.LrsError, match="stride") as e:
        _Host(lrs).tree_attention(_cache(lrs), _trees(lrs), A, A, 4, q_ld=q_ld, out_ld=out_ld)
    assert e.value.code == INVALID


# ---------------------------------------------------------- products of terms --
@pytest.mark.parametrize("hd,at", [(64, 0), (64, 35), (128, 40), (128, 97)])
@pytest.mark.parametrize("before", [0, 100])
@pytest.mark.parametrize("dtype", list(kv_terms.PRODUCTS))
def test_each_case_shows_the_product_that_it_is_for(lrs, dtype, before, hd, at):
    """All products: within an eighth of the bar that the GPU test sets, which is half of
    what losing the one product does.  Every product but the largest has its case."""
    got = kv_terms.cases(dtype, hd, at)
    assert set(got) == {(part, a, b) for part in (0, 1) for a, b in kv_terms.PRODUCTS[dtype] if (a, b) != (0, 0)}
    for (part, a, b), case in got.items():
        q, k, v = kv_terms.padded(case, before, (at + 10) % hd)
        hk, hv = (kv_plain.held(lrs, lrs.KvType[dtype], x) for x in (k, v))
        assert np.array_equal(hk, k) and np.array_equal(hv, v)  # the cache holds them as they are
        want, _ = kv_plain.attention(q.reshape(1, 1, hd), hk[None], hv[None], len(k) - 1, [1], kv_terms.SCALE)
        want = want.reshape(hd)
        lost = kv_terms.emulate(dtype, q, hk, hv, *(((a, b),) if i == part else () for i in (0, 1)))
        full = kv_terms.emulate(dtype, q, hk, hv)
        effect = np.abs(lost - want)
        assert (effect > 0.25).all(), (part, a, b)
        assert (np.abs(full - want) <= effect / 16).all(), (part, a, b)
