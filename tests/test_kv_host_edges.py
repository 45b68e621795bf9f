"""Refusals of the paged cache's operators on the host that keep a launch from
reaching past its arrays."""
import pytest

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
