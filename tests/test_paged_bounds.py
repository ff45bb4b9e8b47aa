"""What a plan takes of memory, without a device: sizes whose arrays of words reach 2^32 are refused, those below are counted in full."""
import pytest

import lapid_b200 as lp
from lapid_b200.paged import PagedSpec, plan_bytes

ONE = dict(dtype=lp.DType.BF16, q_heads=1, kv_heads=1, head_dim=16, page_size=16, pages=1, tokens=1, max_blocks=1, max_new=1)


@pytest.mark.parametrize("requests", [(1 << 28) + 1, 1 << 29, (1 << 30) - 2, 1 << 30, (1 << 31) - 1])
def test_more_requests_than_a_plan_has_words_for_are_refused(requests):
    with pytest.raises(lp.LapidError) as e:
        plan_bytes(PagedSpec(requests=requests, **ONE))
    assert e.value.code == "too_large"


@pytest.mark.parametrize("requests", [1 << 10, 1 << 20, 1 << 28])
def test_a_plan_has_room_for_what_it_holds_of_every_request(requests):
    """The first row, the keys and two counts of units before each request, 4 bytes each, at least."""
    assert plan_bytes(PagedSpec(requests=requests, **ONE)) >= 16 * requests
