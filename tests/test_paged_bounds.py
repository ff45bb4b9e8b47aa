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


def test_the_bound_on_the_logarithm_tells_one_polynomial_from_the_next():
    """The sum's logarithm with exponentials of degree 4 stays inside the bound, with degree 3 it does not: where a row sees one key or two, both in columns whose
    exponentials are polynomials."""
    import numpy as np

    from tests.paged_more import exp2_polynomial, lse_bound, lse_with
    rng = np.random.default_rng(1)
    share = {3: [], 4: []}
    for _ in range(200):
        s = rng.integers(-20, 21, int(rng.integers(1, 3))) / 8.0
        want = lse_with(np.exp2, s)
        for degree in share:
            share[degree].append(abs(lse_with(exp2_polynomial(degree), s) - want) / lse_bound(want, np.abs(s).max(), len(s)))
    assert max(share[4]) <= 1.0 and np.median(share[3]) > 5.0
