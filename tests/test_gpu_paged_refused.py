"""Requests that take no part in a step of the paged cache (lengths outside the bounds, rows behind the last one of q): they keep their rows, pages and lengths, and the
requests beside them are what they would be without the fault. Whole numbers are equal; attention by ``paged_ref.bound``."""
import numpy as np
import pytest

import lapid_b200 as lp
from tests import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    return lp.Backend(0)


def refused(be, code="shape_mismatch"):
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == code
    be.synchronize()


def i32(buf, n):
    return buf.download().view(np.int32)[:n]


@pytest.mark.parametrize("bad", ["blocks", "negative"])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 2]])
def test_a_refused_request_keeps_its_length(be, bad, new):
    """What the next step takes as `cached_lens`: not 0, with which it would begin anew over its own pages."""
    s = R.Step(be, new, [20, 40, 33]).upload()
    cached = [20, s.blocks * s.page if bad == "blocks" else -7, 33]
    s.b["cached"].write(0, np.array(cached, np.int32))
    s.make_plan()
    refused(be)
    assert i32(s.b["kv"], 3).tolist() == [20 + new[0], cached[1], 33 + new[2]]
