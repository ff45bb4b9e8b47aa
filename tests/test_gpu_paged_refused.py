"""Requests that take no part in a step of the paged cache (lengths outside the bounds, rows behind the last one of q): they keep their rows, pages and lengths, and the
requests beside them are what they would be without the fault. Whole numbers are equal; attention by ``paged_ref.bound``."""
import dataclasses

import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200.paged import Mask
from tests import paged_ref as R
from tests.paged_more import plan_with_refusals

pytestmark = pytest.mark.gpu
F32 = lp.DType.F32


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


def want_of(s, new, cached, table, free):
    return plan_with_refusals(new, cached, table, free, s.page, s.blocks, s.spec.max_new, s.spec.tokens, s.mask == Mask.CROSS)


def check_plan(s, want):
    b, r = s.b, len(s.new)
    assert np.array_equal(i32(b["kv"], r), want[3])
    assert i32(b["used"], 1)[0] == want[4]
    assert np.array_equal(i32(b["positions"], s.spec.tokens), want[2])
    assert np.array_equal(i32(b["slots"], s.spec.tokens), want[1])
    assert np.array_equal(i32(b["table"], want[0].size).reshape(want[0].shape), want[0])


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


@pytest.mark.parametrize("bad", ["blocks", "negative"])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 2, 60, 1], [40, 70, 1, 90]])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_the_rows_of_the_others_stay_where_they_are(be, bad, new, which):
    """The rows of q belong to the requests by the new lengths; one that cannot grow any more does not hand its rows to the next."""
    s = R.Step(be, new, [20, 40, 33, 90], hq=8, hkv=2, d=64).upload()
    cached = list(s.cached)
    cached[which] = s.blocks * s.page if bad == "blocks" else -1
    s.b["cached"].write(0, np.array(cached, np.int32))
    s.make_plan()
    s.attend()
    refused(be)
    # (the pages that the refused one does not take go to the requests behind it: their new tokens' keys lie there)
    want = want_of(s, new, cached, s.table0, s.free)
    check_plan(s, want)
    kc, vc = np.full((s.pages, s.hkv, s.page, s.d), np.nan), np.full((s.pages, s.hkv, s.page, s.d), np.nan)
    for r, x in enumerate(s.kv):
        if r != which:
            for j in range(x):
                p = want[0][r, j // s.page]
                kc[p, :, j % s.page], vc[p, :, j % s.page] = s.k[r][j], s.v[r][j]
    s.b["k"].write(0, R.to_half(kc, s.dtype)[1])
    s.b["v"].write(0, R.to_half(vc, s.dtype)[1])
    s.attend()
    be.synchronize()
    out, lse = s.outputs()
    raw, at = s.b["out"].download().view(np.int16)[: s.tokens * s.hq * s.d].reshape(s.tokens, -1), 0
    for r, n in enumerate(new):
        if r == which:
            assert np.all(raw[at:at + n] == 0x7e7e) and np.all(lse[at:at + n] == 77.0)
        else:
            o, l, size = R.attention(s.q[at:at + n], s.k[r], s.v[r], s.g, s.mask, 0, s.scale, n, s.kv[r])
            assert np.all(np.abs(out[at:at + n] - o) <= R.bound(s.dtype, o, size, s.kv[r], float(np.abs(s.v[r]).max()))), r
        at += n


@pytest.mark.parametrize("tokens", [4, 5, 7, 13, 17])
@pytest.mark.parametrize("mask", [Mask.CAUSAL, Mask.CROSS])
def test_a_request_whose_rows_pass_the_last_one_is_left_out_whole(be, tokens, mask):
    """No page taken, none of its tokens stored; and a step of fewer tokens from these lengths goes on where the one before left off."""
    new, cached = [5, 0, 9, 0, 4, 17], [20, 3, 15, 0, 40, 0]
    s = R.Step(be, new, cached, mask=mask)
    s.spec = dataclasses.replace(s.spec, tokens=tokens)
    s.upload()
    s.make_plan()
    refused(be)
    want = want_of(s, new, cached, s.table0, s.free)
    assert not all(want[5])
    check_plan(s, want)
    # the next step, on the device's own results
    free, kv, table = s.free[want[4]:], want[3].tolist(), want[0]
    new = [1, 0, 2, 0, 1, 0]
    s.b["new"].write(0, np.array(new, np.int32))
    s.b["cached"].write(0, i32(s.b["kv"], 6).copy())
    s.b["free"].write(0, np.concatenate([free, np.full(want[4], -1, np.int32)]).astype(np.int32))
    s.make_plan()
    be.synchronize()
    check_plan(s, want_of(s, new, kv, table, free))


@pytest.mark.parametrize("requests", [7, 256, 257, 1024, 1500, 2100])
@pytest.mark.parametrize("mask", [Mask.CAUSAL, Mask.CROSS])
def test_plans_with_requests_that_take_no_part(be, requests, mask):
    """Some of many requests, whichever chunk of the scan they lie in, and rows that end somewhere between them."""
    rng = np.random.default_rng(requests)
    base, cached = rng.integers(0, 9, requests).tolist(), rng.integers(0, 70, requests).tolist()
    for share in (0.05, 0.5):
        s = R.Step(be, base, cached, hq=1, hkv=1, d=16, mask=mask, max_new=9)
        s.spec = dataclasses.replace(s.spec, tokens=int(sum(base) * (0.7 if share < 0.5 else 0.3)) + 1)
        s.upload()
        new, c = list(base), list(cached)
        for r in np.nonzero(rng.random(requests) < share)[0].tolist():
            what = int(rng.integers(4))
            if what == 0:
                new[r] = -3
            elif what == 1:
                new[r] = 10
            else:
                c[r] = -1 if what == 2 else s.blocks * s.page + 1
        s.b["new"].write(0, np.array(new, np.int32))
        s.b["cached"].write(0, np.array(c, np.int32))
        s.make_plan()
        want = want_of(s, new, c, s.table0, s.free)
        if all(want[5]):
            be.synchronize()
        else:
            refused(be)
        check_plan(s, want)


def test_free_pages_may_end_in_none(be):
    """A list whose length only the device knows ends in -1: out of memory, not a bad index, and the pages in front are given out."""
    s = R.Step(be, [40, 40], [0, 0]).upload()
    free = s.free.copy()
    free[4:] = -1
    s.b["free"].write(0, free)
    s.make_plan()
    refused(be, "out_of_memory")
    want = want_of(s, s.new, s.cached, s.table0, free)
    assert want[4] == 6
    check_plan(s, want)
    # such entries that no request asks for are not looked at
    s = R.Step(be, [40, 8], [0, 0]).upload()
    free = s.free.copy()
    free[4:] = -1
    s.b["free"].write(0, free)
    s.make_plan()
    be.synchronize()
    check_plan(s, want_of(s, s.new, s.cached, s.table0, free))


@pytest.mark.parametrize("slots,positions,code", [([5, -2, 7], [0, 1, 2], "index_out_of_range"), ([5, 6, 7], [0, 1, -2], "index_out_of_range"),
                                                  ([5, -2 ** 31, 7], [0, 1, 2], "index_out_of_range"), ([5, 6, 7], [0, -2 ** 31, 2], "index_out_of_range"),
                                                  ([5, -1, 7], [0, 1, -1], None)])
def test_append_reports_every_slot_and_position_outside_but_minus_one(be, slots, positions, code):
    s = R.Step(be, [3], [0], hq=2, hkv=2, d=16).upload()
    x = be.upload(np.ones((3, 2, 16), np.float32))
    before = s.b["k"].download().view(np.int16).reshape(s.pages, 2, 16, 16).copy()
    be.paged_append(s.spec, F32, None, x, x, be.upload(np.array(slots, np.int32)), be.upload(np.array(positions, np.int32)), s.b["k"], s.b["v"], None)
    if code:
        refused(be, code)
    else:
        be.synchronize()
    after = s.b["k"].download().view(np.int16).reshape(s.pages, 2, 16, 16)
    stored = [sl for sl, p in zip(slots, positions) if sl >= 0 and p >= 0]
    touched = np.zeros((s.pages, 16), bool)
    for sl in stored:
        touched[sl // 16, sl % 16] = True
    assert np.array_equal(after.transpose(0, 2, 1, 3)[~touched], before.transpose(0, 2, 1, 3)[~touched])
    assert np.all(after.transpose(0, 2, 1, 3)[touched] == R.to_half(np.ones(1), s.dtype)[1][0])
