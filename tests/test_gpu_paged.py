"""The paged key/value cache on the device against plain restatements in Python integers and 64-bit floats.

Whole numbers (block tables, slots, positions) are equal. Attention: the bound is ``paged_ref.bound`` -- one rounding of the softmax's weights and one of the
result to the cache's type, 1e-4 for the f32 parts; its logarithm 1.5e-4 + 1e-6 of its size. Append: f32 arithmetic, then one rounding to the type."""
import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200.backend import MatView
from lapid_b200.paged import Mask, PagedSpec, plan_bytes, rope_table
from tests import paged_ref as R

pytestmark = pytest.mark.gpu
BF16, F16, F32 = lp.DType.BF16, lp.DType.F16, lp.DType.F32


@pytest.fixture(scope="module")
def be():
    return lp.Backend(0)


# ---- plan
def check_plan(s):
    b, (table, slots, positions, kv, used) = s.b, s.want
    assert np.array_equal(b["table"].download().view(np.int32).reshape(table.shape), table)
    assert np.array_equal(b["slots"].download().view(np.int32)[: s.tokens], slots)
    assert np.array_equal(b["positions"].download().view(np.int32)[: s.tokens], positions)
    assert np.array_equal(b["kv"].download().view(np.int32)[: len(s.new)], kv)
    assert b["used"].download().view(np.int32)[0] == used


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("mask", [Mask.CAUSAL, Mask.CROSS])
def test_plan_of_ragged_requests(be, page, mask):
    rng = np.random.default_rng(page)
    new = [1, 0, page, page + 1, 3, 2 * page - 1, 1, 5]
    cached = [0, 7, page - 1, 0, page, page + 1, 4 * page, 3 * page - 3]
    s = R.Step(be, new, cached, page=page, mask=mask, pad=5, seed=int(rng.integers(1000))).upload()
    for _ in range(2):  # on its own result: the same again
        s.make_plan()
        be.synchronize()
        check_plan(s)


@pytest.mark.parametrize("requests", [1, 31, 1023, 1024, 1025, 2500])
def test_plan_of_many_requests(be, requests):
    """More requests than a CTA scans at once, tokens of several CTAs."""
    rng = np.random.default_rng(requests)
    new, cached = rng.integers(0, 9, requests), rng.integers(0, 70, requests)
    s = R.Step(be, new.tolist(), cached.tolist(), hq=1, hkv=1, d=16, pad=3).upload()
    s.make_plan()
    be.synchronize()
    check_plan(s)


def test_plan_of_one_long_prompt(be):
    s = R.Step(be, [5000], [0], hq=1, hkv=1, d=16, page=32).upload()
    s.make_plan()
    be.synchronize()
    check_plan(s)


def test_plan_says_when_the_free_pages_run_out(be):
    s = R.Step(be, [40, 40], [0, 0]).upload()
    table, slots, positions, kv, used = R.plan(s.new, s.cached, s.table0, s.free, 4, s.page, s.blocks, s.tokens)
    assert used == 6
    b = s.b
    be.paged_plan(s.spec, b["new"], b["cached"], b["table"], b["slots"], b["positions"], b["kv"], b["used"], b["plan"], free_pages=b["free"], n_free=4)
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "out_of_memory"
    s.want = (table, slots, positions, kv, used)
    check_plan(s)   # the pages that there were are given out all the same, the others are -1
    be.synchronize()


def test_plan_refuses_lengths_whose_sum_passes_32_bits(be):
    s = R.Step(be, [1], [4]).upload()
    spec = PagedSpec(dtype=BF16, q_heads=1, kv_heads=1, head_dim=16, page_size=16, pages=4, requests=1, tokens=4, max_blocks=4, max_new=2 ** 31 - 1)
    big = np.array([2 ** 31 - 1], np.int32)
    z = lambda n: be.upload(np.zeros(n, np.int32))
    table, used = z(4), z(1)
    be.paged_plan(spec, be.upload(big), be.upload(big), table, z(4), z(4), z(1), used, be.alloc(plan_bytes(spec)), free_pages=s.b["free"], n_free=1)
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "shape_mismatch" and not used.download().any() and not table.download().any()


@pytest.mark.parametrize("new,cached", [([1, -1, 2], [4, 4, 4]), ([1, 2, 2], [4, -3, 4]), ([1, 9, 2], [4, 4, 4]), ([1, 1, 2], [4, 1000, 4]), ([8, 8, 8], [0, 0, 0])])
def test_plan_refuses_lengths_outside_the_bounds(be, new, cached):
    s = R.Step(be, [1, 3, 2], [4, 4, 4], max_new=8).upload()
    s.b["new"].write(0, np.array(new, np.int32))
    s.b["cached"].write(0, np.array(cached, np.int32))
    s.make_plan()
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "shape_mismatch"
    be.synchronize()


# ---- append
def rotate(x, pos, table, rot, neighbours):
    x, y = x.astype(np.float64), x.astype(np.float64).copy()
    for t, p in enumerate(pos):
        if p < 0:
            continue
        c, s = table[p, : rot // 2].astype(np.float64), table[p, rot // 2:].astype(np.float64)
        i = np.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + rot // 2)
        y[t][:, a] = x[t][:, a] * c - x[t][:, b] * s
        y[t][:, b] = x[t][:, b] * c + x[t][:, a] * s
    return y


def half_bound(dtype, want, x):
    """One rounding to the type (in f16 at least half its smallest step), and 2^-22 of the pair's size for the f32 products."""
    return R.U[dtype] * np.abs(want) + (2.0 ** -25 if dtype == F16 else 0.0) + 2.0 ** -22 * (np.abs(want) + np.abs(x).max())


@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,rot,neighbours", [(4, 2, 64, 64, False), (4, 2, 64, 32, True), (6, 3, 80, 80, True), (2, 1, 128, 0, False), (40, 8, 128, 128, False), (3, 3, 16, 8, False)])
def test_append(be, src, hq, hkv, d, rot, neighbours):
    dtype = F16 if src == F16 else BF16
    s = R.Step(be, [1, 17, 0, 30], [3, 15, 4, 0], hq=hq, hkv=hkv, d=d, dtype=dtype, pad=2).upload()
    s.make_plan()
    _, slots, positions, _, _ = s.want
    rng = np.random.default_rng(5)
    host = {}
    for n, h in (("q", hq), ("k", hkv), ("v", hkv)):
        x = rng.normal(size=(s.tokens, h, d))
        host[n] = (x.astype(np.float32), x.astype(np.float32)) if src == F32 else R.to_half(x, src)
    table = rope_table(64, max(rot, 8))
    kc0, vc0 = s.b["k"].download().view(np.int16).copy(), s.b["v"].download().view(np.int16).copy()
    q_out = be.upload(np.full((s.tokens, hq, d), 0x1111, np.int16))
    be.paged_append(s.spec, src, be.upload(host["q"][1]), be.upload(host["k"][1]), be.upload(host["v"][1]), s.b["slots"], s.b["positions"], s.b["k"], s.b["v"], q_out,
                    rope=be.upload(table) if rot else None, rope_rows=64, rot=rot, neighbours=neighbours)
    be.synchronize()
    turn = lambda x: rotate(x, positions, table, rot, neighbours) if rot else x.astype(np.float64)
    got = R.from_half(q_out.download().view(np.int16), dtype).reshape(s.tokens, hq, d)
    real = positions >= 0
    q = turn(host["q"][0])
    assert np.all(np.abs(got[real] - q[real]) <= half_bound(dtype, q[real], host["q"][0]))
    assert np.all(q_out.download().view(np.int16).reshape(s.tokens, hq, d)[~real] == 0x1111)
    for name, before, x in (("k", kc0, turn(host["k"][0])), ("v", vc0, host["v"][0].astype(np.float64))):
        bits = s.b[name].download().view(np.int16).reshape(s.pages, hkv, s.page, d)
        after, touched = R.from_half(bits, dtype).reshape(bits.shape), np.zeros((s.pages, s.page), bool)
        for t in np.nonzero(real)[0]:
            pg, i = slots[t] // s.page, slots[t] % s.page
            touched[pg, i] = True
            assert np.all(np.abs(after[pg, :, i] - x[t]) <= half_bound(dtype, x[t], host[name][0]))
        assert np.array_equal(bits.transpose(0, 2, 1, 3)[~touched], before.reshape(bits.shape).transpose(0, 2, 1, 3)[~touched])


@pytest.mark.parametrize("src", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_append_from_views_of_one_fused_row(be, src, shift):
    """q, k and v as parts of one projection's row, heads apart, starting where no vector load may."""
    hq, hkv, d, tokens = 4, 2, 64, 9
    s = R.Step(be, [4, 5], [3, 15], hq=hq, hkv=hkv, d=d).upload()
    s.make_plan()
    hs = d + 2 * shift
    row = (hq + 2 * hkv) * hs + 3 * shift
    x = np.random.default_rng(shift).normal(size=(tokens + 1) * row)
    x, bits = (x.astype(np.float32), x.astype(np.float32)) if src == F32 else R.to_half(x, src)
    buf, q_out = be.upload(bits), be.alloc(tokens * hq * d * 2)
    view = lambda first: MatView(shift + first * hs, hs, row)
    be.paged_append(s.spec, src, buf, buf, buf, s.b["slots"], s.b["positions"], s.b["k"], s.b["v"], q_out, q_view=view(0), k_view=view(hq), v_view=view(hq + hkv))
    be.synchronize()
    at = lambda t, h: x[shift + t * row + h * hs:][:d].astype(np.float64)
    q = R.from_half(q_out.download().view(np.int16), BF16).reshape(tokens, hq, d)
    k = R.from_half(s.b["k"].download().view(np.int16), BF16).reshape(s.pages, hkv, s.page, d)
    v = R.from_half(s.b["v"].download().view(np.int16), BF16).reshape(s.pages, hkv, s.page, d)
    for t in range(tokens):
        pg, i = s.want[1][t] // s.page, s.want[1][t] % s.page
        for h in range(hq):
            assert np.all(np.abs(q[t, h] - at(t, h)) <= half_bound(BF16, at(t, h), x))
        for h in range(hkv):
            assert np.all(np.abs(k[pg, h, i] - at(t, hq + h)) <= half_bound(BF16, at(t, hq + h), x))
            assert np.all(np.abs(v[pg, h, i] - at(t, hq + hkv + h)) <= half_bound(BF16, at(t, hq + hkv + h), x))


def test_append_of_keys_alone_and_skipped_rows(be):
    s = R.Step(be, [3], [0], hq=2, hkv=2, d=16).upload()
    s.make_plan()
    x = np.arange(3 * 2 * 16, dtype=np.float32).reshape(3, 2, 16)
    buf = be.upload(x)
    before = R.from_half(s.b["k"].download().view(np.int16), BF16).reshape(s.pages, 2, 16, 16)
    s.b["slots"].write(0, np.array([s.want[1][0], -1, s.want[1][2]], np.int32))
    be.paged_append(s.spec, F32, None, buf, buf, s.b["slots"], s.b["positions"], s.b["k"], s.b["v"], None)
    be.synchronize()
    k = R.from_half(s.b["k"].download().view(np.int16), BF16).reshape(s.pages, 2, 16, 16)
    pg = s.want[1][0] // 16
    assert np.array_equal(k[pg, :, 0], x[0]) and np.array_equal(k[pg, :, 2], x[2]) and np.array_equal(k[pg, :, 1], before[pg, :, 1])


@pytest.mark.parametrize("slots,positions", [([5, 10 ** 6, 7], [0, 1, 2]), ([5, 6, 7], [0, 64, 2])])
def test_append_reports_slots_and_positions_outside(be, slots, positions):
    s = R.Step(be, [3], [0], hq=2, hkv=2, d=16).upload()
    x = be.upload(np.ones((3, 2, 16), np.float32))
    be.paged_append(s.spec, F32, None, x, x, be.upload(np.array(slots, np.int32)), be.upload(np.array(positions, np.int32)), s.b["k"], s.b["v"], None,
                    rope=be.upload(rope_table(64, 16)), rope_rows=64, rot=16)
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "index_out_of_range"
    be.synchronize()


# ---- attention
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 2, 128), (7, 1, 128), (2, 2, 16), (10, 2, 80), (6, 2, 96), (16, 1, 64), (20, 1, 64), (3, 3, 120), (64, 2, 64)])
def test_decode_of_one_token(be, dtype, hq, hkv, d):
    R.Step(be, [1] * 6, [0, 1, 15, 16, 63, 200], hq=hq, hkv=hkv, d=d, dtype=dtype, seed=d).run()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("cached", [[62, 63, 64, 65], [126, 127, 128, 129], [700, 1, 1500, 31]])
def test_decode_lengths_around_the_steps(be, page, cached):
    R.Step(be, [1, 1, 1, 1], cached, hq=8, hkv=2, d=128, page=page, seed=page).run()


@pytest.mark.parametrize("new", [2, 3, 4, 5])
def test_decode_of_several_tokens(be, new):
    R.Step(be, [new, 1, new, 0, new], [77, 300, 0, 50, 129], hq=8, hkv=2, d=64, seed=new).run()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 2, 128), (7, 1, 128), (5, 5, 32), (10, 2, 80), (3, 1, 96)])
@pytest.mark.parametrize("page", [16, 128])
def test_prompts(be, dtype, hq, hkv, d, page):
    """Whole prompts of ragged lengths around the tile's."""
    R.Step(be, [130, 1, 64, 257, 33], [0] * 5, hq=hq, hkv=hkv, d=d, dtype=dtype, page=page, seed=d).run()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,cached", [([70], [300]), ([33, 1, 90], [127, 255, 128]), ([65, 64, 63], [129, 1, 640]), ([300], [5])])
def test_chunks_behind_a_context(be, page, new, cached):
    R.Step(be, new, cached, hq=8, hkv=2, d=128, page=page, seed=len(new)).run()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,d,new,cached", [(8, 8, 128, [900, 1400], [0, 300]), (16, 8, 64, [1, 1500, 700, 60], [50, 0, 900, 2000]), (24, 8, 128, [1300, 40], [77, 1500])])
def test_many_steps_a_cta(be, dtype, hq, hkv, d, new, cached):
    """Enough work that each SM walks several tiles and every ring several times (checked on rows picked at random)."""
    s = R.Step(be, new, cached, hq=hq, hkv=hkv, d=d, dtype=dtype, page=32, seed=d).upload()
    s.make_plan()
    s.attend()
    be.synchronize()
    out, lse = s.outputs()
    rng, at = np.random.default_rng(3), 0
    for r, n in enumerate(new):
        for t in {0, n - 1, *rng.integers(0, n, 12).tolist()}:
            end = cached[r] + t + 1
            o, l, size = R.attention(s.q[at + t:at + t + 1], s.k[r][:end], s.v[r][:end], s.g, s.mask, 0, s.scale, 1, end)
            assert np.all(np.abs(out[at + t] - o[0]) <= R.bound(dtype, o[0], size[0], end, 6.0)), (r, t)
            assert np.all(np.abs(lse[at + t] - l[0]) <= 1.5e-4 + 1e-6 * np.abs(l[0])), (r, t)
        at += n
    first = s.b["out"].download().copy()
    s.attend()
    be.synchronize()
    assert np.array_equal(first, s.b["out"].download())


@pytest.mark.parametrize("window", [1, 17, 64, 128, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_sliding_window(be, window, d):
    R.Step(be, [150, 1, 4, 300, 1], [100, 500, 129, 0, 3], hq=6, hkv=2, d=d, window=window, seed=window).run()


@pytest.mark.parametrize("mask", [Mask.FULL, Mask.CROSS])
def test_other_masks_and_requests_without_keys(be, mask):
    """CROSS with nothing cached: rows that no key is left to are 0, the logarithm of their sum -inf."""
    s = R.Step(be, [5, 1, 100, 1, 70], [300, 0, 0, 65, 129], hq=8, hkv=2, d=64, mask=mask).run()
    if mask == Mask.CROSS:
        out, lse = s.outputs()
        assert not out[5:106].any() and np.all(np.isneginf(lse[5:106]))


def test_mixed_step_and_rows_behind_the_sum(be):
    s = R.Step(be, [1, 1, 200, 1, 3, 0, 1], [1000, 31, 64, 0, 500, 9, 2000], hq=8, hkv=2, d=128, pad=7).run()
    raw = s.b["out"].download().view(np.int16).reshape(s.tokens, -1)
    assert np.all(raw[sum(s.new):] == 0x7e7e) and np.all(s.outputs()[1][sum(s.new):] == 77.0)


def test_no_tokens_at_all(be):
    s = R.Step(be, [0, 0], [5, 0]).upload()
    s.make_plan()
    s.attend()
    be.synchronize()


@pytest.mark.parametrize("new,cached,hq,hkv", [([1], [9000], 4, 1), ([1, 1], [6000, 3000], 8, 2), ([40], [9000], 4, 1), ([300, 1], [2000, 8000], 4, 1)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_rows_over_many_keys_are_split_and_joined(be, new, cached, hq, hkv, dtype):
    s = R.Step(be, new, cached, hq=hq, hkv=hkv, d=64, dtype=dtype, page=64).run()
    first = s.b["out"].download().copy()
    for _ in range(3):  # the joins do not depend on which CTA comes last
        s.attend()
        be.synchronize()
        assert np.array_equal(first, s.b["out"].download())


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("spread", [3.0, 6.0])
def test_scores_that_grow_along_the_keys(be, new, spread):
    """Large scores: the running maximum moves again and again, weights span the type's whole range."""
    s = R.Step(be, [new, new], [700, 90], hq=4, hkv=2, d=64, spread=spread)
    for k in s.k:
        k *= np.linspace(0.0, 1.0, k.shape[0])[:, None, None]
        k[:] = R.to_half(k, s.dtype)[0]
    # scores of this size round by more than the bound's 1e-4: d products of f32 sums
    s.upload()
    s.make_plan()
    s.attend()
    be.synchronize()
    out, _ = s.outputs()
    at = 0
    for r, n in enumerate(s.new):
        o, l, size = R.attention(s.q[at:at + n], s.k[r], s.v[r], s.g, s.mask, s.window, s.scale, n, s.kv[r])
        top = float(np.abs(s.q).max() * np.abs(s.k[r]).max()) * s.d * s.scale   # no score is larger
        rounding = 2 * (s.d + 4) * 2.0 ** -24 * top
        vmax = float(np.abs(s.v[r]).max())
        assert np.all(np.abs(out[at:at + n] - o) <= R.bound(s.dtype, o, size, s.kv[r], vmax) + rounding * vmax)
        at += n


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [0.01, 1.0, -0.3])
def test_other_scales(be, new, scale):
    R.Step(be, [new], [200], hq=4, hkv=2, d=64, scale=scale).run()


def test_nan_and_inf_stay_in_their_rows(be):
    """A NaN in one row's q reaches that row alone; an infinite value in v the rows that see it, and at most those of their tile (the token in front of it here);
    what lies behind the keys of a tile reaches none."""
    s = R.Step(be, [130, 1], [20, 60], hq=4, hkv=2, d=64)
    s.q[7, 1, 3] = np.nan
    s.q_bits = R.to_half(s.q, s.dtype)[1]
    s.v[0][149] = np.inf   # the last new token's: causally, it alone sees it
    s.k[0][149] = 0.0
    s.upload()
    s.make_plan()
    s.attend()
    be.synchronize()
    out, lse = s.outputs()
    bad = np.zeros((131, 4), bool)
    bad[7, 1] = True
    bad[128:130] = True
    assert np.all(np.isnan(out[7, 1])) and np.isnan(lse[7, 1])
    assert np.all(np.isinf(out[129]))
    o, l, size = R.attention(s.q[:130], s.k[0], np.where(np.isinf(s.v[0]), 0.0, s.v[0]), s.g, s.mask, 0, s.scale, 130, 150)
    ok = ~bad[:130]
    assert np.all(np.abs(out[:130][ok] - o[ok]) <= R.bound(s.dtype, o[ok], size[ok], 150, 6.0))
    o, l, size = R.attention(s.q[130:], s.k[1], s.v[1], s.g, s.mask, 0, s.scale, 1, 61)
    assert np.all(np.abs(out[130:] - o) <= R.bound(s.dtype, o, size, 61, 6.0))


@pytest.mark.parametrize("new", [[1, 1, 2], [100, 1, 30]])
@pytest.mark.parametrize("shift", [0, 3, 8])
def test_q_and_out_through_views(be, new, shift):
    """Heads apart and token-major, head-major, and starts where no vector access may."""
    s = R.Step(be, new, [40, 100, 0], hq=6, hkv=2, d=64).upload()
    s.make_plan()
    t, hs = s.tokens, 64 + shift
    for head, token in ((hs, 6 * hs + shift), (t * hs, hs)):
        size = shift + 6 * t * hs + 7 * shift * t + 64
        host = np.zeros(size, np.int16)
        index = shift + np.arange(t)[:, None, None] * token + np.arange(6)[None, :, None] * head + np.arange(64)[None, None, :]
        host[index] = s.q_bits
        q, out = be.upload(host), be.upload(np.full(size, 0x1234, np.int16))
        be.paged_attention(s.spec, s.b["plan"], q, s.b["k"], s.b["v"], s.b["table"], out, lse=s.b["lse"], q_view=MatView(shift, head, token), out_view=MatView(shift, head, token))
        be.synchronize()
        bits = out.download().view(np.int16)
        s.check((R.from_half(bits[index], s.dtype).reshape(t, 6, 64), s.outputs()[1]))
        rest = np.ones(size, bool)
        rest[index] = False
        assert np.all(bits[rest] == 0x1234)


@pytest.mark.parametrize("new", [1, 90])
def test_pages_outside_the_cache_are_reported_and_not_read(be, new):
    s = R.Step(be, [new, new], [100, 100], hq=4, hkv=2, d=64).upload()
    s.make_plan()
    be.synchronize()
    table = s.want[0].copy()
    for bad in (-1, s.pages, 2 ** 31 - 1):
        table[1, 2] = bad
        s.b["table"].write(0, table)
        s.attend()
        with pytest.raises(lp.LapidError) as e:
            be.synchronize()
        assert e.value.code == "index_out_of_range"
    s.b["table"].write(0, s.want[0])
    s.attend()
    be.synchronize()
    s.check()


def test_pages_that_no_row_sees_need_not_exist(be):
    """Behind a window the pages may have been given away."""
    s = R.Step(be, [1, 40], [500, 500], hq=4, hkv=2, d=64, window=100).upload()
    s.make_plan()
    table = s.want[0].copy()
    table[:, : (500 - 100) // 16 - 8] = -1
    s.b["table"].write(0, table)
    s.attend()
    be.synchronize()
    s.check()


def test_a_plan_for_another_step_is_refused(be):
    s, o = R.Step(be, [1, 1], [30, 30], hq=4, hkv=2).upload(), R.Step(be, [1, 1], [30, 30], hq=4, hkv=1).upload()
    o.make_plan()
    be.paged_attention(s.spec, o.b["plan"] if plan_bytes(o.spec) >= plan_bytes(s.spec) else s.b["plan"], s.b["q"], s.b["k"], s.b["v"], s.b["table"], s.b["out"])
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "invalid_launch"
    be.synchronize()


def test_offsets_beyond_32_bits(be):
    """A cache of more than 2^32 bytes, its last pages in use."""
    import torch
    pages, hkv, page, d = 70000, 4, 128, 64
    assert pages * hkv * page * d * 2 > 1 << 32
    kc, vc = (torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    new, cached = [1, 70], [140, 60]
    s = R.Step(be, new, cached, hq=8, hkv=hkv, d=d, page=page)
    s.spec = PagedSpec(dtype=BF16, q_heads=8, kv_heads=hkv, head_dim=d, page_size=page, pages=pages, requests=2, tokens=71, max_blocks=s.blocks, max_new=70)
    table = np.full((2, s.blocks), -1, np.int32)
    table[0, :2], table[1, :2] = [pages - 1, 3], [pages - 2, pages - 3]
    s.table0, s.free = table, np.zeros(1, np.int32)
    s.table0[1, 1] = -1
    s.free = np.array([pages - 3], np.int32)
    rows = {0: [pages - 1, 3], 1: [pages - 2, pages - 3]}
    for r, pgs in rows.items():
        for j in range(s.kv[r]):
            kc[pgs[j // page], :, j % page] = torch.from_numpy(s.k[r][j]).to(torch.bfloat16)
            vc[pgs[j // page], :, j % page] = torch.from_numpy(s.v[r][j]).to(torch.bfloat16)
    torch.cuda.synchronize()
    z = lambda n: be.upload(np.zeros(n, np.int32))
    s.b = {"new": be.upload(np.array(new, np.int32)), "cached": be.upload(np.array(cached, np.int32)), "table": be.upload(s.table0), "free": be.upload(s.free), "slots": z(71),
           "positions": z(71), "kv": z(2), "used": z(1), "plan": be.alloc(plan_bytes(s.spec)), "k": be.wrap_tensor(kc), "v": be.wrap_tensor(vc), "q": be.upload(s.q_bits),
           "out": be.alloc(71 * 8 * d * 2), "lse": be.alloc(71 * 8 * 4)}
    s.make_plan()
    x = be.upload(np.stack([np.concatenate([s.k[0][140:], s.k[1][60:]]), np.concatenate([s.v[0][140:], s.v[1][60:]])]).astype(np.float32))
    kc[pages - 3], vc[pages - 3] = 0, 0   # the new tokens in the last pages come through append
    torch.cuda.synchronize()
    n = 71 * hkv * d
    be.paged_append(s.spec, F32, None, x, x, s.b["slots"], s.b["positions"], s.b["k"], s.b["v"], None, v_view=MatView(n, d, hkv * d))
    s.attend()
    be.synchronize()
    s.check()


def test_on_another_stream_and_in_a_graph(be):
    """A captured step (plan, attention) replayed with other lengths."""
    import torch
    stream = torch.cuda.Stream()
    s = R.Step(be, [1, 60, 1], [40, 64, 600], hq=8, hkv=2, d=64).upload()
    be.set_stream(stream.cuda_stream)
    try:
        s.make_plan()
        s.attend()
        be.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            be.set_stream(torch.cuda.current_stream().cuda_stream)
            s.make_plan()
            s.attend()
        be.set_stream(stream.cuda_stream)
        new, cached = [1, 7, 0], [20, 113, 600]   # (lengths that need no page beyond those of the table)
        s.b["new"].write(0, np.array(new, np.int32))
        s.b["cached"].write(0, np.array(cached, np.int32))
        s.b["table"].write(0, s.want[0])
        with torch.cuda.stream(stream):
            graph.replay()
        be.synchronize()
        torch.cuda.synchronize()
        s.new, s.cached, s.kv = new, cached, [21, 120, 600]
        s.check()
    finally:
        be.set_stream(0)


def test_refusals_of_buffers(be):
    s = R.Step(be, [1, 20], [30, 30], hq=4, hkv=2, d=64).upload()
    b, small = s.b, be.alloc(16)
    other = lp.Backend(0)
    foreign = other.alloc(1 << 20)
    attend = lambda **kw: be.paged_attention(s.spec, *[kw.get(n, b[n]) for n in ("plan", "q", "k", "v", "table", "out")], lse=kw.get("lse"), q_view=kw.get("q_view"), out_view=kw.get("out_view"))
    for name in ("plan", "q", "k", "v", "table", "out", "lse"):
        for buf, code in ((small, "out_of_bounds"), (foreign, "wrong_backend")):
            with pytest.raises(lp.LapidError) as e:
                attend(**{name: buf})
            assert e.value.code == code, name
    for kw in ({"out": b["q"]}, {"out": b["k"]}, {"lse": b["out"]}):
        with pytest.raises(lp.LapidError) as e:
            attend(**kw)
        assert e.value.code == "buffer_aliasing"
    for kw in ({"q_view": MatView(1, 64, 256)}, {"q_view": MatView(1 << 61, 64, 256)}, {"out_view": MatView(0, 64, 257)}):
        with pytest.raises(lp.LapidError) as e:
            attend(**kw)
        assert e.value.code in ("out_of_bounds", "too_large")
    with pytest.raises(lp.LapidError) as e:
        attend(out_view=MatView(0, 32, 128))
    assert e.value.code == "invalid_launch"
    plan = lambda **kw: be.paged_plan(s.spec, *[kw.get(n, b[n]) for n in ("new", "cached", "table", "slots", "positions", "kv", "used", "plan")], free_pages=kw.get("free", b["free"]), n_free=kw.get("n", 3))
    for kw, code in (({"table": small}, "out_of_bounds"), ({"plan": small}, "out_of_bounds"), ({"kv": b["cached"]}, "buffer_aliasing"), ({"slots": b["positions"]}, "buffer_aliasing"),
                     ({"n": 1 << 20}, "out_of_bounds"), ({"new": foreign}, "wrong_backend")):
        with pytest.raises(lp.LapidError) as e:
            plan(**kw)
        assert e.value.code == code, kw
    append = lambda **kw: be.paged_append(s.spec, kw.get("src", BF16), *[kw.get(n, b[m]) for n, m in (("q", "q"), ("kn", "q"), ("vn", "q"), ("slots", "slots"), ("positions", "positions"), ("k", "k"), ("v", "v"))],
                                          kw.get("q_out", b["out"]), rope=kw.get("rope"), rope_rows=kw.get("rows", 0), rot=kw.get("rot", 0))
    for kw, code in (({"src": lp.DType.Q4K}, "unsupported_dtype"), ({"q": None}, "invalid_argument"), ({"rot": 64}, "invalid_argument"), ({"rope": b["plan"], "rot": 12, "rows": 4}, "invalid_launch"),
                     ({"rope": small, "rot": 64, "rows": 4}, "out_of_bounds"), ({"rope": b["plan"], "rot": 72, "rows": 4}, "invalid_launch"), ({"k": b["v"]}, "buffer_aliasing"), ({"q_out": b["q"]}, "buffer_aliasing"),
                     ({"kn": small}, "out_of_bounds"), ({"src": F32}, "out_of_bounds")):
        with pytest.raises(lp.LapidError) as e:
            append(**kw)
        assert e.value.code == code, kw


@pytest.mark.parametrize("new,cached,hq,hkv,d,mask,window", [
    ([700], [0], 16, 8, 64, Mask.CAUSAL, 0),          # spans of several tiles: a cut tile's first piece finds the second there
    ([130], [900], 64, 16, 64, Mask.CAUSAL, 0),       # tiles longer than a span: two to three pieces
    ([90, 3, 90], [700, 5, 650], 32, 8, 128, Mask.FULL, 0),
    ([400], [300], 14, 2, 64, Mask.CAUSAL, 200),
])
def test_cut_tiles_are_added_up_alike_whoever_does_it(be, new, cached, hq, hkv, d, mask, window):
    """The formula, and the same bits in every run: which CTA adds a cut tile's pieces up depends on timing, the sum's order must not."""
    s = R.Step(be, new, cached, hq=hq, hkv=hkv, d=d, mask=mask, window=window, seed=12).run()
    first = [s.b[n].download().copy() for n in ("out", "lse")]
    for _ in range(30):
        s.attend()
        be.synchronize()
        for a, n in zip(first, ("out", "lse")):
            assert np.array_equal(a, s.b[n].download())


@pytest.mark.parametrize("new,cached", [([1, 3], [10, 100]), ([20], [70])])
@pytest.mark.parametrize("hq,d", [(128, 64), (136, 64), (200, 128)])
def test_more_heads_of_a_key_head_than_a_tile_has_rows(be, new, cached, hq, d):
    R.Step(be, new, cached, hq=hq, hkv=1, d=d, seed=21).run()


@pytest.mark.parametrize("d", [16, 24, 40, 104, 120])
@pytest.mark.parametrize("new,cached", [([1, 2], [33, 0]), ([70, 1], [20, 99])])
def test_odd_head_sizes(be, d, new, cached):
    R.Step(be, new, cached, hq=6, hkv=2, d=d, dtype=F16, seed=22).run()
