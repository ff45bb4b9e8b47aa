"""Attention over the paged cache where an error would be small or far away: keys that a mask leaves out with values of any size, the logarithm of the sum by what f32 allows,
plans of more requests than one scan takes, and q alone (a step that appends nothing)."""
import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200.backend import MatView
from lapid_b200.paged import Mask, rope_table
from tests import paged_ref as R
from tests.paged_more import lse_bound

pytestmark = pytest.mark.gpu
BF16, F16, F32 = lp.DType.BF16, lp.DType.F16, lp.DType.F32


@pytest.fixture(scope="module")
def be():
    return lp.Backend(0)


@pytest.mark.parametrize("new,cached", [([50], [30]), ([130], [0]), ([3], [70])])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("why", ["causal", "window", "weight"])
def test_a_key_without_weight_adds_nothing_whatever_its_value(be, new, cached, d, why):
    """2^120 where a mask, or a score 1000 below the others, leaves a key no weight. Every 16 neighbouring keys in turn: the kernels do not treat them alike."""
    window = 12 if why == "window" else 0
    s = R.Step(be, new, cached, hq=8, hkv=2, d=d, window=window, seed=d)
    n, c, kv = new[0], cached[0], s.kv[0]
    first = {"causal": kv - min(n - 1, 16), "window": 0, "weight": 2}[why]   # (keys that the first rows, the last rows, no row takes part of)
    for key in range(first, min(first + 16, kv)):
        k, v = s.k[0].copy(), s.v[0].copy()
        v[key] = 2.0 ** 120
        s.k[0], s.v[0] = k, v
        if why == "weight":   # q's first element 16, the key's -1000 * sqrt(d) / 16; the others' 0
            s.q[:, :, 0] = 16.0
            s.q_bits = R.to_half(s.q, s.dtype)[1]
            k[:, :, 0] = 0.0
            k[key, :, 0] = R.to_half(np.array([-1000.0 / (16.0 * s.scale)]), s.dtype)[0][0]
        s.upload()
        s.make_plan()
        s.attend()
        be.synchronize()
        out, _ = s.outputs()
        v[key] = 0.0
        o, _, size = R.attention(s.q, k, v, s.g, s.mask, window, s.scale, n, kv)
        rows = [t for t in range(n) if why == "weight" or not R.seen(s.mask, window, n, kv, t)[0] <= key < R.seen(s.mask, window, n, kv, t)[1]]
        assert rows or why == "window"
        assert np.all(np.abs(out[rows] - o[rows]) <= R.bound(s.dtype, o[rows], size[rows], kv, 6.0)), key


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("new,cached", [([40], [0]), ([1, 1, 2], [0, 1, 37]), ([300], [0]), ([70, 1], [33, 200])])
def test_the_logarithm_of_the_sum_is_as_close_as_f32_allows(be, dtype, d, new, cached):
    """q and k are whole numbers, so the scores are exact. The first rows see one key, two keys, ...: there a single exponential's error stands in the result."""
    s = R.Step(be, new, cached, hq=8, hkv=2, d=d, dtype=dtype, seed=d + len(new))
    rng = np.random.default_rng(d)
    s.q = rng.integers(-2, 3, s.q.shape).astype(np.float64)
    s.q_bits = R.to_half(s.q, dtype)[1]
    s.k = [rng.integers(-2, 3, x.shape).astype(np.float64) for x in s.k]
    s.upload()
    s.make_plan()
    s.attend()
    be.synchronize()
    _, lse = s.outputs()
    at = 0
    for r, n in enumerate(new):
        _, want, _ = R.attention(s.q[at:at + n], s.k[r], s.v[r], s.g, s.mask, 0, s.scale, n, s.kv[r])
        top = s.scale * max(float(np.abs(s.q[at + t, h] @ s.k[r][:, h // s.g].T).max()) for t in range(n) for h in range(s.hq))
        keys = cached[r] + 1 + np.arange(n)[:, None]
        err = np.abs(lse[at:at + n] - want)
        assert np.all(err <= lse_bound(want, top, keys)), (r, float(err.max()))
        at += n


@pytest.mark.parametrize("requests", [257, 300, 1024, 1025, 1500])
@pytest.mark.parametrize("most", [3, 30])
def test_attention_of_many_requests(be, requests, most):
    """Plans of 1024 threads, and those that take the requests in several chunks and read the cut back from the plan buffer; few rows alone, and both kinds."""
    rng = np.random.default_rng(requests + most)
    new = np.where(rng.random(requests) < 0.1, rng.integers(0, most + 1, requests), rng.integers(0, 3, requests)).tolist()
    cached = np.where(rng.random(requests) < 0.02, rng.integers(0, 400, requests), rng.integers(0, 40, requests)).tolist()
    new[requests - 1], cached[requests - 1] = most, 70
    s = R.Step(be, new, cached, hq=2, hkv=1, d=16, seed=most, pad=2).run()
    first = s.b["out"].download().copy()
    s.attend()
    be.synchronize()
    assert np.array_equal(first, s.b["out"].download())


def test_few_rows_beside_many_read_what_was_appended_just_before(be):
    """Append and attention queued behind each other, other keys and values every time: a prompt's chunk and single tokens, whose kernels run side by side."""
    new, cached, hq, hkv, d = [1, 70, 1, 1, 2], [200, 40, 63, 31, 500], 8, 2, 64
    s = R.Step(be, new, cached, hq=hq, hkv=hkv, d=d).upload()
    rng = np.random.default_rng(7)
    sets, t = [], s.tokens
    for _ in range(6):
        k, v = rng.normal(size=(t, hkv, d)).astype(np.float32), rng.normal(size=(t, hkv, d)).astype(np.float32)
        sets.append((k, v, be.upload(k), be.upload(v), be.upload(np.zeros(t * hq * d, np.int16)), be.upload(np.zeros(t * hq, np.float32))))
    b = s.b
    be.synchronize()
    for i in range(30):
        _, _, kb, vb, out, lse = sets[i % 6]
        s.make_plan()
        be.paged_append(s.spec, F32, None, kb, vb, b["slots"], b["positions"], b["k"], b["v"], None)
        be.paged_attention(s.spec, b["plan"], b["q"], b["k"], b["v"], b["table"], out, lse=lse)
    be.synchronize()
    for k, v, _, _, out, lse in sets:
        at = 0
        for r, n in enumerate(new):
            s.k[r][cached[r]:], s.v[r][cached[r]:] = R.to_half(k[at:at + n], BF16)[0], R.to_half(v[at:at + n], BF16)[0]
            at += n
        s.check((R.from_half(out.download().view(np.int16)[: t * hq * d], BF16).reshape(t, hq, d), lse.download().view(np.float32)[: t * hq].astype(np.float64).reshape(t, hq)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("mask", [Mask.CROSS, Mask.CAUSAL])
@pytest.mark.parametrize("rot", [0, 32])
def test_q_alone(be, dtype, mask, rot):
    """From f32 projections to the attention over keys that are there already: cross attention, and a layer that reads another one's cache."""
    new, cached, hq, hkv, d = [5, 1, 40], [100, 33, 64], 8, 2, 64
    s = R.Step(be, new, cached, hq=hq, hkv=hkv, d=d, dtype=dtype, mask=mask, pad=1).upload()
    s.make_plan()
    x = np.random.default_rng(2).normal(size=(s.tokens, hq, d)).astype(np.float32)
    q_out, table = be.upload(np.full((s.tokens, hq, d), 0x1111, np.int16)), rope_table(128, 32)
    kc = s.b["k"].download().copy()
    kw = dict(rope=be.upload(table), rope_rows=128, rot=32) if rot else {}
    be.paged_append(s.spec, F32, be.upload(x), None, None, None, s.b["positions"], None, None, q_out, **kw)
    be.paged_attention(s.spec, s.b["plan"], q_out, s.b["k"], s.b["v"], s.b["table"], s.b["out"], lse=s.b["lse"])
    be.synchronize()
    assert np.array_equal(kc, s.b["k"].download())
    bits = q_out.download().view(np.int16).reshape(s.tokens, hq, d)
    assert np.all(bits[sum(new):] == 0x1111)
    want, pos = x.astype(np.float64), s.want[2]
    if rot:
        c, sn = (table[np.maximum(pos, 0)][:, i * 16:(i + 1) * 16].astype(np.float64)[:, None] for i in (0, 1))
        a, b = want[..., :16].copy(), want[..., 16:32].copy()
        want[..., :16], want[..., 16:32] = a * c - b * sn, b * c + a * sn
    got = R.from_half(bits, dtype).reshape(bits.shape)
    n = sum(new)
    assert np.all(np.abs(got[:n] - want[:n]) <= R.U[dtype] * np.abs(want[:n]) + (2.0 ** -25 if dtype == F16 else 0.0) + 2.0 ** -22 * (np.abs(want[:n]) + np.abs(x).max()))
    s.q[:n] = got[:n]
    s.check()


def test_refusals_of_an_append_of_q_alone(be):
    s = R.Step(be, [3], [20], hq=4, hkv=2, d=64).upload()
    c = R.Step(be, [3], [20], hq=4, hkv=2, d=64, mask=Mask.CROSS).upload()
    b, x = s.b, be.upload(np.zeros(3 * 4 * 64, np.float32))
    for spec, args, code in ((s.spec, (x, x, None, b["slots"], b["positions"], b["k"], b["v"], b["out"]), "invalid_argument"),
                             (s.spec, (x, None, x, b["slots"], b["positions"], b["k"], b["v"], b["out"]), "invalid_argument"),
                             (s.spec, (x, None, None, b["slots"], b["positions"], b["k"], None, b["out"]), "invalid_argument"),
                             (s.spec, (x, x, x, None, b["positions"], b["k"], b["v"], b["out"]), "invalid_argument"),
                             (s.spec, (None, None, None, b["slots"], b["positions"], None, None, None), "invalid_argument"),
                             (s.spec, (x, None, None, None, None, None, None, b["out"]), "invalid_argument"),
                             (c.spec, (x, x, x, b["slots"], b["positions"], b["k"], b["v"], b["out"]), "invalid_launch")):
        with pytest.raises(lp.LapidError) as e:
            be.paged_append(spec, F32, *args)
        assert e.value.code == code, args
    with pytest.raises(lp.LapidError) as e:
        be.paged_append(s.spec, F32, x, None, None, None, b["positions"], None, None, b["out"], q_view=MatView(1, 64, 256))
    assert e.value.code == "out_of_bounds"
