"""Tree attention whose tiles are cut into four pieces and more: added up by the kernel for that (above 32 rows a request) and by a tile's last CTA, against the definition in 64 bits (``draft_ref``)."""
import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200 import MatView

from . import draft_ref as D
from . import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = lp.Backend(0)
    yield b
    b.close()


def pieces(s):
    """How many CTAs at least have a part of the tile with the most steps: all tiles' steps and three more for each, evenly cut over the SMs (three a CTA at least)."""
    import torch
    keys, tt = (80 if s.d > 64 else 96), 128 // s.g
    tiles = []
    for n, kv in zip(s.new, s.kv):
        low = max(0, kv - n + 1 - s.window) if s.window else 0
        tiles += [-(-(kv - max(0, n - t - 2 * tt)) // keys) - low // keys for t in range(0, n, 2 * tt)]
    units = s.hkv * sum(x + 3 for x in tiles)
    ctas = min(torch.cuda.get_device_properties(0).multi_processor_count, -(-units // 3))
    return -(-max(tiles) // -(-units // ctas))


@pytest.mark.parametrize("dtype,window", [(lp.DType.BF16, 0), (lp.DType.F16, 0), (lp.DType.F16, 1300)])
@pytest.mark.parametrize("d", [64, 72, 120, 128])
@pytest.mark.parametrize("sizes,hq,hkv", [
    ([21, 17, 2], 6, 2),   # 63 rows of 126: groups of 32 that are not full
    ([13, 5, 9], 14, 2),   # 91 of 126
    ([50], 7, 1),          # 350 rows: a tile of 36 tokens, each stream its own, and one of 14
    ([1, 100, 3], 3, 1),   # tiles of both streams beside ones of each its own
    ([5, 3, 2], 6, 2),     # 15 rows: the last CTA of a tile adds up
    ([4, 1, 4], 7, 1),     # 28
    ([2, 2, 1], 4, 1)])    # 8
def test_long_caches(be, sizes, hq, hkv, d, window, dtype):
    rng = np.random.default_rng(d + window + sizes[0])
    cached = [2000, 1500, 2600][:len(sizes)]
    s = D.TreeStep(be, [D.random_parents(rng, n, 4, 0.05) for n in sizes], cached, dtype=dtype, hq=hq, hkv=hkv, d=d, page=32, window=window, seed=sizes[0] + d, pad=1)
    assert pieces(s) >= 4
    s.run()


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("sizes", [[9, 20], [3, 2]])
@pytest.mark.parametrize("shift", [1, 3, 8])
def test_outputs_of_any_alignment(be, shift, sizes, dtype):
    rng = np.random.default_rng(shift)
    hq, d = 6, 72
    s = D.TreeStep(be, [D.random_parents(rng, n, 4) for n in sizes], [1500, 2100], dtype=dtype, hq=hq, hkv=2, d=d, seed=shift).upload()
    assert pieces(s) >= 4
    s.make_plan()
    row = hq * d + 2 * shift
    s.b["out"] = be.upload(np.full((s.tokens, row), 0x7e7e, np.int16))
    s.attend(out_view=MatView(shift, d, row))
    be.synchronize()
    raw = s.b["out"].download().view(np.int16).reshape(s.tokens, row)
    assert np.all(raw[:, :shift] == 0x7e7e) and np.all(raw[:, shift + hq * d:] == 0x7e7e)
    lse = s.b["lse"].download().view(np.float32)[: s.tokens * hq].astype(np.float64).reshape(s.tokens, hq)
    s.check((R.from_half(raw[:, shift:shift + hq * d], s.dtype).reshape(s.tokens, hq, d), lse))


@pytest.mark.parametrize("requests,most,d", [(70, 24, 128), (200, 5, 64), (300, 2, 128)])
def test_many_requests(be, requests, most, d):
    """More than there are SMs, from no token to the most, short and long."""
    rng = np.random.default_rng(requests)
    parents = [D.random_parents(rng, int(rng.integers(0, most + 1)), 3, 0.1) for _ in range(requests)]
    D.TreeStep(be, parents, [int(x) for x in 2 ** rng.uniform(0, 10, requests)], hq=4, hkv=2, d=d, seed=requests, max_new=most).run()


def test_more_requests_than_a_plan_counts_at_once(be):
    rng = np.random.default_rng(1100)
    parents = [D.random_parents(rng, int(rng.integers(0, 8)), 3, 0.1) for _ in range(1100)]
    D.TreeStep(be, parents, [int(x) for x in rng.integers(0, 40, 1100)], hq=4, hkv=1, d=32, seed=2).run()


@pytest.mark.parametrize("sizes,window", [([1, 1], 100), ([2, 1], 33), ([20, 9], 100), ([60, 37], 300)])
def test_pages_in_front_of_the_window(be, sizes, window):
    """What lies in front of the window of a request's first token is not read: its pages may be given back."""
    rng = np.random.default_rng(window)
    s = D.TreeStep(be, [D.random_parents(rng, n, 3, 0.1) for n in sizes], [900, 1333], hq=8, hkv=4, d=128, window=window, seed=window).upload()
    table = s.table0.copy()
    for r, c in enumerate(s.cached):
        table[r, : (c + 1 - window) // s.page] = -1
    s.b["table"].write(0, table)
    s.make_plan()
    s.attend()
    be.synchronize()
    s.check()
