"""Drafted tokens over the paged cache: tree, attention, verification and commit against the definitions in 64 bits (``draft_ref``)."""
import math

import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200.paged import Mask, PagedSpec, plan_bytes, tree_bytes

from . import draft_ref as D
from . import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = lp.Backend(0)
    yield b
    b.close()


# ------------------------------------------------------------------ tree
def chain(n):
    return list(range(-1, n - 1))


TREES = {
    "one": [[-1]], "chain33": [chain(33)], "star": [[-1] + [0] * 70], "ragged": [chain(5), [], [-1, 0, 0, 1, 1, 2, 2], [-1, -1, 0, 1, -1, 4]],
    "wide": None, "long": [chain(1024), [-1] + [0] * 9],
}


@pytest.mark.parametrize("window", [0, 1, 3, 40])
@pytest.mark.parametrize("name", sorted(TREES))
def test_tree(be, name, window):
    rng = np.random.default_rng(3)
    parents = TREES[name] or [D.random_parents(rng, int(rng.integers(0, 100)), 6, 0.1) for _ in range(300)]
    s = D.TreeStep(be, parents, [int(x) for x in rng.integers(0, 90, len(parents))], hq=1, hkv=1, d=16, window=window, pad=3).upload()
    s.make_plan()
    be.synchronize()
    got, positions, at = s.tree_rows(), s.b["positions"].download().view(np.int32), 0
    for p, c in zip(parents, s.cached):
        depth, _ = D.tree(p)
        assert np.array_equal(got[at:at + len(p)], D.tree_words(p, window, got.shape[1] - 1))
        assert list(positions[at:at + len(p)]) == [c + x for x in depth]
        at += len(p)
    assert np.all(got[at:] == 0x5a5a5a5a) and np.all(positions[at:s.tokens] == -1)


@pytest.mark.parametrize("bad", [-2, 3, 4, 1 << 30, -(1 << 31)])
def test_a_parent_out_of_range_is_reported_and_counts_as_none(be, bad):
    s = D.TreeStep(be, [[-1, 0, 1, 2, 3], [-1, 0]], [7, 0], hq=1, hkv=1, d=16).upload()
    s.b["parents"].write(4 * 3, np.array([bad], np.int32))
    s.make_plan()
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "index_out_of_range"
    assert np.array_equal(s.tree_rows()[:5], D.tree_words([-1, 0, 1, -1, 3], 0, 1)) and np.array_equal(s.tree_rows()[5:7], D.tree_words([-1, 0], 0, 1))
    assert list(s.b["positions"].download().view(np.int32)[:7]) == [7, 8, 9, 7, 8, 0, 1]


# ------------------------------------------------------------------ attention
CASES = {
    # few rows: one tile and a part of one; steps of 64 keys that end, begin and lie around the first drafted token
    "few": dict(sizes=[1, 2, 5, 8], cached=[0, 63, 64, 65], hq=2, hkv=1, d=128),
    "few_d64": dict(sizes=[3, 16, 1, 7], cached=[200, 1, 0, 130], hq=3, hkv=3, d=64, page=32),
    "few_odd": dict(sizes=[4, 3], cached=[5, 0], hq=5, hkv=1, d=24, page=128),
    # more query heads a key head than a tile of many rows has: the kernel for few rows, several tiles
    "group_200": dict(sizes=[3, 1], cached=[70, 10], hq=200, hkv=1, d=16),
    # many rows: one tile, both, several
    "many_32": dict(sizes=[8, 9, 20], cached=[0, 79, 81], hq=8, hkv=2, d=128),
    "many_d64": dict(sizes=[37, 64, 5], cached=[95, 96, 300], hq=14, hkv=2, d=64, page=32),
    "many_256": dict(sizes=[64, 100, 130], cached=[17, 0, 161], hq=8, hkv=2, d=128, page=64),
    "many_odd": dict(sizes=[33, 50], cached=[3, 64], hq=3, hkv=1, d=80),
    "alone": dict(sizes=[70, 300], cached=[1, 1], hq=1, hkv=1, d=96, page=128),
    # a tile of one token and of two, more words of ancestors than one
    "group_100": dict(sizes=[3, 1, 5], cached=[200, 0, 33], hq=100, hkv=1, d=24),
    "group_50": dict(sizes=[1, 2, 7], cached=[700, 1, 40], hq=100, hkv=2, d=64, page=64),
    "words": dict(sizes=[600, 33], cached=[70, 1500], hq=1, hkv=1, d=32),
    # few and many beside each other, a request without tokens
    "mixed": dict(sizes=[1, 40, 0, 3, 90], cached=[300, 150, 20, 0, 2], hq=4, hkv=1, d=128),
}


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("window", [0, 6, 70])
@pytest.mark.parametrize("name", sorted(CASES))
def test_attention(be, name, window, dtype):
    c = dict(CASES[name])
    rng = np.random.default_rng(len(name) + window)
    parents = [D.random_parents(rng, n, 4, 0.1) for n in c.pop("sizes")]
    D.TreeStep(be, parents, c.pop("cached"), dtype=dtype, window=window, pad=2, seed=window + 5, **c).run()


@pytest.mark.parametrize("n,hq,hkv", [(4, 4, 1), (16, 4, 1), (64, 4, 1)])
def test_long_caches_are_cut_and_joined(be, n, hq, hkv):
    rng = np.random.default_rng(n)
    D.TreeStep(be, [D.random_parents(rng, n, 3)], [7000], hq=hq, hkv=hkv, d=128, page=64, seed=n).run()


@pytest.mark.parametrize("sizes,cached,g", [([8] * 40, 400, 4), ([8] * 16, 3000, 4), ([40] * 9, 500, 4), ([64], 6000, 4), ([3, 90], 1000, 2)])
def test_the_same_bits_call_after_call(be, sizes, cached, g):
    """Whoever adds up the pieces of a cut tile, and whenever they come."""
    rng = np.random.default_rng(7)
    s = D.TreeStep(be, [D.random_parents(rng, n, 3) for n in sizes], [cached + 17 * i for i in range(len(sizes))], hq=2 * g, hkv=2, d=128, seed=3).upload()
    s.make_plan()
    s.attend()
    be.synchronize()
    first = s.b["out"].download(), s.b["lse"].download()
    for _ in range(6):
        for _ in range(25):
            s.attend()
        be.synchronize()
        assert np.array_equal(s.b["out"].download(), first[0]) and np.array_equal(s.b["lse"].download(), first[1])


@pytest.mark.parametrize("shape", ["star", "chain", "roots"])
@pytest.mark.parametrize("n", [4, 40])
def test_shapes(be, n, shape):
    parents = {"star": [-1] + [0] * (n - 1), "chain": chain(n), "roots": [-1] * n}[shape]
    D.TreeStep(be, [parents, parents], [0, 33], hq=4, hkv=2, d=64, spread=3.0).run()


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("sizes", [[1, 1, 1], [1, 3, 4], [40, 64, 7]])
def test_a_chain_is_the_causal_mask(be, sizes, dtype):
    """Both against the definition (in `run`); of single tokens, where a tree's keys are added up in the same order, bit for bit."""
    cached = [70, 0, 131]
    a = R.Step(be, sizes, cached, dtype=dtype, hq=8, hkv=2, d=128, seed=4).run()
    b = D.TreeStep(be, [chain(n) for n in sizes], cached, dtype=dtype, hq=8, hkv=2, d=128, seed=4).run()
    if max(sizes) == 1:
        assert np.array_equal(a.b["out"].download(), b.b["out"].download()) and np.array_equal(a.b["lse"].download(), b.b["lse"].download())
    assert np.array_equal(a.b["positions"].download(), b.b["positions"].download())


def test_without_lse_through_views_and_with_a_negative_scale(be):
    from lapid_b200 import MatView
    rng = np.random.default_rng(8)
    for sizes in ([3, 2], [30, 45]):
        s = D.TreeStep(be, [D.random_parents(rng, n, 3) for n in sizes], [50, 9], hq=4, hkv=2, d=64, scale=-0.2).upload()
        s.make_plan()
        t, hq, d = s.tokens, s.hq, s.d
        wide = np.zeros((t, 6 * d + 8), np.int16)
        wide[:, 8:8 + hq * d] = s.q_bits.reshape(t, -1)
        s.b["q"] = be.upload(wide)
        view = MatView(8, d, 6 * d + 8)
        s.b["out"] = be.upload(np.full((t, 6 * d + 8), 0x7e7e, np.int16))
        s.attend(lse=False, q_view=view, out_view=view)
        be.synchronize()
        raw = s.b["out"].download().view(np.int16).reshape(t, -1)
        assert np.all(raw[:, :8] == 0x7e7e) and np.all(raw[:, 8 + hq * d:] == 0x7e7e)
        s.check((R.from_half(raw[:, 8:8 + hq * d], s.dtype).reshape(t, hq, d), None), lse=False)


# ------------------------------------------------------------------ verification
class Walks:
    """Requests' logits, drafts and random numbers, on the device and as f64."""

    def __init__(self, be, parents, vocab, *, dtype=lp.DType.F32, drawn=False, temperature=1.0, seed=0, pad=0, spread=2.0, row=0, near=0.5, chain=False):
        rng = np.random.default_rng(seed)
        self.be, self.parents, self.vocab, self.chain = be, parents, vocab, chain
        self.new, r = [len(p) for p in parents], len(parents)
        t = self.tokens = sum(self.new) + pad
        row = self.row = row or vocab
        z = rng.normal(size=(t, row)) * spread
        if dtype == lp.DType.F32:
            bits = z.astype(np.float32)
            self.logits = bits.astype(np.float64)[:, :vocab]
        else:
            self.logits, bits = R.to_half(z, dtype)
            self.logits = self.logits[:, :vocab]
        self.bits, self.dtype = bits, dtype
        d = np.exp(self.logits + near * rng.normal(size=(t, vocab)))
        self.draft = (d / d.sum(1, keepdims=True)).astype(np.float32) if drawn else None
        self.tokens_of, at = np.zeros(t, np.int32), 0
        for p in parents:
            for c, v in enumerate(p):
                if v < 0:
                    continue
                if drawn:
                    self.tokens_of[at + c] = min(vocab - 1, int(np.searchsorted(np.cumsum(self.draft[at + v].astype(np.float64)), rng.random())))
                else:
                    order = np.argsort(-self.logits[at + v])
                    self.tokens_of[at + c] = order[min(vocab - 1, int(rng.integers(0, 4)))]
            at += len(p)
        self.accept, self.pick = rng.random(t).astype(np.float32), rng.random(r).astype(np.float32)
        self.accept[self.accept == 1.0], self.pick[self.pick == 1.0] = 0.5, 0.5
        self.temperature = None if temperature is None else np.broadcast_to(np.float32(temperature), (r,)).copy()

    def run(self, wait=True):
        be, r, most = self.be, len(self.new), max([1] + self.new)
        pages = max(1, sum(-(-n // 16) for n in self.new))
        spec = self.spec = PagedSpec(dtype=lp.DType.BF16, q_heads=1, kv_heads=1, head_dim=16, page_size=16, pages=pages, requests=r, tokens=self.tokens, max_blocks=-(-most // 16), max_new=most,
                                     mask=Mask.CAUSAL if self.chain else Mask.TREE)
        z = lambda n: be.upload(np.zeros(max(1, n), np.int32))
        up = lambda x: be.upload(x) if x is not None else None
        flat = np.array([p for q in self.parents for p in q] + [0] * (self.tokens - sum(self.new) + 1), np.int32)
        self.plan = be.alloc(plan_bytes(spec))
        be.paged_plan(spec, be.upload(np.array(self.new, np.int32)), z(r), z(r * spec.max_blocks), z(self.tokens), z(self.tokens), z(r), z(1), self.plan,
                      free_pages=be.upload(np.arange(pages, dtype=np.int32)), n_free=pages)
        self.path, self.accepted, self.next = (be.upload(np.full(n, 99, np.int32)) for n in (r * most, r, r))
        raw = np.concatenate([self.bits.reshape(-1), np.zeros(8, self.bits.dtype)])
        self.packed = be.packed_paged_verify(spec, self.plan, self.dtype, self.vocab, be.upload(raw), be.upload(self.tokens_of), be.upload(self.accept), be.upload(self.pick), self.path, self.accepted,
                                             self.next, parents=None if self.chain else be.upload(flat), draft=up(self.draft), temperature=up(self.temperature), logits_row=self.row)
        self.packed()
        if wait:
            be.synchronize()
        return self

    def got(self):
        r = len(self.new)
        return self.path.download().view(np.int32).reshape(r, -1), self.accepted.download().view(np.int32)[:r], self.next.download().view(np.int32)[:r]

    def want(self, r):
        at, n = sum(self.new[:r]), self.new[r]
        if n == 0:
            return [], -1
        f64 = lambda x: x[at:at + n].astype(np.float64)
        return D.verify(self.logits[at:at + n], self.parents[r], self.tokens_of[at:at + n], f64(self.accept), float(self.pick[r]), 1.0 if self.temperature is None else float(self.temperature[r]),
                        f64(self.draft) if self.draft is not None else None)

    def check(self):
        path, accepted, nxt = self.got()
        for r in range(len(self.new)):
            p, x = self.want(r)
            assert list(path[r]) == p + [-1] * (path.shape[1] - len(p)) and accepted[r] == len(p) and nxt[r] == x, (r, p, x, list(path[r]), accepted[r], nxt[r])
        return self


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("dtype", [lp.DType.F32, lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 129, 1000, 4099, 32000, 70001])
def test_verify(be, vocab, dtype, drawn):
    rng = np.random.default_rng(vocab)
    parents = [D.random_parents(rng, n, 3) for n in ([1, 2, 9, 0, 17, 5] if vocab < 30000 else [6, 3])]
    Walks(be, parents, vocab, dtype=dtype, drawn=drawn, seed=vocab + 1, pad=1, temperature=None if vocab == 31 else 0.9).run().check()


@pytest.mark.parametrize("drawn", [False, True])
def test_verify_many_requests_and_wide_trees(be, drawn):
    rng = np.random.default_rng(5)
    parents = [D.random_parents(rng, int(rng.integers(1, 12)), 4, 0.05) for _ in range(150)] + [[-1] + [0] * 40, [-1] + [0] * 9 + [9] * 9]
    w = Walks(be, parents, 300, drawn=drawn, seed=6, spread=3.0, temperature=1.3).run().check()
    assert w.got()[1].max() >= 3  # (some walks go somewhere)


@pytest.mark.parametrize("drawn", [False, True])
def test_verify_full_servers(be, drawn):
    """More requests than there are SMs, so that a CTA or two have a row and go over it many times."""
    rng = np.random.default_rng(15)
    Walks(be, [D.random_parents(rng, 3, 2) for _ in range(200)], 20011, dtype=lp.DType.F32 if drawn else lp.DType.BF16, drawn=drawn, seed=16, spread=3.0).run().check()


@pytest.mark.parametrize("vocab,dtype,drawn", [(300007, lp.DType.F32, True), (1 << 20, lp.DType.F16, False), (1 << 22, lp.DType.BF16, False)])
def test_verify_large_vocabularies(be, vocab, dtype, drawn):
    Walks(be, [[-1, 0]], vocab, dtype=dtype, drawn=drawn, seed=17).run().check()


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("row", [1000, 1001, 1003, 1004])
def test_rows_of_any_distance(be, row, drawn):
    rng = np.random.default_rng(row)
    parents = [D.random_parents(rng, 6, 2) for _ in range(5)]
    for dtype in (lp.DType.F32, lp.DType.F16):
        Walks(be, parents, 1000, dtype=dtype, drawn=drawn, seed=row, row=row).run().check()


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), 1e-38, 0.01, 100.0, float("inf")])
@pytest.mark.parametrize("drawn", [False, True])
def test_temperatures(be, temperature, drawn):
    rng = np.random.default_rng(2)
    w = Walks(be, [D.random_parents(rng, 7, 2) for _ in range(12)], 500, drawn=drawn, seed=9, temperature=temperature)
    w.logits[3:9, 40:60] = -np.inf   # tokens that are never taken
    w.bits[3:9, 40:60] = -np.inf
    w.logits[5, [7, 300]] = 50.0     # the first of the largest
    w.bits[5, [7, 300]] = 50.0
    w.run().check()


@pytest.mark.parametrize("dtype", [lp.DType.F32, lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("requests,vocab", [(1, 300), (1, 4099), (200, 4099), (1, 32000), (40, 32000), (1, 70001)])
def test_the_first_of_two_zeros_whatever_their_signs(be, requests, vocab, drawn, dtype):
    """At temperature 0 the largest logit is a zero: -0.0 and 0.0 are equal, and the first one is taken, in whichever warps or CTAs of the request they lie."""
    w = Walks(be, [[-1, 0, 0, 1] for _ in range(requests)], vocab, dtype=dtype, drawn=drawn, seed=vocab, temperature=0.0)
    w.logits[:] = w.logits - 20.0 - np.abs(w.logits)
    at = np.array([3, vocab // 5, vocab // 2, vocab - 2])
    signs = np.array([[-1, 1, -1, 1], [1, -1, 1, -1], [-1, -1, -1, 1], [-1, 1, 1, 1]])
    for t in range(w.tokens):
        first = t // 4 % 4
        w.logits[t, at[first:]] = np.copysign(0.0, signs[t % 4][first:])
    if dtype == lp.DType.F32:
        w.bits = w.logits.astype(np.float32)
    else:
        w.logits, w.bits = R.to_half(w.logits, dtype)
    w.logits = w.logits + 0.0  # (the definition's: one zero)
    w.tokens_of[:] = at[np.arange(w.tokens) % 4]
    for r in range(requests):  # children of the first node: the second of the zeros, then the first
        first = r % 4
        w.tokens_of[4 * r + 1], w.tokens_of[4 * r + 2] = at[min(first + 1, 3)], at[first]
    w.run().check()


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("scale,temperature", [(1e5, 1e-4), (1e5, 2e-5), (-3e4, 5e-5), (1e30, 1.0), (65504.0, 0.3)])
def test_large_logits_at_low_temperatures(be, scale, temperature, drawn):
    """Neighbouring numbers are many times T apart: a weight whose exponent is past what 64 bits hold is 0."""
    rng = np.random.default_rng(3)
    w = Walks(be, [D.random_parents(rng, 5, 2) for _ in range(6)], 333, drawn=drawn, seed=19, temperature=temperature)
    step = np.spacing(np.float32(abs(scale))).astype(np.float64)
    w.bits[:] = (scale - step * rng.integers(0, 15, w.bits.shape)).astype(np.float32)
    w.logits = w.bits.astype(np.float64)
    w.pick[:] = 0.3 + 0.1 * np.arange(6)
    w.run().check()


def test_a_chain_without_parents(be):
    for drawn in (False, True):
        Walks(be, [chain(n) for n in (1, 4, 0, 9)], 777, drawn=drawn, seed=3, near=0.2, chain=True).run().check()


def test_the_longest_walk(be):
    """1024 drafted tokens that are all accepted, and as many children of one token of which the last is."""
    w = Walks(be, [chain(1024), [-1] + [0] * 1023], 1025, seed=1)
    w.accept[:] = 0.0
    at = 1024
    w.tokens_of[at + 1:] = np.arange(1, 1024)
    w.accept[at + 1: 2 * at - 1] = np.float32(1 - 2.0 ** -24)
    w.run()
    path, accepted, _ = w.got()
    assert accepted[0] == 1024 and list(path[0]) == list(range(1024))
    assert accepted[1] == 2 and list(path[1][:3]) == [0, 1023, -1]
    w.check()


@pytest.mark.parametrize("pick", [0.0, float(np.float32(1 - 2.0 ** -24)), 0.5])
@pytest.mark.parametrize("drawn", [False, True])
def test_ends_of_the_random_numbers(be, drawn, pick):
    for accept in (0.0, float(np.float32(1 - 2.0 ** -24))):
        w = Walks(be, [[-1, 0, 0, 1, 2], [-1], [-1, 0, 1]], 130, drawn=drawn, seed=4)
        w.accept[:], w.pick[:] = accept, pick
        w.run().check()


def test_what_remains_is_small(be):
    """Candidates that have nearly all of the probability and fail: what is left must not be lost in a difference."""
    v = 2000
    w = Walks(be, [[-1, 0, 0, 0]], v, seed=8, spread=0.5)
    big = np.float32(1 - 2.0 ** -24)
    z = np.full(v, -30.0)
    z[[5, 900, 1999]] = [20.0, 4.0, -12.0]  # 1 - 1.2e-7, 1e-7, 1e-14: each nearly all of what the ones before it leave
    z[:5] = -29.0
    w.bits[0], w.logits[0] = z, z.astype(np.float32).astype(np.float64)
    w.tokens_of[:] = [0, 5, 900, 1999]
    w.accept[:] = big
    for pick in (0.0, 0.3, 0.999):
        w.pick[:] = pick
        w.run()
        p, x = w.want(0)
        assert p == [0] or len(p) == 2
        w.check()


def test_siblings_with_the_same_token(be):
    for drawn in (False, True):
        for accept in (0.2, 0.99):
            w = Walks(be, [[-1, 0, 0, 0, 0, 3]], 40, drawn=drawn, seed=11)
            w.tokens_of[:] = [0, 7, 7, 7, 9, 1]
            w.accept[:] = accept
            w.run().check()


def test_a_draft_that_is_the_model(be):
    """D = P but for f32: nearly all is accepted, and what is left of P is rounding (or nothing, and then P stays)."""
    w = Walks(be, [chain(6) for _ in range(40)], 257, drawn=True, seed=12, near=0.0)
    w.run()
    path, accepted, nxt = w.got()
    assert accepted.min() == 6 and (nxt >= 0).all()


def test_borders_of_what_a_rejected_draft_leaves(be):
    """The draft is the model but for the rounding to 32 bits: a hundred millionth of the probability is left, and an error of a weight counts a hundred million times as much. The numbers drawn are the f32 ones next to
    the borders between the tokens of what is left, outside of what arithmetic of 64 bits allows. With u = 2^-53 and m the mean of x: a weight e^-x is off by x u (log2(e) / T is rounded once where T is 1) and 8 u (the
    series 4 u, its last sum, the table and the product 1 u each, what is before them less than one); their sum by (m + 8) u, and 10 u for at most ten additions; the differences, relative to all probability, by the
    sum of the two; a border is a quotient of two sums of these, so twice that over what is left, and 40 u for the additions."""
    u, vocab, each = 2.0 ** -53, 40, []
    rng = np.random.default_rng(31)
    while len(each) < 1000:
        # the largest logit apart, half of the probability; the others half a step of the table of 16 below one another's places
        z = (-(rng.integers(70, 110, vocab) + 0.49) * math.log(2) / 16).astype(np.float32)
        x, top = (int(i) for i in rng.choice(vocab, 2, replace=False))
        z[top] = 0.0
        low = z.astype(np.longdouble)
        p = np.exp(low)
        p /= p.sum()
        d = p.astype(np.float64).astype(np.float32)
        d[x] = d[x] * np.float32(1 + 2.0 ** -21)  # (the drafted token: rejected by any number near 1)
        left = np.maximum(p - d.astype(np.longdouble), 0)
        all_left = left.sum()
        border = np.cumsum(left) / all_left
        m = float(-(p * low).sum())
        slack = (2 * (2 * (m + 8) + 10) * u) / float(all_left) + 40 * u
        for b in border[left > 0][:-1]:
            for side in (-1, 1):
                pick = np.float32(b + side * slack)
                while side * (np.longdouble(pick) - b) < slack:
                    pick = np.nextafter(pick, np.float32(side))
                if 0 < pick < 1 and np.abs(border - np.longdouble(pick)).min() >= slack:
                    each.append((z, d, x, pick, int(np.nonzero(border > np.longdouble(pick))[0][0])))
    w = Walks(be, [[-1, 0] for _ in each], vocab, drawn=True, seed=1)
    want = []
    for r, (z, d, x, pick, token) in enumerate(each):
        w.bits[2 * r], w.draft[2 * r], w.tokens_of[2 * r + 1], w.pick[r] = z, d, x, pick
        want.append(token)
    w.accept[:] = np.float32(1 - 2.0 ** -24)
    path, accepted, nxt = w.run().got()
    assert np.all(accepted == 1) and np.array_equal(nxt, want)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), "none"])
def test_rows_that_are_no_distribution(be, value):
    w = Walks(be, [chain(4), chain(3), [-1, 0, 0]], 600, seed=2)
    w.accept[:] = 0.0
    if value == "none":
        w.bits[2], w.logits[2] = -np.inf, -np.inf
    else:
        w.bits[2, 577] = value
        w.logits[2, 577] = value
    w.run(wait=False)
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "invalid_argument"
    w.check()
    path, accepted, nxt = w.got()
    assert accepted[0] == 3 and nxt[0] == -1 and nxt[1] >= 0
    be.synchronize()  # reported once


@pytest.mark.parametrize("token", [-1, 600, 1 << 30])
def test_a_token_outside_the_vocabulary(be, token):
    w = Walks(be, [[-1, 0, 0, 2], [-1, 0]], 600, seed=2)
    w.accept[:] = 0.0
    w.tokens_of[1] = token
    w.run(wait=False)
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "index_out_of_range"
    w.check()
    assert w.got()[0][0].tolist()[:3] == [0, 2, 3]


def test_random_numbers_that_are_none_stay_in_range(be):
    for bad in (1.0, 2.0, float("nan"), -1.0):
        for drawn in (False, True):
            w = Walks(be, [D.random_parents(np.random.default_rng(1), 8, 3) for _ in range(9)], 300, drawn=drawn, seed=3)
            w.accept[:], w.pick[:] = bad, bad
            w.run()
            path, accepted, nxt = w.got()
            assert accepted.min() >= 1 and accepted.max() <= 8 and (nxt >= 0).all() and (nxt < 300).all() and path.max() < 8


@pytest.mark.parametrize("drawn", [False, True])
def test_tokens_are_distributed_as_the_models(be, drawn):
    """The first token that a walk gives, over 6000 requests of one distribution: within 5 standard deviations of 6000 P (a normal's 1.2e-6 for 2 x 24 counts; the numbers are seeded)."""
    rng = np.random.default_rng(21)
    r, vocab = 6000, 24
    w = Walks(be, [[-1, 0, 0] for _ in range(r)], vocab, drawn=drawn, seed=22, near=1.0)
    w.bits[:], w.logits[:] = w.bits[0], w.logits[0]
    if drawn:
        w.draft[:] = w.draft[0]
        drawn_tokens = rng.choice(vocab, size=3 * r, p=w.draft[0].astype(np.float64) / w.draft[0].astype(np.float64).sum())
        w.tokens_of[:] = drawn_tokens
    w.run()
    path, accepted, nxt = w.got()
    first = np.where(accepted > 1, w.tokens_of.reshape(r, 3)[np.arange(r), np.maximum(path[:, 1], 0)], nxt)
    p = np.exp(w.logits[0] - w.logits[0].max())
    p /= p.sum()
    count = np.bincount(first, minlength=vocab)
    assert np.all(np.abs(count - r * p) <= 5 * np.sqrt(r * p * (1 - p)) + 1)


# ------------------------------------------------------------------ commit
class Kept:
    """A step whose accepted paths are given: caches of random bits, and what is to be in them."""

    def __init__(self, be, new, cached, accepted, path, *, hkv=2, d=64, page=16, caches=4, dtype=lp.DType.BF16, seed=0, mask=Mask.TREE, max_new=None):
        rng = np.random.default_rng(seed)
        self.be, self.new, self.cached, self.accepted, self.path_of, self.page = be, new, cached, accepted, path, page
        r, most = len(new), max_new or max([1] + new)
        blocks = max(1, max(-(-(c + n) // page) for n, c in zip(new, cached)))
        pages = r * blocks + 2
        order = rng.permutation(pages).astype(np.int32)
        table, at = np.full((r, blocks), -1, np.int32), 0
        for i, c in enumerate(cached):
            have = -(-c // page)
            table[i, :have] = order[at:at + have]
            at += have
        self.free = np.concatenate([order[at:], np.full(3, -1, np.int32)])
        self.spec = PagedSpec(dtype=dtype, q_heads=hkv, kv_heads=hkv, head_dim=d, page_size=page, pages=pages, requests=r, tokens=sum(new) + 1, max_blocks=blocks, max_new=most, mask=mask)
        up, z = be.upload, lambda n: be.upload(np.zeros(max(1, n), np.int32))
        self.b = {"table": up(table), "free": up(self.free), "kv": z(r), "used": z(1), "plan": be.alloc(plan_bytes(self.spec)), "accepted": up(np.array(accepted, np.int32))}
        full = np.full((r, most), -1, np.int32)
        for i, p in enumerate(path or []):
            full[i, :len(p)] = p
        self.b["path"] = up(full) if path is not None else None
        self.before = [rng.integers(-30000, 30000, (pages, hkv, page, d)).astype(np.int16) for _ in range(caches)]
        self.caches = [up(x) for x in self.before]
        be.paged_plan(self.spec, up(np.array(new, np.int32)), up(np.array(cached, np.int32)), self.b["table"], z(sum(new) + 1), z(sum(new) + 1), self.b["kv"], self.b["used"], self.b["plan"],
                      free_pages=self.b["free"], n_free=len(self.free))
        be.synchronize()
        self.table = self.b["table"].download().view(np.int32)[: r * blocks].reshape(r, blocks)

    def layers(self):
        return [(self.caches[i], self.caches[i + 1]) for i in range(0, len(self.caches), 2)]

    def commit(self):
        b = self.b
        self.be.paged_commit(self.spec, b["plan"], self.layers(), b["table"], b["path"], b["accepted"], b["kv"], b["used"], free_pages=b["free"], n_free=len(self.free))

    def check(self, accepted=None):
        accepted = self.accepted if accepted is None else accepted
        path = self.path_of or [list(range(a)) for a in accepted]
        moves, kv, used, free = D.commit(self.new, self.cached, self.table, accepted, path, self.free, self.page)
        at = lambda r, x: (self.table[r, x // self.page], x % self.page)
        for x, buf in zip(self.before, self.caches):
            want = x.copy()
            rows = [x[at(r, a)[0], :, at(r, a)[1]].copy() for r, a, _ in moves]
            for row, (r, _, c) in zip(rows, moves):
                want[at(r, c)[0], :, at(r, c)[1]] = row
            assert np.array_equal(buf.download().view(np.int16).reshape(want.shape), want)
        assert list(self.b["kv"].download().view(np.int32)[: len(kv)]) == kv
        assert int(self.b["used"].download().view(np.int32)[0]) == used
        assert list(self.b["free"].download().view(np.int32)[: len(free)]) == [int(x) for x in free]
        assert np.array_equal(self.b["table"].download().view(np.int32)[: self.table.size], self.table.reshape(-1))


def paths(rng, new):
    out = []
    for n in new:
        k = int(rng.integers(0, n + 1))
        rest = sorted(rng.choice(np.arange(1, n), size=min(max(0, k - 1), n - 1), replace=False).tolist()) if n > 1 else []
        out.append(([0] + rest) if k else [])
    return out


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("new,cached,kw", [
    ([5, 1, 0, 9], [3, 16, 7, 0], {}), ([40, 33, 17, 64], [15, 16, 17, 0], {"page": 32}), ([3, 2], [100, 31], {"hkv": 1, "d": 16, "page": 128}), ([7, 20], [1, 2], {"hkv": 5, "d": 80}),
    ([1023, 1024], [9, 0], {"hkv": 1, "d": 24}), ([12, 6], [4, 60], {"hkv": 8, "d": 128, "page": 64, "caches": 2})])
def test_commit(be, new, cached, kw, dtype):
    for seed in range(3):
        path = paths(np.random.default_rng(seed), new)
        k = Kept(be, new, cached, [len(p) for p in path], path, seed=seed, dtype=dtype, **kw)
        k.commit()
        be.synchronize()
        k.check()


@pytest.mark.parametrize("requests", [127, 128, 129, 700])
def test_commit_of_many_requests(be, requests):
    rng = np.random.default_rng(requests)
    new, cached = rng.integers(0, 40, requests).tolist(), rng.integers(0, 50, requests).tolist()
    path = paths(rng, new)
    k = Kept(be, new, cached, [len(p) for p in path], path, hkv=1, d=16, caches=2)
    k.commit()
    be.synchronize()
    k.check()


def test_commit_of_more_caches_than_a_launch_takes(be):
    path = [[0, 2, 3, 7], [0, 1, 5]]
    k = Kept(be, [8, 6], [5, 14], [4, 3], path, hkv=1, d=16, caches=600)
    k.commit()
    be.synchronize()
    k.check()


def test_commit_of_chains_and_without_caches(be):
    k = Kept(be, [5, 33, 16], [15, 1, 0], [2, 17, 0], None, mask=Mask.CAUSAL)
    k.commit()
    be.synchronize()
    k.check()
    k = Kept(be, [5, 4], [15, 1], [2, 3], [[0, 4], [0, 1, 3]], caches=0)
    k.commit()
    be.synchronize()
    k.check()


def test_commit_of_more_requests_than_a_grid_is_high(be):
    rng = np.random.default_rng(70)
    new, cached = rng.integers(0, 4, 70000).tolist(), rng.integers(0, 13, 70000).tolist()
    path = paths(rng, new)
    k = Kept(be, new, cached, [len(p) for p in path], path, hkv=1, d=16, caches=2)
    k.commit()
    be.synchronize()
    k.check()


def test_commit_of_long_chains(be):
    """Without a path there is no largest number of new tokens."""
    k = Kept(be, [2000, 1500, 0], [30, 0, 5], [1999, 3, 0], None, mask=Mask.CAUSAL)
    k.commit()
    be.synchronize()
    k.check()


@pytest.mark.parametrize("ends", ["list", "entries"])
@pytest.mark.parametrize("requests", [5, 128, 300])
def test_a_step_whose_pages_ran_out_keeps_nothing(be, requests, ends):
    """Plan and commit may lie in one graph: where the pages ran out, lengths and list stay, so that the step can be run again."""
    rng = np.random.default_rng(requests)
    new, cached = rng.integers(1, 40, requests).tolist(), rng.integers(0, 50, requests).tolist()
    path = paths(rng, new)
    k = Kept(be, new, cached, [len(p) for p in path], path, hkv=1, d=16, caches=2)
    taken = int(k.b["used"].download().view(np.int32)[0])
    lens, z = [be.upload(np.array(x, np.int32)) for x in (new, cached)], [be.upload(np.zeros(sum(new) + 1, np.int32)) for _ in range(2)]
    plan = lambda free, n: be.paged_plan(k.spec, *lens, k.b["table"], *z, k.b["kv"], k.b["used"], k.b["plan"], free_pages=free, n_free=n)
    few = k.free[:taken - 2] if ends == "list" else np.concatenate([k.free[:taken - 2], np.full(9, -1, np.int32)])
    short = be.upload(few)
    plan(short, len(few))
    be.paged_commit(k.spec, k.b["plan"], k.layers(), k.b["table"], k.b["path"], k.b["accepted"], k.b["kv"], k.b["used"], free_pages=short, n_free=len(few))
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "out_of_memory"
    assert k.b["kv"].download().view(np.int32)[:requests].tolist() == cached
    assert int(k.b["used"].download().view(np.int32)[0]) == 0
    assert np.array_equal(short.download().view(np.int32)[:len(few)], few)
    k.before = [c.download().view(np.int16)[: x.size].reshape(x.shape).copy() for c, x in zip(k.caches, k.before)]  # (what lies behind the cached tokens may have moved)
    plan(k.b["free"], len(k.free))
    k.commit()
    be.synchronize()
    k.check()


@pytest.mark.parametrize("accepted,path", [([3, 2], [[0, 2, 2], [0, 1]]), ([3, 2], [[0, 3, 2], [0, 1]]), ([2, 2], [[0, 5], [0, 1]]), ([2, 2], [[-1, 1], [0, 1]]), ([6, 2], [[0, 1, 2, 3, 4], [0, 1]]),
                                           ([-1, 2], [[], [0, 1]]), ([1 << 30, 2], [[], [0, 1]])])
def test_a_path_that_is_none_keeps_nothing(be, accepted, path):
    k = Kept(be, [5, 20], [14, 3], accepted, path)
    k.commit()
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "index_out_of_range"
    k.path_of = [[], path[1]]
    k.check([0, accepted[1]])


def test_a_plan_of_another_description_is_refused_by_all(be):
    from dataclasses import replace
    s = D.TreeStep(be, [[-1, 0, 0]], [4], hq=4, hkv=2, d=64).upload()
    s.make_plan()
    be.synchronize()
    other = replace(s.spec, max_new=2)
    b, z = s.b, lambda n: be.upload(np.zeros(n, np.int32))
    rows, one = be.upload(np.full(64, 7, np.int32)), z(16)
    outs = [z(16) for _ in range(4)]
    calls = [lambda: be.paged_tree(other, b["plan"], b["parents"], rows, b["tree"]),
             lambda: be.paged_tree_attention(other, b["plan"], b["tree"], b["q"], b["k"], b["v"], b["table"], b["out"]),
             lambda: be.paged_commit(other, b["plan"], [(b["k"], b["v"])], b["table"], one, one, outs[0], outs[1]),
             lambda: be.paged_verify(other, b["plan"], lp.DType.F32, 8, be.upload(np.zeros(64, np.float32)), one, one, one, outs[1], outs[2], outs[3], parents=one)]
    for call in calls:
        call()
        with pytest.raises(lp.LapidError) as e:
            be.synchronize()
        assert e.value.code == "invalid_launch"
        be.synchronize()
    assert np.all(rows.download().view(np.int32) == 7)


# ------------------------------------------------------------------ refusals, streams, graphs
def test_calls_that_are_refused(be):
    from dataclasses import replace
    s = D.TreeStep(be, [[-1, 0, 0], [-1]], [4, 20], hq=4, hkv=2, d=64).upload()
    s.make_plan()
    b, f = s.b, lambda n: be.upload(np.zeros(n, np.float32))
    i = lambda n: be.upload(np.zeros(n, np.int32))
    causal, full, cross = (replace(s.spec, mask=m) for m in (Mask.CAUSAL, Mask.FULL, Mask.CROSS))
    other = lp.Backend(0)
    foreign = other.upload(np.zeros(1 << 16, np.int32))

    def refused(code, fn, *a, **kw):
        with pytest.raises(lp.LapidError) as e:
            fn(*a, **kw)
        assert e.value.code == code, (e.value.code, str(e.value))
    # attention
    att = lambda spec=s.spec, tree=b["tree"], out=b["out"], q=b["q"], **kw: be.paged_tree_attention(spec, b["plan"], tree, q, b["k"], b["v"], b["table"], out, **kw)
    refused("invalid_launch", att, causal)
    refused("out_of_bounds", att, tree=i(4))
    refused("wrong_backend", att, tree=foreign)
    refused("buffer_aliasing", att, out=b["q"])
    refused("buffer_aliasing", att, lse=b["plan"])
    refused("invalid_launch", be.paged_attention, s.spec, b["plan"], b["q"], b["k"], b["v"], b["table"], b["out"])
    # tree
    grow = lambda spec=s.spec, parents=b["parents"], positions=b["positions"], tree=b["tree"]: be.paged_tree(spec, b["plan"], parents, positions, tree)
    refused("invalid_launch", grow, causal)
    refused("out_of_bounds", grow, parents=i(3))
    refused("out_of_bounds", grow, tree=i(7))
    refused("buffer_aliasing", grow, positions=b["parents"])
    refused("buffer_aliasing", grow, tree=b["plan"])
    refused("wrong_backend", grow, parents=foreign)
    # verification
    ok = dict(vocab=10, logits=f(40), tokens=i(4), accept=f(4), pick=f(4), path=i(6), accepted=i(4), next=i(4), parents=i(8))

    def ver(spec=s.spec, dtype=lp.DType.F32, **kw):
        a = {**ok, **kw}
        be.paged_verify(spec, b["plan"], dtype, a["vocab"], a["logits"], a["tokens"], a["accept"], a["pick"], a["path"], a["accepted"], a["next"], parents=a["parents"], draft=a.get("draft"),
                        temperature=a.get("temperature"), logits_row=a.get("logits_row", 0), draft_row=a.get("draft_row", 0))
    refused("invalid_launch", ver, full)
    refused("invalid_launch", ver, cross)
    refused("invalid_argument", ver, parents=None)
    refused("invalid_argument", ver, causal)
    refused("unsupported", ver, replace(causal, max_new=1025, tokens=1), parents=None)
    refused("unsupported_dtype", ver, dtype=lp.DType.Q4K)
    refused("unsupported", ver, vocab=0)
    refused("unsupported", ver, vocab=(1 << 22) + 1)
    refused("out_of_bounds", ver, vocab=11)
    refused("out_of_bounds", ver, logits_row=11)
    refused("invalid_launch", ver, logits_row=9)
    refused("too_large", ver, logits_row=1 << 62)
    refused("out_of_bounds", ver, draft=f(39))
    refused("invalid_launch", ver, draft=f(40), draft_row=3)
    for name, size in (("tokens", 3), ("accept", 3), ("pick", 1), ("path", 5), ("accepted", 1), ("next", 1), ("parents", 3), ("temperature", 1)):
        refused("out_of_bounds", ver, **{name: i(size)})
    for name in ("path", "accepted", "next"):
        refused("buffer_aliasing", ver, **{name: ok["parents"]})
        refused("wrong_backend", ver, **{name: foreign})
    refused("buffer_aliasing", ver, next=ok["accepted"])
    # commit
    com = lambda spec=s.spec, layers=((b["k"], b["v"]),), path=ok["path"], accepted=ok["accepted"], free=b["free"], n_free=len(s.free), kv=b["kv"], used=b["used"], table=b["table"]: \
        be.paged_commit(spec, b["plan"], list(layers), table, path, accepted, kv, used, free_pages=free, n_free=n_free)
    refused("invalid_launch", com, full)
    refused("invalid_launch", com, cross)
    refused("invalid_argument", com, path=None)
    refused("unsupported", com, replace(causal, max_new=1025, tokens=1))
    refused("out_of_bounds", com, layers=((b["k"], i(8)),))
    refused("buffer_aliasing", com, layers=((b["k"], b["k"]),))
    refused("buffer_aliasing", com, layers=((b["k"], b["v"]), (b["v"], be.alloc(1 << 20))))
    refused("buffer_aliasing", com, path=b["k"])
    refused("buffer_aliasing", com, used=b["kv"])
    refused("buffer_aliasing", com, kv=ok["accepted"])
    refused("wrong_backend", com, layers=((b["k"], foreign),))
    refused("out_of_bounds", com, path=i(5))
    refused("out_of_bounds", com, n_free=len(s.free) + 1000)
    refused("invalid_argument", com, free=None, n_free=3)
    be.synchronize()  # none of them left anything behind
    other.close()


def test_empty_steps(be):
    """No requests, no tokens, or requests that have none."""
    for new, cached in (([], []), ([0], [0]), ([0, 0], [5, 16])):
        s = D.TreeStep(be, [[] for _ in new], cached, hq=2, hkv=1, d=16).upload()
        s.make_plan()
        s.attend()
        r = max(1, len(new))
        i = [be.upload(np.full(r, 9, np.int32)) for _ in range(4)]
        z, f = be.upload(np.zeros(16, np.int32)), be.upload(np.zeros(16, np.float32))
        be.paged_verify(s.spec, s.b["plan"], lp.DType.F32, 4, f, z, f, f, i[0], i[1], i[2], parents=z)
        be.paged_commit(s.spec, s.b["plan"], [(s.b["k"], s.b["v"])], s.b["table"], i[0], i[1], s.b["kv"], s.b["used"], free_pages=s.b["free"], n_free=len(s.free))
        be.synchronize()
        get = lambda b: b.download().view(np.int32)[: len(new)].tolist()
        assert get(i[1]) == [0] * len(new) and get(i[2]) == [-1] * len(new) and get(s.b["kv"]) == cached and s.b["used"].download().view(np.int32)[0] == 0


def test_requests_that_take_no_part(be):
    """A length out of bounds: its request is left out by every call, the others are what they would be."""
    rng = np.random.default_rng(0)
    parents = [D.random_parents(rng, n, 2) for n in (4, 6, 3)]
    s = D.TreeStep(be, parents, [5, 7, 9], hq=4, hkv=2, d=64, max_new=6).upload()
    s.b["cached"].write(4, np.array([-3], np.int32))
    s.make_plan()
    s.attend()
    with pytest.raises(lp.LapidError) as e:
        be.synchronize()
    assert e.value.code == "shape_mismatch"
    rows = s.tree_rows()
    assert np.array_equal(rows[:4], D.tree_words(parents[0], 0, 1)) and np.all(rows[4:10] == 0x5a5a5a5a) and np.array_equal(rows[10:13], D.tree_words(parents[2], 0, 1))
    i = [be.upload(np.full(18, 9, np.int32)) for _ in range(3)]
    t, f = be.upload(np.zeros(13, np.int32)), be.upload(np.zeros(13, np.float32))
    be.paged_verify(s.spec, s.b["plan"], lp.DType.F32, 5, be.upload(np.zeros(65, np.float32)), t, f, f, i[0], i[1], i[2], parents=s.b["parents"])
    be.paged_commit(s.spec, s.b["plan"], [], s.b["table"], i[0], i[1], s.b["kv"], s.b["used"], free_pages=s.b["free"], n_free=len(s.free))
    be.synchronize()
    got = [x.download().view(np.int32) for x in i]
    # (accept 0 against a fifth: every first child is accepted)
    assert got[1][0] >= 2 and got[1][1] == 0 and got[1][2] >= 2 and got[2][1] == -1 and np.all(got[0][6:12] == -1)
    kv = s.b["kv"].download().view(np.int32)
    assert kv[0] == 5 + got[1][0] and kv[1] == -3 and kv[2] == 9 + got[1][2]


def test_calls_on_another_stream_and_in_a_graph(be):
    """Verification and commit captured once and replayed on new inputs, on a stream of the caller's."""
    import torch
    stream = torch.cuda.Stream()
    mine = lp.Backend(0)
    mine.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(1)
    w = Walks(mine, [D.random_parents(rng, 6, 2) for _ in range(7)], 900, drawn=True, seed=5).run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        w.packed()
    for seed in range(3):
        again = np.random.default_rng(seed).random(w.tokens).astype(np.float32) * 0.9
        w.packed.keep[2][5].write(0, again)
        w.accept = again
        graph.replay()
        torch.cuda.synchronize()
        mine.synchronize()
        w.check()
    del graph
    mine.close()


@pytest.mark.parametrize("n,cached", [(8, 2000), (64, 3000), (1, 900)])
def test_attention_in_a_graph(be, n, cached):
    """Tree and attention captured once and replayed on other trees: what calls give."""
    import torch
    stream = torch.cuda.Stream()
    mine = lp.Backend(0)
    mine.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(n)
    s = D.TreeStep(mine, [D.random_parents(rng, n, 3)], [cached], hq=8, hkv=2, d=128, page=64).upload()
    b = s.b
    s.make_plan()
    s.attend()
    mine.synchronize()
    calls = [mine.packed_paged_tree(s.spec, b["plan"], b["parents"], b["positions"], b["tree"]),
             mine.packed_paged_tree_attention(s.spec, b["plan"], b["tree"], b["q"], b["k"], b["v"], b["table"], b["out"], lse=b["lse"])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for call in calls:
            call()
    for _ in range(3):
        s.parents = [D.random_parents(rng, n, 4, 0.1)]
        b["parents"].write(0, np.array(s.parents[0], np.int32))
        graph.replay()
        torch.cuda.synchronize()
        mine.synchronize()
        s.check()
    del graph
    mine.close()


def test_two_calls_at_once(be):
    """Two handles' verifications on two streams side by side."""
    import torch
    handles = [lp.Backend(0), lp.Backend(0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rng = np.random.default_rng(1)
    parents = [D.random_parents(rng, 5, 2) for _ in range(30)]
    for h, st in zip(handles, streams):
        h.set_stream(st.cuda_stream)
    walks = [Walks(h, parents, 5000, drawn=True, seed=k).run() for k, h in enumerate(handles)]
    for _ in range(20):
        for w in walks:
            w.packed()
    for h, w in zip(handles, walks):
        h.synchronize()
        w.check()
        h.close()
