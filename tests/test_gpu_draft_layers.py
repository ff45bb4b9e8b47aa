"""Decoder layers for drafted tokens (``tp.DraftLayers``): whole steps of plan, tree, layers, logits, verification and commit, each part against its definition in 64 bits from
what the one in front of it gave, several behind each other and captured."""
import math

import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200.paged import Mask, PagedSpec

from . import draft_ref as D
from . import paged_ref as R
from .test_gpu_paged_layers import BLOCKS, LAYERS, PAGE, PAGES, Stack

pytestmark = pytest.mark.gpu

VOCAB, MOST = 384, 7


class Drafts(Stack):
    """``Stack`` with layers for drafted tokens, which share its weights, caches, table and pages."""

    def __init__(self, dtype, prompts, drawn, window=0, seed=3):
        super().__init__(dtype, prompts, 0)
        from lapid_b200 import quant, tp
        t, r = self.torch, len(prompts)
        self.rng = np.random.default_rng(seed)
        self.head = t.from_numpy(quant.quantize(self.be, tp.Q6_K, self.rng.normal(size=VOCAB * 512).astype(np.float32) * 0.2, VOCAB, 512)).to(self.dev)
        spec = PagedSpec(dtype=dtype, q_heads=8, kv_heads=2, head_dim=64, page_size=PAGE, pages=PAGES, requests=r, tokens=r * MOST + 1, max_blocks=BLOCKS, max_new=MOST, mask=Mask.TREE, window=window)
        self.layers = tp.DraftLayers(self.be, self.shape, spec, self.weights, self.formats, self.caches, self.table, self.free, self.head, tp.Q6_K, VOCAB, rope=self.rope, drawn=drawn)
        self.window, self.drawn = window, drawn

    def drop(self, layers):
        with self.torch.cuda.stream(self.stream):
            layers.drop_used()
        self.stream.synchronize()

    def draft(self, new):
        """Trees, drafted tokens and random numbers of a step."""
        t, l, rng = self.torch, self.layers, self.rng
        self.parents = [D.random_parents(rng, n, 3) for n in new]
        pad = l.m - sum(new)
        put = lambda to, x: to.copy_(t.from_numpy(np.asarray(x)).to(to.dtype))
        put(l.parents, np.concatenate([np.array(p, np.int32) for p in self.parents] + [np.full(pad, -1, np.int32)]))
        put(l.drafted, rng.integers(0, VOCAB, l.m))
        put(l.accept, rng.random(l.m) * 10.0 ** -rng.integers(0, 9, l.m))   # (so that walks go somewhere: the layers' probabilities are random ones, of large logits)
        put(l.pick, rng.random(len(new)) * 0.999)
        put(l.temperature, rng.choice([0.0, 0.7, 1.0], len(new)))
        if self.drawn:
            d = np.exp(rng.normal(size=(l.m, VOCAB)))
            put(l.draft, (d / d.sum(1, keepdims=True)).astype(np.float32))
        t.cuda.synchronize(self.dev)

    def run(self):
        with self.torch.cuda.stream(self.stream):
            self.layers.step()
        self.stream.synchronize()
        self.be.synchronize()

    def check(self, new, cached, before):
        """`before`: the caches in front of the step."""
        l, d, f64 = self.layers, 64, lambda t, *s: t.double().cpu().numpy().reshape(*s)
        table, slots, positions = l.table.cpu().numpy(), l.slots.cpu().numpy(), l.positions.cpu().numpy()
        q, mixed, logits = f64(l.q_half, l.m, 8, d), f64(l.mixed, l.m, 8, d), f64(l.logits, l.m, VOCAB)
        keys, values = (f64(c, PAGES, 2, PAGE, d) for c in self.caches[LAYERS - 1])
        # what the last layer's append stored, from its projections' rows: the caches have been changed by the commit since
        k_rows, v_rows = f64(l.outs["k"], l.m, 2, d), R.to_half(f64(l.outs["v"], l.m, 2, d), self.dtype)[0]
        at = 0
        for r, (n, c) in enumerate(zip(new, cached)):
            depth, _ = D.tree(self.parents[r])
            rows = slice(at, at + n)
            assert list(positions[rows]) == [c + x for x in depth] and list(slots[rows]) == [table[r, x // PAGE] * PAGE + x % PAGE for x in range(c, c + n)]
            path, nxt = (D.verify(logits[rows], self.parents[r], l.drafted[rows].tolist(), f64(l.accept, l.m)[rows], float(l.pick[r]), float(l.temperature[r]),
                                  f64(l.draft, l.m, VOCAB)[rows] if self.drawn else None) if n else ([], -1))
            assert l.path[r].tolist() == path + [-1] * (MOST - len(path)) and int(l.accepted[r]) == len(path) and int(l.next[r]) == nxt
            assert int(l.kv[r]) == c + len(path)
            # keys: turned by their positions, stored, and of the path's tokens moved; the others' may have been written over
            x = np.array([c + y for y in depth])[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)[None, :]
            cos, sin = np.cos(x)[:, None], np.sin(x)[:, None]
            a, b = k_rows[rows][..., :d // 2], k_rows[rows][..., d // 2:]
            turned, size = np.concatenate([a * cos - b * sin, a * sin + b * cos], axis=-1), np.concatenate([np.hypot(a, b)] * 2, axis=-1)
            u = R.U[self.dtype]
            place = lambda j: (table[r, j // PAGE], slice(None), j % PAGE)
            for i, t in enumerate(path):
                assert np.array_equal(values[place(c + i)], v_rows[at + t])
                assert np.all(np.abs(keys[place(c + i)] - turned[t]) <= u * np.abs(turned[t]) + 2.0 ** -21 * size[t] + 2.0 ** -25)
            for j in range(c):  # the cached ones stay
                assert np.array_equal(self.caches[0][0].cpu().view(self.torch.int16).numpy()[place(j)], before[0][0].view(self.torch.int16).numpy()[place(j)])
            # the attention, from keys rounded as the cache has them
            all_k = np.concatenate([np.stack([keys[place(j)] for j in range(c)]) if c else np.zeros((0, 2, d)), R.to_half(turned, self.dtype)[0]])
            all_v = np.concatenate([np.stack([values[place(j)] for j in range(c)]) if c else np.zeros((0, 2, d)), v_rows[rows]])
            out, _, size_o = D.tree_attention(q[rows], all_k, all_v, 4, self.parents[r], self.window, 1 / math.sqrt(d), c)
            # (a drafted key may be rounded the other way than here, by two units of its elements: the scores of n drafted keys are off by at most 2 u |q||k| / 8, and the result by twice that times max |v|)
            slack = 0.0
            if n:
                move = 2 * u * np.linalg.norm(q[rows], axis=-1).max() * np.linalg.norm(all_k[c:], axis=-1).max() / math.sqrt(d)
                slack = 2 * move * np.abs(all_v).max() * 2.0 ** -6  # (and but one in 64 elements is that near a border)
            vmax = float(np.abs(all_v).max()) if len(all_v) else 0.0
            assert np.all(np.abs(mixed[rows] - out) <= R.bound(self.dtype, out, size_o, c + n, vmax) + slack)
            at += n


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("window", [0, 9])
def test_steps_behind_a_prompt(dtype, drawn, window):
    prompts = [20, 1, 9]
    s = Drafts(dtype, prompts, drawn, window)
    s.fill(s.prompt, prompts, [0] * 3)
    s.step(s.prompt)
    s.drop(s.prompt)
    cached, kept = list(prompts), []
    for new in ([7, 4, 1], [1, 7, 0], [6, 5, 7], [7, 7, 7]):
        s.fill(s.layers, new, cached)
        s.draft(new)
        before = [(k.cpu().clone(), v.cpu().clone()) for k, v in s.caches]
        s.run()
        s.check(new, cached, before)
        used = int(s.layers.used)
        assert used == sum(-(-int(k) // PAGE) - -(-c // PAGE) for k, c in zip(s.layers.kv, cached))
        s.drop(s.layers)
        cached = s.layers.kv.tolist()
        kept += s.layers.accepted.tolist()
        # every page is a request's or free, once
        own = [int(s.table[r, b]) for r, c in enumerate(cached) for b in range(-(-c // PAGE))]
        assert sorted(own + [int(x) for x in s.free if x >= 0]) == list(range(PAGES))
    assert max(kept) >= 2


def test_the_logits_are_the_heads_product():
    from lapid_b200.backend import matmul_launch
    from lapid_b200 import tp
    s = Drafts(lp.DType.BF16, [5, 3], False)
    s.fill(s.prompt, [5, 3], [0, 0])
    s.step(s.prompt)
    s.drop(s.prompt)
    s.fill(s.layers, [7, 2], [5, 3])
    s.draft([7, 2])
    s.run()
    out = s.torch.zeros_like(s.layers.logits)
    s.torch.cuda.synchronize(s.dev)
    wrap = s.be.wrap_tensor
    s.be.execute([matmul_launch(tp.Q6_K, s.layers.m, VOCAB, 512)], [wrap(s.layers.x), wrap(s.head), wrap(out)])
    assert float(out.abs().max()) > 0 and s.torch.equal(out, s.layers.logits)


def test_a_captured_step_serves_growing_requests():
    """One graph of a whole step, replayed while the requests grow by what each step accepts, gives what calls give."""
    prompts, outs = [17, 5, 30], []
    for captured in (False, True):
        s = Drafts(lp.DType.BF16, prompts, True, seed=9)
        s.fill(s.prompt, prompts, [0, 0, 0])
        s.step(s.prompt)
        s.drop(s.prompt)
        new = [7, 3, 5]
        s.fill(s.layers, new, prompts)
        t, l = s.torch, s.layers

        def queue():
            l.step()
            l.cached.copy_(l.kv)
            l.drop_used()
        graph = t.cuda.CUDAGraph()
        if captured:
            with t.cuda.graph(graph, stream=s.stream):
                queue()
        mine = []
        for _ in range(4):
            s.draft(new)
            l.h.copy_(s.rows(l.m))
            t.cuda.synchronize(s.dev)
            with t.cuda.stream(s.stream):
                graph.replay() if captured else queue()
            s.stream.synchronize()
            mine.append(t.cat([l.path.reshape(-1), l.accepted, l.next, l.kv, l.free, l.logits[: sum(new)].view(t.int32).reshape(-1)]).clone())
        s.be.synchronize()
        assert int(l.kv.sum()) > sum(prompts) + 12
        outs.append(t.stack(mine).cpu())
        del graph
    assert s.torch.equal(outs[0], outs[1])


def test_refusals():
    from lapid_b200 import tp
    s = Stack(lp.DType.BF16, [2, 1], 0)
    kw = dict(caches=s.caches, table=s.table, free=s.free, rope=s.rope, head=s.weights[0]["q"], head_format=tp.Q4_K, vocab=512)
    with pytest.raises(ValueError, match="TREE"):
        tp.DraftLayers(s.be, s.shape, s.single.spec, s.weights, s.formats, **kw)
