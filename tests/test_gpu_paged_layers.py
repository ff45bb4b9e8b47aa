"""Decoder layers over a paged cache (``tp.PagedLayers``): a prompt step and single-token steps of a small stack, each layer's attention against the
formula in 64 bits from the rows that the projections gave, the projections around it against calls of their own, and a captured step."""
import math

import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200.paged import PagedSpec, rope_table

from . import paged_ref as R

pytestmark = pytest.mark.gpu

SHAPE = (512, 8, 2, 64, 1024)      # d_model, heads, key/value heads, head size, ffn
PAGE, BLOCKS, PAGES, LAYERS = 16, 5, 24, 2


class Stack:
    """Two layers' weights and caches, a table and its free pages, and the layers for prompts and for single tokens that share them."""

    def __init__(self, dtype, prompts, extra_rows):
        import torch
        from lapid_b200 import quant, tp
        self.torch, self.dtype, self.prompts = torch, dtype, prompts
        self.dev = torch.device("cuda", 0)
        self.be = lp.Backend(0)
        self.stream = torch.cuda.Stream(device=self.dev)
        self.be.set_stream(self.stream.cuda_stream)
        rng = np.random.default_rng(5)
        self.shape = tp.LayerShape(*SHAPE)
        self.weights, self.formats = [], []
        for layer in range(LAYERS):
            w, f = {}, {}
            for name, n, k, _ in self.shape.projections():
                fmt = tp.q4km_format(name, layer, LAYERS) if name != "k" else tp.INT8
                w[name] = torch.from_numpy(quant.quantize(self.be, fmt, rng.normal(size=n * k).astype(np.float32) * 0.04, n, k)).to(self.dev)
                f[name] = fmt
            self.weights.append(w)
            self.formats.append(f)
        half = torch.bfloat16 if dtype == lp.DType.BF16 else torch.float16
        r = len(prompts)
        spec = lambda tokens, max_new: PagedSpec(dtype=dtype, q_heads=8, kv_heads=2, head_dim=64, page_size=PAGE, pages=PAGES, requests=r, tokens=tokens,
                                                 max_blocks=BLOCKS, max_new=max_new)
        cache = lambda: torch.full((PAGES, 2, PAGE, 64), float("nan"), dtype=half, device=self.dev)
        self.caches = [(cache(), cache()) for _ in range(LAYERS)]
        self.table = torch.full((r, BLOCKS), -1, dtype=torch.int32, device=self.dev)
        self.order = rng.permutation(PAGES).astype(np.int32)
        self.free = torch.from_numpy(self.order).to(self.dev)
        self.rope = torch.from_numpy(rope_table(BLOCKS * PAGE, 64)).to(self.dev)
        shared = dict(caches=self.caches, table=self.table, free=self.free, rope=self.rope)
        self.prompt = tp.PagedLayers(self.be, self.shape, spec(sum(prompts) + extra_rows, max(prompts)), self.weights, self.formats, **shared)
        self.single = tp.PagedLayers(self.be, self.shape, spec(r, 1), self.weights, self.formats, **shared)
        self.rows = lambda n: torch.from_numpy(rng.normal(size=(n, SHAPE[0])).astype(np.float32)).to(self.dev)
        self.taken = 0

    def fill(self, layers, new, cached):
        t = self.torch
        layers.h.copy_(self.rows(layers.m))
        layers.new.copy_(t.tensor(new, dtype=t.int32))
        layers.cached.copy_(t.tensor(cached, dtype=t.int32))
        t.cuda.synchronize(self.dev)

    def step(self, layers, n=LAYERS):
        with self.torch.cuda.stream(self.stream):
            out = layers.token(n)
        self.stream.synchronize()
        return out

    def take_pages(self, layers):
        """Drops the pages that the step used from the front of the list."""
        self.taken += int(layers.used.item())
        left = self.torch.from_numpy(self.order[self.taken:]).to(self.dev)
        self.free[: left.numel()].copy_(left)
        self.torch.cuda.synchronize(self.dev)

    def check_attention(self, layers, layer, new, cached):
        """What the layer's append and attention left, from the projections' rows that are still there: the last layer's only."""
        g = lambda t, *s: t.double().cpu().numpy().reshape(*s)
        d, u = 64, R.U[self.dtype]
        q, k, v = (g(layers.outs[n], layers.m, -1, d) for n in ("q", "k", "v"))
        table, slots, positions = layers.table.cpu().numpy(), layers.slots.cpu().numpy(), layers.positions.cpu().numpy()
        keys, values = (g(c, PAGES, 2, PAGE, d) for c in self.caches[layer])
        got_q, mixed = g(layers.q_half, layers.m, 8, d), g(layers.mixed, layers.m, 8, d)
        at = 0
        for r, (n, c) in enumerate(zip(new, cached)):
            assert list(positions[at:at + n]) == list(range(c, c + n)) and list(slots[at:at + n]) == [table[r, x // PAGE] * PAGE + x % PAGE for x in range(c, c + n)]
            all_k = np.stack([keys[table[r, x // PAGE], :, x % PAGE] for x in range(c + n)]) if c + n else np.zeros((0, 2, d))
            all_v = np.stack([values[table[r, x // PAGE], :, x % PAGE] for x in range(c + n)]) if c + n else np.zeros((0, 2, d))
            assert np.isfinite(all_k).all() and np.isfinite(all_v).all()
            # v is rounded once; q and k are turned first: f32 angles and products, then one rounding
            assert np.array_equal(all_v[c:], R.to_half(v[at:at + n], self.dtype)[0])
            x = np.arange(c, c + n)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)[None, :]
            cos, sin = np.cos(x)[:, None], np.sin(x)[:, None]
            for rows, have in ((q[at:at + n], got_q[at:at + n]), (k[at:at + n], all_k[c:])):
                a, b = rows[..., :d // 2], rows[..., d // 2:]
                want = np.concatenate([a * cos - b * sin, a * sin + b * cos], axis=-1)
                size = np.concatenate([np.hypot(a, b)] * 2, axis=-1)
                assert np.all(np.abs(have - want) <= u * np.abs(want) + 2.0 ** -21 * size + 2.0 ** -25)
            out, _, size = R.attention(got_q[at:at + n], all_k, all_v, 4, lp.paged.Mask.CAUSAL, 0, 1.0 / math.sqrt(d), n, c + n)
            vmax = float(np.abs(all_v).max()) if c + n else 0.0
            assert np.all(np.abs(mixed[at:at + n] - out) <= R.bound(self.dtype, out, size, c + n, vmax)), r
            at += n
        assert np.all(slots[at:] == -1) and np.all(positions[at:] == -1)
        return at


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("prompts,extra", [([20, 1, 33, 0], 3), ([3, 2], 1)])
def test_prompts_then_single_tokens(dtype, prompts, extra):
    s = Stack(dtype, prompts, extra)
    n = len(prompts)
    s.fill(s.prompt, prompts, [0] * n)
    for layers in range(1, LAYERS + 1):          # a stack of one layer, then of two: the same pages again
        assert s.torch.isfinite(s.step(s.prompt, layers)[: sum(prompts)]).all()
        assert s.check_attention(s.prompt, layers - 1, prompts, [0] * n) == sum(prompts)
    assert int(s.prompt.used.item()) == sum(-(-p // PAGE) for p in prompts)
    s.take_pages(s.prompt)
    cached = list(prompts)
    for _ in range(3):
        new = [1] * n
        s.fill(s.single, new, cached)
        out = s.step(s.single)
        assert s.torch.isfinite(out).all()
        s.check_attention(s.single, LAYERS - 1, new, cached)
        assert s.single.kv.tolist() == [c + 1 for c in cached]
        s.take_pages(s.single)
        cached = s.single.kv.tolist()


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("prompts", [[20, 9], [2, 3]])
def test_the_output_projection_reads_what_the_attention_wrote(dtype, prompts):
    """o of the mixed rows, widened exactly: the same product from f32 rows, bit for bit."""
    from lapid_b200 import tp
    from lapid_b200.backend import matmul_launch
    s = Stack(dtype, prompts, 0)
    s.fill(s.prompt, prompts, [0] * len(prompts))
    s.step(s.prompt)
    got = s.prompt.outs["o"].cpu()
    wide, out = s.prompt.mixed.float(), s.torch.zeros_like(s.prompt.outs["o"])
    s.torch.cuda.synchronize(s.dev)
    wrap = s.be.wrap_tensor
    s.be.execute([matmul_launch(s.formats[1]["o"], s.prompt.m, 512, 512)], [wrap(wide), wrap(s.weights[1]["o"]), wrap(out)])
    s.be.synchronize()
    assert float(got.abs().max()) > 0 and s.torch.equal(got, out.cpu())


def test_a_captured_step_serves_growing_requests():
    """One graph of a single-token step, replayed with `cached` taken from the step before on the device, gives what calls give."""
    prompts = [17, 5, 30]
    outs = []
    for captured in (False, True):
        s = Stack(lp.DType.BF16, prompts, 0)
        s.fill(s.prompt, prompts, [0, 0, 0])
        s.step(s.prompt)
        s.take_pages(s.prompt)
        s.fill(s.single, [1, 1, 1], prompts)
        t = s.torch
        rows = [s.rows(3) for _ in range(4)]

        def queue():
            out = s.single.token(LAYERS)
            s.single.cached.copy_(s.single.kv)
            return out
        graph = t.cuda.CUDAGraph()
        if captured:
            with t.cuda.graph(graph, stream=s.stream):
                queue()
        mine = []
        for x in rows:
            s.single.h.copy_(x)
            t.cuda.synchronize(s.dev)
            with t.cuda.stream(s.stream):
                graph.replay() if captured else queue()
            s.stream.synchronize()
            s.take_pages(s.single)
            mine.append(s.single.hw.clone())
        s.be.synchronize()
        assert s.single.kv.tolist() == [p + 4 for p in prompts]
        outs.append(t.stack(mine).cpu())
        del graph
    assert s.torch.isfinite(outs[0]).all() and s.torch.equal(outs[0], outs[1])


def test_refusals():
    from lapid_b200 import tp
    s = Stack(lp.DType.BF16, [2, 1], 0)
    kw = dict(caches=s.caches, table=s.table, free=s.free, rope=s.rope)
    make = lambda spec, **over: tp.PagedLayers(s.be, s.shape, spec, s.weights, s.formats, **{**kw, **over})
    with pytest.raises(ValueError, match="caches for"):
        s.single.token(LAYERS + 1)
    with pytest.raises(ValueError, match="heads"):
        make(PagedSpec(dtype=lp.DType.BF16, q_heads=4, kv_heads=2, head_dim=64, page_size=PAGE, pages=PAGES, requests=2, tokens=2, max_blocks=BLOCKS, max_new=1))
    with pytest.raises(ValueError, match="block table"):
        make(s.single.spec, table=s.table[:1])
    with pytest.raises(ValueError, match="rope"):
        make(s.single.spec, rope=s.rope[0])
    short = [(k[:4].contiguous(), v) for k, v in s.caches]
    broken = make(s.single.spec, caches=short)
    with pytest.raises(lp.LapidError):
        broken.token(1)
