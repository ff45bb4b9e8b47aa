"""What a step of decoder layers for drafted tokens (``tp.DraftLayers``) leaves in the caches of all layers, bit for bit, and a captured step whose pages run out."""
import math

import numpy as np
import pytest

import lapid_b200 as lp

from . import draft_ref as D
from . import paged_ref as R
from .test_gpu_draft_layers import Drafts, MOST, VOCAB
from .test_gpu_paged_layers import LAYERS, PAGE, PAGES

pytestmark = pytest.mark.gpu


def bits(s):
    """The caches as whole numbers [layer][keys, values]: pages, heads, places, elements."""
    return [[c.cpu().view(s.torch.int16).numpy().copy() for c in pair] for pair in s.caches]


@pytest.mark.parametrize("dtype", [lp.DType.BF16, lp.DType.F16])
@pytest.mark.parametrize("drawn,window", [(False, 0), (True, 9)])
def test_all_layers_caches(dtype, drawn, window):
    """Layers and verification change the drafted tokens' places alone; the commit moves the path's, and nothing else. The last layer's attention is that of the keys and values as they lay there in between."""
    prompts = [20, 1, 9]
    s = Drafts(dtype, prompts, drawn, window, seed=8)
    s.fill(s.prompt, prompts, [0] * 3)
    s.step(s.prompt)
    s.drop(s.prompt)
    l, cached, moved = s.layers, list(prompts), 0
    for new in ([7, 4, 1], [2, 7, 0], [7, 7, 7]):
        s.fill(l, new, cached)
        s.draft(new)
        before = bits(s)
        with s.torch.cuda.stream(s.stream):
            l.token(LAYERS)
            l._head()
            l._verify()
        s.stream.synchronize()
        between, table = bits(s), l.table.cpu().numpy()
        with s.torch.cuda.stream(s.stream):
            l._commit()
        s.stream.synchronize()
        s.be.synchronize()
        after = bits(s)
        place = lambda r, j: (table[r, j // PAGE], slice(None), j % PAGE)
        paths = [[t for t in row if t >= 0] for row in l.path.tolist()]
        for layer in range(LAYERS):
            for half in range(2):
                drafted = np.zeros(between[layer][half].shape[:1] + between[layer][half].shape[2:3], bool)
                want = between[layer][half].copy()
                for r, (n, c) in enumerate(zip(new, cached)):
                    for j in range(c, c + n):
                        drafted[table[r, j // PAGE], j % PAGE] = True
                    for i, t in enumerate(paths[r]):
                        want[place(r, c + i)] = between[layer][half][place(r, c + t)]
                        moved += t != i
                same = (before[layer][half] == between[layer][half]).all(axis=(1, 3))
                assert np.all(same | drafted)
                assert np.array_equal(after[layer][half], want)
        keys, values = (R.from_half(x, dtype) for x in between[LAYERS - 1])
        q, mixed, at = l.q_half.double().cpu().numpy().reshape(l.m, 8, 64), l.mixed.double().cpu().numpy().reshape(l.m, 8, 64), 0
        for r, (n, c) in enumerate(zip(new, cached)):
            if n == 0:
                continue
            k, v = (np.stack([x[place(r, j)] for j in range(c + n)]) for x in (keys, values))
            out, _, size = D.tree_attention(q[at:at + n], k, v, 4, s.parents[r], window, 1 / math.sqrt(64), c)
            assert np.all(np.abs(mixed[at:at + n] - out) <= R.bound(dtype, out, size, c + n, float(np.abs(v).max())))
            at += n
        s.drop(l)
        cached = l.kv.tolist()
    assert drawn or moved  # (few of the tokens drawn here are accepted)


def test_a_captured_step_whose_pages_ran_out_is_run_again():
    """The step keeps nothing and says so; with more pages the same graph on the same inputs gives what it would have given."""
    prompts, new = [15, 16, 30], [7, 3, 5]
    outs = []
    for short in (False, True):
        s = Drafts(lp.DType.BF16, prompts, True, seed=4)
        s.fill(s.prompt, prompts, [0, 0, 0])
        s.step(s.prompt)
        s.drop(s.prompt)
        t, l = s.torch, s.layers
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph, stream=s.stream):
            l.step()
        s.fill(l, new, prompts)
        s.draft(new)
        rows, all_free, before = l.h.clone(), s.free.clone(), bits(s)
        if short:
            s.free[1:] = -1
            t.cuda.synchronize(s.dev)
            with t.cuda.stream(s.stream):
                graph.replay()
            s.stream.synchronize()
            with pytest.raises(lp.LapidError) as e:
                s.be.synchronize()
            assert e.value.code == "out_of_memory"
            assert l.kv.tolist() == prompts and int(l.used) == 0 and s.free[1:].tolist() == [-1] * (PAGES - 1) and int(s.free[0]) == int(all_free[0])
            table, now = l.table.cpu().numpy(), bits(s)
            for layer in range(LAYERS):
                for half in range(2):
                    for r, c in enumerate(prompts):
                        for j in range(c):
                            at = (table[r, j // PAGE], slice(None), j % PAGE)
                            assert np.array_equal(now[layer][half][at], before[layer][half][at])
            s.free.copy_(all_free)
            l.h.copy_(rows)
            t.cuda.synchronize(s.dev)
        with t.cuda.stream(s.stream):
            graph.replay()
        s.stream.synchronize()
        s.be.synchronize()
        outs.append(t.cat([l.path.reshape(-1), l.accepted, l.next, l.kv, l.used, l.free, l.logits[: sum(new)].view(t.int32).reshape(-1)]).cpu())
        assert int(l.accepted.sum()) >= 3 and l.logits.shape[1] == VOCAB and l.path.shape[1] == MOST
        del graph
    assert s.torch.equal(outs[0], outs[1])
