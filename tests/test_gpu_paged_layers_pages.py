"""Decoder layers over a paged cache when the free pages end, and a first exchange by itself."""
import numpy as np
import pytest

import lapid_b200 as lp

from .test_gpu_paged_layers import LAYERS, PAGE, SHAPE, Stack

pytestmark = pytest.mark.gpu


def start(prompts, pages):
    """The prompts' step with `pages` free pages in the list."""
    s = Stack(lp.DType.BF16, prompts, 0)
    s.free[pages:] = -1
    s.fill(s.prompt, prompts, [0] * len(prompts))
    s.step(s.prompt)
    s.be.synchronize()
    with s.torch.cuda.stream(s.stream):
        s.prompt.drop_used()
    s.stream.synchronize()
    return s


def test_drop_used_moves_the_list_up():
    s = start([20, 5, 33], 9)           # 2 + 1 + 3 pages
    assert s.prompt.used.tolist() == [6]
    assert s.free.tolist() == s.order[6:9].tolist() + [-1] * (len(s.order) - 3)
    with s.torch.cuda.stream(s.stream):
        s.prompt.drop_used()            # more than there are: nothing is left
    s.stream.synchronize()
    assert s.free.tolist() == [-1] * len(s.order)


@pytest.mark.parametrize("captured", [False, True])
def test_pages_that_run_out_are_said_and_no_ones_keys_are_written_over(captured):
    """Three free pages behind the prompts. The first step takes one, the second two, the third asks for two more and says so; every page in a table row stays its row's alone."""
    prompts = [15, 16, 14, 30, 31]
    s = start(prompts, 1 + 1 + 1 + 2 + 2 + 3)
    s.fill(s.single, [1] * 5, prompts)
    t, graph = s.torch, s.torch.cuda.CUDAGraph()

    def queue():
        s.single.token(LAYERS)
        s.single.drop_used()
        s.single.cached.copy_(s.single.kv)
    if captured:
        with t.cuda.graph(graph, stream=s.stream):
            queue()
    asked, failed = list(prompts), None
    for step in range(4):
        s.single.h.copy_(s.rows(5))
        before = [(k.clone(), v.clone()) for k, v in s.caches]
        table = s.table.cpu().numpy()
        t.cuda.synchronize(s.dev)
        with t.cuda.stream(s.stream):
            graph.replay() if captured else queue()
        s.stream.synchronize()
        try:
            s.be.synchronize()
        except lp.LapidError as e:
            failed = (step, e.code)
        asked = [c + 1 for c in asked]
        after = s.table.cpu().numpy()
        owned = after[after >= 0].tolist()
        assert len(owned) == len(set(owned))                       # no page in two rows
        assert np.array_equal(after[table >= 0], table[table >= 0])  # none taken away
        new = {(int(after[r, (c - 1) // PAGE]), (c - 1) % PAGE) for r, c in enumerate(asked)}
        for (k0, v0), (k1, v1) in zip(before, s.caches):
            for x, y in ((k0, k1), (v0, v1)):
                same = (x.view(t.int16) == y.view(t.int16)).all(dim=3).all(dim=1).cpu().numpy()   # [page, place]
                changed = {(int(p), int(i)) for p, i in zip(*np.nonzero(~same))}
                assert changed <= new, (step, changed - new)       # only places of this step's own tokens
        if failed:
            break
    assert failed == (2, "out_of_memory")
    del graph


def test_the_first_row_parallel_result_makes_its_plan():
    s = Stack(lp.DType.BF16, [20, 3], 0)
    s.fill(s.prompt, [20, 3], [0, 0])
    with s.torch.cuda.stream(s.stream):
        out = s.prompt.first_row_parallel()
    s.stream.synchronize()
    s.be.synchronize()
    assert s.check_attention(s.prompt, 0, [20, 3], [0, 0]) == 23
    h, o = s.prompt.h.double(), s.prompt.outs["o"].double()
    assert float(o.abs().max()) > 0
    assert s.torch.all((out.double() - (h + o)).abs() <= 2.0 ** -22 * (h.abs() + o.abs()))
    assert out.shape == (23, SHAPE[0])
