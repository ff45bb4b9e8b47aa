"""Drafted tokens over the paged key/value cache: a tree of them checked by the model in one step, and what is kept of it.

``listed()`` gives the cases that are always timed, ``draw(rng)`` more of the same ranges, ``prepare(case, seed)`` what a
serving program holds before the call, ``run(state)`` one pass, ``work(case)`` the bytes and operations that a pass
cannot do without, ``exact(case, seed)`` the outputs from the definitions in 64 bits.

Operators (``op``):

  tree    once a step: positions and ancestors of every drafted token, from its parent's index
  attend  once a layer: attention of every drafted token over the cached keys, its ancestors' and its own
  verify  once a step: which drafted tokens the model's probabilities accept, with given random numbers, and the token behind them
  commit  once a step: keys and values of the accepted tokens moved behind the cached ones in every layer, other pages given back

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits (verify in 64: its decisions are
comparisons); with ``own`` true it makes the framework's calls. Inputs are synthetic, made on the GPU from the seed.
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_backend = None
_stream = None


def listed():
    return [
        # eight users with a small tree each: latency
        {"name": "tree_8x16", "op": "tree", "requests": 8, "nodes": 16, "spread": 1.0, "branch": 4, "roots": 0.0, "cached": 2048, "page": 16, "window": 0},
        # a full server with large trees of different sizes, a window shorter than some of their paths
        {"name": "tree_512x64_ragged", "op": "tree", "requests": 512, "nodes": 64, "spread": 0.3, "branch": 3, "roots": 0.05, "cached": 512, "page": 32, "window": 9},
        # one user, a small tree, a context of a few thousand tokens: latency
        {"name": "attend_b1_n8_4k", "op": "attend", "requests": 1, "nodes": 8, "spread": 1.0, "branch": 3, "roots": 0.0, "cached": 4096, "ragged": 1.0, "page": 16, "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "window": 0, "lse": False},
        # one user, a large tree, a long context
        {"name": "attend_b1_n64_32k", "op": "attend", "requests": 1, "nodes": 64, "spread": 1.0, "branch": 4, "roots": 0.0, "cached": 32768, "ragged": 1.0, "page": 64, "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "window": 0, "lse": True},
        # sixteen users, trees of eight, contexts of all lengths: the usual step of a server that drafts
        {"name": "attend_b16_n8_ragged", "op": "attend", "requests": 16, "nodes": 8, "spread": 1.0, "branch": 3, "roots": 0.0, "cached": 8192, "ragged": 0.2, "page": 16, "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "window": 0, "lse": False},
        # trees of different sizes, an odd group of small heads, a sliding window
        {"name": "attend_b8_n37_d64", "op": "attend", "requests": 8, "nodes": 37, "spread": 0.4, "branch": 3, "roots": 0.1, "cached": 3001, "ragged": 0.3, "page": 32, "dtype": "f16", "hq": 14, "hkv": 2, "d": 64,
         "window": 1024, "lse": False},
        # one user, a chain of drafted tokens with the draft model's probabilities: latency
        {"name": "verify_b1_chain8", "op": "verify", "requests": 1, "nodes": 8, "branch": 1, "vocab": 128256, "dtype": "f32", "draft": True, "temperature": 1.0},
        # sixteen users, trees of candidates that were chosen, not drawn
        {"name": "verify_b16_tree16", "op": "verify", "requests": 16, "nodes": 16, "branch": 4, "vocab": 32000, "dtype": "f32", "draft": False, "temperature": 0.8},
        # a full server, drawn candidates, some of them siblings
        {"name": "verify_b64_tree8", "op": "verify", "requests": 64, "nodes": 8, "branch": 2, "vocab": 128256, "dtype": "f32", "draft": True, "temperature": 1.0},
        # greedy users, half-precision logits, an odd vocabulary
        {"name": "verify_b32_greedy", "op": "verify", "requests": 32, "nodes": 6, "branch": 2, "vocab": 50257, "dtype": "bf16", "draft": False, "temperature": 0.0},
        # one user, all layers of a model: latency
        {"name": "commit_b1_l32", "op": "commit", "requests": 1, "nodes": 16, "spread": 1.0, "branch": 3, "cached": 100, "page": 16, "layers": 32, "dtype": "bf16", "hkv": 8, "d": 128},
        # a full server, long accepted paths
        {"name": "commit_b32_l32", "op": "commit", "requests": 32, "nodes": 24, "spread": 0.5, "branch": 2, "cached": 49, "page": 16, "layers": 32, "dtype": "f16", "hkv": 8, "d": 128},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (64, 8, 128), (16, 4, 64), (8, 8, 128), (28, 4, 128), (14, 2, 64), (12, 4, 96), (8, 1, 128), (16, 16, 64), (20, 5, 80)]


def draw(rng):
    op = rng.choice(["tree", "attend", "attend", "verify", "verify", "commit"])
    page = rng.choice([16, 32, 64, 128])
    if op == "tree":
        r = _log_int(rng, 1, 512)
        return {"op": op, "requests": r, "nodes": _log_int(rng, 1, min(256, 32768 // r)), "spread": rng.choice([0.0, 0.5, 1.0]), "branch": rng.randint(1, 9), "roots": rng.choice([0.0, 0.1]),
                "cached": _log_int(rng, 1, 8192), "page": page, "window": rng.choice([0, 0, 5, 100])}
    hq, hkv, d = rng.choice(HEADS)
    if op == "attend":
        r = _log_int(rng, 1, 32)
        return {"op": op, "requests": r, "nodes": _log_int(rng, 2, min(128, 512 // r)), "spread": rng.choice([0.0, 0.5, 1.0]), "branch": rng.randint(1, 6), "roots": rng.choice([0.0, 0.0, 0.1]),
                "cached": _log_int(rng, 16, min(32768, 131072 // r)), "ragged": rng.choice([0.0, 0.4, 1.0]), "page": page, "dtype": rng.choice(["f16", "bf16"]), "hq": hq, "hkv": hkv, "d": d,
                "window": rng.choice([0, 0, 0, 127, 1024]), "lse": rng.random() < 0.3}
    if op == "verify":
        r, vocab = _log_int(rng, 1, 64), _log_int(rng, 1000, 131072)
        return {"op": op, "requests": r, "nodes": min(_log_int(rng, 1, 24), 60_000_000 // (r * vocab)), "branch": rng.randint(1, 4), "vocab": vocab, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
                "draft": rng.random() < 0.5, "temperature": rng.choice([0.0, 0.7, 1.0, 1.0, 1.3])}
    r = _log_int(rng, 1, 32)
    return {"op": op, "requests": r, "nodes": _log_int(rng, 1, 24), "spread": rng.choice([0.0, 0.5, 1.0]), "branch": rng.randint(1, 4), "cached": _log_int(rng, 1, 100), "page": min(page, 32),
            "layers": rng.randint(1, 32), "dtype": rng.choice(["f16", "bf16"]), "hkv": hkv, "d": d}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _between(most, part, count, gen, device):
    """``count`` whole numbers from ``part * most`` to ``most``."""
    lo = int(part * most)
    return (lo + (torch.rand(count, generator=gen, device=device) * (most - lo + 1)).long()).clamp(max=most)


def _requests(case, gen, device):
    """Lengths, the block table as the step before left it, the free pages in an order of their own, and every drafted token's parent."""
    r, n, page = case["requests"], case["nodes"], case["page"]
    new_lens = _between(n, case["spread"], r, gen, device).clamp(min=1)
    cached = _between(case["cached"], case.get("ragged", 0.5), r, gen, device)
    blocks = -(-(case["cached"] + n) // page)
    pages = r * blocks + 3
    order = torch.randperm(pages, generator=gen, device=device)
    table = order[: r * blocks].reshape(r, blocks)
    have = -(-cached // page)
    taken = torch.arange(blocks, device=device)[None, :] < have[:, None]
    free = torch.cat([table[~taken], order[r * blocks:]])
    free = free[torch.randperm(free.numel(), generator=gen, device=device)]
    padded = torch.full((pages,), -1, dtype=torch.int32, device=device)  # the list has room for every page; its first entries count
    padded[: free.numel()] = free.int()
    end = torch.cumsum(new_lens, 0)
    token = torch.arange(r * n, device=device)
    request = torch.searchsorted(end, token, right=True)
    real = request < r
    request = request.clamp(max=r - 1)
    index = torch.where(real, token - (end - new_lens)[request], 0)
    return {"new_lens": new_lens.int(), "cached": cached.int(), "table": torch.where(taken, table, -1).int().contiguous(), "free": padded, "n_free": free.numel(), "tokens": r * n, "blocks": blocks,
            "pages": pages, "request": request, "index": index, "real": real, "parents": _parents(index, case["branch"], case.get("roots", 0.0), gen)}


def _parents(index, branch, roots, gen):
    """The index in its request of each token's parent, one of the ``branch`` before it; the first token of a request, and the given part of the others, has none (-1)."""
    back = 1 + (torch.rand(index.shape, generator=gen, device=index.device) * branch).long().clamp(max=branch - 1)
    alone = torch.rand(index.shape, generator=gen, device=index.device) < roots
    return torch.where((index == 0) | alone, -1, (index - back).clamp(min=0)).int()


def _inputs(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=device)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device=device)  # noqa: E731
    if case["op"] == "verify":
        return _verify_inputs(case, gen, normal, uniform)
    s = _requests(case, gen, device)
    page, r, words = case["page"], case["requests"], -(-case["nodes"] // 32)
    if case["op"] == "tree":
        s["positions"] = torch.where(s["real"], s["cached"].long()[s["request"]] + s["index"], -1).int()  # as the plan leaves them
        s["tree"] = torch.zeros(s["tokens"], 1 + words, dtype=torch.int32, device=device)
        return s
    s["table"], s["kv_lens"], s["used"] = _plan(s, page)
    dtype, hkv, d = DTYPE[case["dtype"]], case["hkv"], case["d"]
    if case["op"] == "commit":
        s["cache"] = torch.empty(case["layers"], 2, s["pages"], hkv, page, d, dtype=dtype, device=device).normal_(generator=gen)
        step = 1 + (uniform(r, case["nodes"]) * case["branch"]).long().clamp(max=case["branch"] - 1)
        step[:, 0] = 0
        path = torch.cumsum(step, 1)                                                    # a path's tokens: rising, from the first
        fits = (path < s["new_lens"].long()[:, None]).sum(1)
        s["accepted"] = (1 + (uniform(r) * fits).long()).clamp(max=fits).int()
        s["path"] = torch.where(torch.arange(case["nodes"], device=device)[None, :] < s["accepted"][:, None], path, -1).int().contiguous()
        return s
    s["q"] = normal(s["tokens"], case["hq"], d).to(dtype)
    s["k_cache"] = torch.empty(s["pages"], hkv, page, d, dtype=dtype, device=device).normal_(generator=gen)
    s["v_cache"] = torch.empty(s["pages"], hkv, page, d, dtype=dtype, device=device).normal_(generator=gen)
    s["k_cache"] *= 1.5  # some keys stand out, as they do in trained heads
    s["out"] = torch.zeros(s["tokens"], case["hq"], d, dtype=dtype, device=device)
    s["lse"] = torch.zeros(s["tokens"], case["hq"], dtype=torch.float32, device=device) if case["lse"] else None
    return s


def _verify_inputs(case, gen, normal, uniform):
    """Rows of logits with a few tokens that stand out; candidates that are these (chosen), or drawn from a draft model's distribution that is near the model's."""
    r, n, branch, vocab = case["requests"], case["nodes"], case["branch"], case["vocab"]
    t = r * n
    index = torch.arange(t, device="cuda") % n
    parents = _parents(index, branch, 0.0, gen)
    logits = normal(t, vocab).mul_(2.0)
    best = (uniform(t, branch) * vocab).long().clamp(max=vocab - 1)
    logits.scatter_(1, best, 2.0 + math.log(vocab) + normal(t, branch) - torch.arange(branch, device="cuda")[None, :])
    draft, candidates = None, best
    if case["draft"]:
        draft = torch.softmax(logits + 0.7 * normal(t, vocab), -1)
        candidates = torch.multinomial(draft, branch, replacement=True, generator=gen)
    parent_row = (torch.arange(t, device="cuda") - index + parents.long()).clamp(min=0)
    which = (index - parents.long() - 1).clamp(0, branch - 1)  # a child takes the candidate of its distance
    tokens = torch.where(index == 0, 0, candidates[parent_row, which]).int()
    return {"tokens": t, "new_lens": torch.full((r,), n, dtype=torch.int32, device="cuda"), "parents": parents, "logits": logits.to(DTYPE[case["dtype"]]), "draft": draft, "drafted": tokens,
            "accept": uniform(t), "pick": uniform(r), "temperature": torch.full((r,), case["temperature"], device="cuda"), "path": torch.full((r, n), -1, dtype=torch.int32, device="cuda"),
            "accepted": torch.zeros(r, dtype=torch.int32, device="cuda"), "next": torch.zeros(r, dtype=torch.int32, device="cuda")}


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plan(s, page):
    """Block table, lengths of the keys, and how many pages the step takes: from the lists as they are before the call."""
    new, cached, table = s["new_lens"].long(), s["cached"].long(), s["table"]
    kv = cached + new
    have, need = -(-cached // page), -(-kv // page)
    first = torch.cumsum(need - have, 0) - (need - have)
    column = torch.arange(s["blocks"], device=table.device)[None, :]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    at = (first[:, None] + column - have[:, None]).clamp(0, s["free"].numel() - 1)
    return torch.where(fresh, s["free"][at], table).contiguous(), kv.int(), (need - have).sum().int().reshape(1)


def _ancestors(s, n, window=0):
    """[tokens, n] whether a token of the same request is its ancestor or itself, and how many ancestors it has: by doubling what each knows. With a window, those nearer than that."""
    t, device = s["tokens"], s["parents"].device
    first = torch.arange(t, device=device) - s["index"]
    parent = s["parents"].long()
    up = torch.where(parent >= 0, first + parent, torch.arange(t, device=device))           # a root's parent is itself
    own_bit = torch.arange(n, device=device)[None, :] == s["index"][:, None]
    seen = own_bit | ((torch.arange(n, device=device)[None, :] == parent[:, None]) & (parent >= 0)[:, None])
    for _ in range(max(1, (n - 1).bit_length())):
        seen = seen | seen[up]
        up = up[up]
    depth = seen.sum(1) - 1
    if window:
        at = (first[:, None] + torch.arange(n, device=device)[None, :]).clamp(max=t - 1)
        seen = seen & (depth[:, None] - depth[at] < window)
    return seen, depth


def _tree(s, c):
    n, words = c["nodes"], -(-c["nodes"] // 32)
    seen, depth = _ancestors(s, n, c["window"])
    bits = torch.zeros(s["tokens"], words * 32, dtype=torch.long, device=seen.device)
    bits[:, :n] = seen.long()
    packed = (bits.view(-1, words, 32) << torch.arange(32, device=seen.device)).sum(-1)
    packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed)
    tree = torch.cat([depth[:, None], packed], 1).int()
    positions = torch.where(s["real"], s["cached"].long()[s["request"]] + depth, -1).int()
    return {"positions": positions, "tree": torch.where(s["real"][:, None], tree, 0)}


def _attend(s, c):
    hq, hkv, d, page, most_new = c["hq"], c["hkv"], c["d"], c["page"], c["nodes"]
    g = hq // hkv
    new, kv = s["new_lens"].long(), s["kv_lens"].long()
    r, blocks, device = new.numel(), s["blocks"], new.device
    end = torch.cumsum(new, 0)
    row = torch.arange(most_new, device=device)
    real = row[None, :] < new[:, None]                                                 # [r, n]
    at = ((end - new)[:, None] + row[None, :]).clamp(max=s["tokens"] - 1)
    ancestors, depth = _ancestors(s, most_new, c["window"])
    q = s["q"].float()[at].view(r, most_new, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, g * most_new, d)
    pages = s["table"].long().clamp(min=0)                                             # [r, blocks]
    k = s["k_cache"][pages].float().permute(0, 2, 1, 3, 4).reshape(r, hkv, blocks * page, d)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(r, hkv, g, most_new, blocks * page)
    del k
    key = torch.arange(blocks * page, device=device)
    cached = kv - new
    lo = (cached[:, None] + depth[at] + 1 - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(at)
    seen = (key[None, None, :] < cached[:, None, None]) & (key[None, None, :] >= lo[:, :, None])
    drafted = (key[None, :] - cached[:, None]).clamp(0, most_new - 1)                  # [r, keys]
    behind = (key[None, :] >= cached[:, None]) & (key[None, :] < kv[:, None])
    seen = seen | (behind[:, None, :] & torch.gather(ancestors[at], 2, drafted[:, None, :].expand(r, most_new, blocks * page)))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(base).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v_cache"][pages].float().permute(0, 2, 1, 3, 4).reshape(r, hkv, blocks * page, d)
    v.masked_fill_((key[None, :] >= kv[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.view(r, hkv, g * most_new, blocks * page), v).view(r, hkv, g, most_new, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(r * most_new, hq, d)
    s["out"][at[real]] = o[real.reshape(-1)].to(s["out"].dtype)
    if s["lse"] is not None:
        lse = (base + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(r * most_new, hq)
        s["lse"][at[real]] = lse[real.reshape(-1)]
    return {"out": s["out"], "lse": s["lse"]}


def _verify(s, c):
    """All requests walk down their trees together, one level at a time; a node's children, at most ``branch`` places behind it, are tried in their order."""
    r, n, branch, vocab = c["requests"], c["nodes"], c["branch"], c["vocab"]
    device = s["logits"].device
    base = torch.arange(r, device=device) * n
    node, going = torch.zeros(r, dtype=torch.long, device=device), torch.ones(r, dtype=torch.bool, device=device)
    path = torch.full((r, n), -1, dtype=torch.int32, device=device)
    path[:, 0] = 0
    length = torch.ones(r, dtype=torch.long, device=device)
    left = torch.zeros(r, vocab, dtype=torch.float64, device=device)                   # what remains of the distribution where a request's walk ended
    cold = s["temperature"][:, None] == 0
    for _ in range(n):
        z = s["logits"][base + node].double()
        z = z - z.amax(-1, keepdim=True)
        best = torch.arange(vocab, device=device)[None, :] == z.argmax(-1, keepdim=True)
        p = torch.where(cold, best.double(), (z / torch.where(cold, 1.0, s["temperature"].double()[:, None])).exp())
        p = p / p.sum(-1, keepdim=True)
        moved = torch.zeros_like(going)
        parent = node
        for j in range(1, branch + 1):
            child = parent + j
            row = (base + child).clamp(max=r * n - 1)
            there = going & ~moved & (child < n) & (s["parents"].long()[row] == parent)
            token = s["drafted"].long()[row][:, None]
            q = s["draft"][base + parent].double() if s["draft"] is not None else None
            weight = q.gather(1, token) if q is not None else 1.0
            yes = there & (s["accept"].double()[row][:, None] * weight < p.gather(1, token)).squeeze(1)
            rest = (p - q).clamp(min=0) if q is not None else p.scatter(1, token, 0.0)
            total = rest.sum(-1, keepdim=True)
            p = torch.where((there & ~yes)[:, None] & (total > 0), rest / total, p)
            node = torch.where(yes, child, node)
            path[torch.arange(r, device=device), length.clamp(max=n - 1)] = torch.where(yes, child.int(), path[torch.arange(r, device=device), length.clamp(max=n - 1)])
            length = length + yes.long()
            moved = moved | yes
        left = torch.where((going & ~moved)[:, None], p, left)
        going = going & moved
    run_sum = torch.cumsum(left, -1)
    over = run_sum > s["pick"].double()[:, None] * run_sum[:, -1:]
    last = vocab - 1 - (left > 0).flip(-1).int().argmax(-1)
    token = torch.where(over.any(-1), over.int().argmax(-1), last)
    return {"path": path, "accepted": length.int(), "next": token.int()}


def _commit(s, c):
    page, n = c["page"], c["nodes"]
    new, cached, accepted, table = s["new_lens"].long(), s["cached"].long(), s["accepted"].long(), s["table"].long()
    device = table.device
    i = torch.arange(n, device=device)[None, :]
    source = torch.where(i < accepted[:, None], s["path"].long(), i)
    inside = (i < accepted[:, None]).reshape(-1)
    place = lambda x: (torch.gather(table, 1, ((cached[:, None] + x) // page).clamp(max=s["blocks"] - 1)).reshape(-1)[inside], ((cached[:, None] + x) % page).reshape(-1)[inside])  # noqa: E731
    (from_page, from_at), (to_page, to_at) = place(source), place(i.expand_as(source))
    s["cache"][:, :, to_page, :, to_at] = s["cache"][:, :, from_page, :, from_at]
    # pages of the step: the kept ones first, then those given back
    have, need, keep = -(-cached // page), -(-(cached + new) // page), -(-(cached + accepted) // page)
    column = torch.arange(s["blocks"], device=device)[None, :]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    kept = fresh & (column < keep[:, None])
    back = fresh & ~kept
    order = torch.where(kept, torch.cumsum(kept.reshape(-1).long(), 0).view_as(kept) - 1, kept.sum() + torch.cumsum(back.reshape(-1).long(), 0).view_as(back) - 1)
    s["free"][order[fresh]] = table[fresh].int()
    return {"cache": s["cache"], "kv_lens": (cached + accepted).int(), "used": kept.sum().int().reshape(1), "free": s["free"]}


# ---- one pass --------------------------------------------------------------------------------------------------------
def _device():
    """The program's one device handle and its stream."""
    global _backend, _stream
    if _backend is None:
        import lapid_b200 as lp
        _stream = torch.cuda.Stream()
        _backend = lp.Backend(0)
        _backend.set_stream(_stream.cuda_stream)
    return _backend


def _own_calls(s, c):
    """What a program sets up once: buffers over its tensors, the shape of its cache, the calls it repeats; and the step's plan, which its layers share."""
    from lapid_b200 import DType
    from lapid_b200.paged import Mask, PagedSpec, plan_bytes
    be = _device()
    kinds = {"f32": DType.F32, "f16": DType.F16, "bf16": DType.BF16}
    w = lambda t: be.wrap_tensor(t)  # noqa: E731
    new = lambda n: torch.empty(max(n, 4), dtype=torch.int32, device="cuda")  # noqa: E731
    verify = c["op"] == "verify"
    half = kinds[c["dtype"]] if c["op"] in ("attend", "commit") else DType.BF16
    spec = PagedSpec(dtype=half, q_heads=c.get("hq", c.get("hkv", 8)), kv_heads=c.get("hkv", 8), head_dim=c.get("d", 128), page_size=c.get("page", 16), pages=s.get("pages", c["requests"] * c["nodes"]),
                     requests=c["requests"], tokens=s["tokens"], max_blocks=s.get("blocks", c["nodes"]), max_new=c["nodes"], mask=Mask.TREE, window=c.get("window", 0))
    if verify:  # a cache with nothing in it yet
        cached = torch.zeros(c["requests"], dtype=torch.int32, device="cuda")
        table = torch.zeros(c["requests"], c["nodes"], dtype=torch.int32, device="cuda")
        free = torch.arange(spec.pages, dtype=torch.int32, device="cuda")
    else:
        cached, table, free = s["cached"], s["table"], s["free"].clone()
    slots, positions, kv_lens, used = new(s["tokens"]), new(s["tokens"]), new(c["requests"]), new(1)
    plan = be.wrap_tensor(torch.zeros(plan_bytes(spec), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    be.paged_plan(spec, w(s["new_lens"]), w(cached), w(table), w(slots), w(positions), w(kv_lens), w(used), plan, free_pages=w(free), n_free=s.get("n_free", free.numel()))
    be.synchronize()
    if c["op"] == "tree":
        s["call"] = be.packed_paged_tree(spec, plan, w(s["parents"]), w(s["positions"]), w(s["tree"]))
        s["result"] = {"positions": s["positions"], "tree": s["tree"]}
    elif c["op"] == "attend":
        tree = w(torch.zeros(s["tokens"], 1 + -(-c["nodes"] // 32), dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        be.paged_tree(spec, plan, w(s["parents"]), w(positions), tree)
        s["call"] = be.packed_paged_tree_attention(spec, plan, tree, w(s["q"]), w(s["k_cache"]), w(s["v_cache"]), w(s["table"]), w(s["out"]), lse=w(s["lse"]) if s["lse"] is not None else None)
        s["result"] = {"out": s["out"], "lse": s["lse"]}
    elif verify:
        s["call"] = be.packed_paged_verify(spec, plan, kinds[c["dtype"]], c["vocab"], w(s["logits"]), w(s["drafted"]), w(s["accept"]), w(s["pick"]), w(s["path"]), w(s["accepted"]), w(s["next"]),
                                           parents=w(s["parents"]), draft=w(s["draft"]) if s["draft"] is not None else None, temperature=w(s["temperature"]))
        s["result"] = {"path": s["path"], "accepted": s["accepted"], "next": s["next"]}
    else:
        layers = [(w(x[0]), w(x[1])) for x in s["cache"]]
        s["call"] = be.packed_paged_commit(spec, plan, layers, w(s["table"]), w(s["path"]), w(s["accepted"]), w(kv_lens), w(used), free_pages=w(s["free"]), n_free=s["n_free"])
        s["result"] = {"cache": s["cache"], "kv_lens": kv_lens[: c["requests"]], "used": used[:1], "free": s["free"]}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _own_calls(s, case)
    return s


def run(state):
    c = state["case"]
    if own:
        state["call"]()
        return state["result"]
    if c["op"] == "tree":
        return _tree(state, c)
    if c["op"] == "attend":
        return _attend(state, c)
    return _verify(state, c) if c["op"] == "verify" else _commit(state, c)


def _mean(most, part):
    return (int(part * most) + most) / 2


def work(case):
    """With the lengths' means: the seed draws them."""
    r, n = case["requests"], case["nodes"]
    if case["op"] == "verify":  # the rows on the path: some six in ten nodes with children have one accepted; where a chosen candidate fails the row is all that is read
        rows = sum(0.6 ** i for i in range(max(1, n // max(1, (case["branch"] + 1) // 2))))
        size = DTYPE[case["dtype"]].itemsize + (4 if case["draft"] else 0)
        return {"bytes": r * rows * case["vocab"] * size, "flops": r * rows * case["vocab"] * 4}
    tokens = r * max(1.0, _mean(n, case["spread"]))
    if case["op"] == "tree":
        return {"bytes": tokens * (4 + 4 + 4 * (1 + -(-n // 32))), "flops": tokens * n}
    if case["op"] == "commit":  # the first token of a path lies where it belongs
        moved = r * max(0.0, (1 + tokens / r / (1 + case["branch"]) * 2) / 2 - 1) * (case["branch"] > 1)
        return {"bytes": moved * case["layers"] * 2 * case["hkv"] * case["d"] * 2 * 2 + 8 * tokens, "flops": 0}
    cached, hq, hkv, d = _mean(case["cached"], case["ragged"]), case["hq"], case["hkv"], case["d"]
    seen = min(cached, case["window"]) if case["window"] else cached
    return {"bytes": 4 * (r * seen + tokens) * hkv * d + 4 * tokens * hq * d + (4 * tokens * hq if case["lse"] else 0),
            "flops": 4 * tokens * (seen + math.log2(1 + n)) * hq * d}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("tree", "verify"):
        return None  # whole numbers: the plain forms' are exact
    s = _inputs(case, seed)
    new, cached, page = s["new_lens"].tolist(), s["cached"].tolist(), case["page"]
    if case["op"] == "commit":
        cache = s["cache"].double()
        for r in range(case["requests"]):
            kept = s["path"][r, : int(s["accepted"][r])].tolist()
            at = [cached[r] + x for x in kept]
            slots = [(int(s["table"][r, x // page]), x % page) for x in at]
            rows = [s["cache"][:, :, p, :, o].double() for p, o in slots]
            for i, row in enumerate(rows):
                x = cached[r] + i
                cache[:, :, int(s["table"][r, x // page]), :, x % page] = row
        return {"cache": cache, "kv_lens": None, "used": None, "free": None}
    hq, hkv, d, window = case["hq"], case["hkv"], case["d"], case["window"]
    g = hq // hkv
    out = torch.zeros(s["tokens"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["tokens"], hq, dtype=torch.float64, device="cuda") if case["lse"] else None
    parents, at = s["parents"].tolist(), 0
    for r, (n, c) in enumerate(zip(new, cached)):
        kv = c + n
        hidden = torch.ones(n, kv, dtype=torch.bool)
        depth = []
        for t in range(n):
            depth.append(0 if parents[at + t] < 0 else depth[parents[at + t]] + 1)
            hidden[t, max(0, c + depth[t] + 1 - window) if window else 0 : c] = False
            x = t
            while x >= 0:
                hidden[t, c + x] = bool(window) and depth[t] - depth[x] >= window
                x = parents[at + x]
        hidden = hidden.cuda()
        used = s["table"][r, : -(-kv // page)].long()
        for h in range(hkv):
            k = s["k_cache"][used, h].double().reshape(-1, d)[:kv]
            v = s["v_cache"][used, h].double().reshape(-1, d)[:kv]
            score = (s["q"][at : at + n, h * g : (h + 1) * g].double().transpose(0, 1) @ k.T / d ** 0.5).masked_fill(hidden, -math.inf)
            out[at : at + n, h * g : (h + 1) * g] = (torch.softmax(score, -1) @ v).transpose(0, 1)
            if lse is not None:
                lse[at : at + n, h * g : (h + 1) * g] = torch.logsumexp(score, -1).T
        at += n
    return {"out": out, "lse": lse}
