"""The paged key/value cache and the attention over it: what lies between the projections of a decoder layer.

``listed()`` gives the cases that are always timed, ``draw(rng)`` more of the same ranges, ``prepare(case, seed)`` what a
serving program holds before the call, ``run(state)`` one pass, ``work(case)`` the bytes and operations that a pass
cannot do without, ``exact(case, seed)`` the outputs from the definitions in 64 bits.

Operators (``op``):

  plan    once a step: block table entries, slot and position of every new token, from the requests' lengths
  append  once a layer: rotary embedding of q and k, rounding to the cache's type, k and v stored at their slots
  attend  once a layer: attention of every request's new tokens over its cached and its new keys

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits; with ``own`` true it makes the
framework's calls. Inputs are synthetic, made on the GPU from the seed.
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_backend = None
_stream = None


def listed():
    return [
        # a decode step of a server with 64 users: 64 lengths to 64 slots, now and then a page
        {"name": "plan_decode_r64", "op": "plan", "requests": 64, "new": 1, "spread": 1.0, "cached": 4096, "ragged": 0.9, "page": 16},
        # a step full of prompts, some behind a cached beginning
        {"name": "plan_prompts_r48", "op": "plan", "requests": 48, "new": 1365, "spread": 0.8, "cached": 1024, "ragged": 1.0, "page": 64},
        # eight users' tokens of one layer: latency
        {"name": "append_decode_b8", "op": "append", "tokens": 8, "src": "f32", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128, "page": 16, "rot": 128, "pairs": "halves"},
        # 8192 tokens of prompts, f32 rows as the projections leave them
        {"name": "append_prompt_8192", "op": "append", "tokens": 8192, "src": "f32", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128, "page": 64, "rot": 128, "pairs": "halves"},
        # an odd number of tokens of a model with small heads, part of each rotated, neighbouring pairs
        {"name": "append_odd_d64", "op": "append", "tokens": 1531, "src": "f16", "dtype": "f16", "hq": 16, "hkv": 16, "d": 64, "page": 32, "rot": 32, "pairs": "neighbours"},
        # one user, one token, a context of a few pages' worth of screens: latency
        {"name": "decode_b1_4k", "op": "attend", "requests": 1, "new": 1, "spread": 1.0, "cached": 4095, "ragged": 1.0, "page": 16, "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128, "mask": "causal", "window": 0, "lse": False},
        # 64 users, one token each, contexts of all lengths: the usual decode step
        {"name": "decode_b64_ragged", "op": "attend", "requests": 64, "new": 1, "spread": 1.0, "cached": 8192, "ragged": 0.1, "page": 16, "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128, "mask": "causal", "window": 0, "lse": False},
        # two users with a very long context, the heads of a large model: split over the keys; the sums' logarithm goes out too
        {"name": "decode_b2_128k", "op": "attend", "requests": 2, "new": 1, "spread": 1.0, "cached": 131071, "ragged": 0.9, "page": 64, "dtype": "f16", "hq": 64, "hkv": 8, "d": 128, "mask": "causal", "window": 0, "lse": True},
        # whole prompts of different lengths in one call
        {"name": "prompts_ragged", "op": "attend", "requests": 4, "new": 4096, "spread": 0.4, "cached": 0, "ragged": 1.0, "page": 64, "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128, "mask": "causal", "window": 0, "lse": False},
        # the next 512 tokens of a long document, the heads of a large model
        {"name": "chunk_512_over_32k", "op": "attend", "requests": 1, "new": 512, "spread": 1.0, "cached": 32255, "ragged": 1.0, "page": 16, "dtype": "bf16", "hq": 64, "hkv": 8, "d": 128, "mask": "causal", "window": 0, "lse": False},
        # one chunk of a prompt beside eleven users who decode
        {"name": "mixed_12", "op": "attend", "requests": 12, "new": 512, "spread": 0.0, "cached": 4096, "ragged": 0.2, "page": 32, "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128, "mask": "causal", "window": 0, "lse": False},
        # prompts through a layer with a sliding window and small heads, odd group
        {"name": "window_d64", "op": "attend", "requests": 3, "new": 3001, "spread": 0.7, "cached": 2047, "ragged": 0.5, "page": 32, "dtype": "f16", "hq": 14, "hkv": 2, "d": 64, "mask": "causal", "window": 1024, "lse": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (64, 8, 128), (16, 4, 64), (8, 8, 128), (28, 4, 128), (14, 2, 64), (12, 4, 96), (8, 1, 128), (16, 16, 64), (20, 5, 80)]


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        r = _log_int(rng, 1, 2048)
        return {"op": op, "requests": r, "new": _log_int(rng, 1, max(1, 65536 // r)), "spread": rng.choice([0.0, 0.5, 1.0]), "cached": _log_int(rng, 1, 8192),
                "ragged": rng.choice([0.0, 0.5, 1.0]), "page": page}
    hq, hkv, d = rng.choice(HEADS)
    if op == "append":
        return {"op": op, "tokens": _log_int(rng, 1, 8192), "src": rng.choice(["f32", "f32", "f16", "bf16"]), "dtype": rng.choice(["f16", "bf16"]), "hq": min(hq, 32), "hkv": hkv if hq <= 32 else 4,
                "d": d, "page": page, "rot": rng.choice([0, 32, d]), "pairs": rng.choice(["halves", "neighbours"])}
    kind = rng.choice(["decode", "prompt", "chunk", "mixed"])
    if kind == "decode":  # at most as many keys as the largest listed case has
        r = _log_int(rng, 1, 64)
        new, spread, cached = rng.choice([1, 1, 1, 2, 4]), 1.0, _log_int(rng, 32, min(65536, 262144 // r))
    elif kind == "prompt":
        r = rng.randint(1, 4)
        new, spread, cached = _log_int(rng, 17, 4096), rng.choice([0.3, 1.0]), 0
    elif kind == "chunk":
        r = rng.randint(1, 2)
        new, spread, cached = _log_int(rng, 16, 512), 1.0, _log_int(rng, 128, 16384)
    else:
        r = rng.randint(2, 12)
        new, spread, cached = _log_int(rng, 32, 512), 0.0, _log_int(rng, 64, 4096)
    mask = rng.choice(["causal", "causal", "causal", "full", "cross"])
    if mask == "cross" and cached == 0:
        cached = _log_int(rng, 16, 2048)
    case = {"op": "attend", "requests": r, "new": new, "spread": spread, "cached": cached, "ragged": rng.choice([0.2, 0.6, 1.0]), "page": page, "dtype": rng.choice(["f16", "bf16"]),
            "hq": hq, "hkv": hkv, "d": d, "mask": mask, "window": rng.choice([0, 0, 127, 1024]) if mask == "causal" else 0, "lse": rng.random() < 0.3}
    while work(case)["flops"] > 5.0e11:  # no more than the largest listed case
        case["new"] = case["new"] * 3 // 4
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _between(most, part, count, gen, device):
    """``count`` whole numbers from ``part * most`` to ``most``."""
    lo = int(part * most)
    return (lo + (torch.rand(count, generator=gen, device=device) * (most - lo + 1)).long()).clamp(max=most)


def _lens(case, gen, device):
    r, new = case["requests"], case["new"]
    if case["spread"] == 0.0:  # one request with a chunk, the others with one token each
        new_lens = torch.ones(r, dtype=torch.long, device=device)
        new_lens[r // 2] = new
    else:
        new_lens = _between(new, case["spread"], r, gen, device).clamp(min=1)
    return new_lens, _between(case["cached"], case["ragged"], r, gen, device)


def _sizes(case):
    """The lengths that the seed does not change: upper bounds, so that every state of a case has the same shapes."""
    page, r = case["page"], case["requests"]
    tokens = r - 1 + case["new"] if case["spread"] == 0.0 else r * case["new"]
    blocks = -(-(case["cached"] + case["new"]) // page)
    return tokens, blocks


def _requests(case, gen, device):
    """Lengths, the block table as the step before left it, and the list of free pages, in an order of their own."""
    new_lens, cached = _lens(case, gen, device)
    tokens, blocks = _sizes(case)
    page, r = case["page"], case["requests"]
    pages = r * blocks + 3
    order = torch.randperm(pages, generator=gen, device=device)
    table = order[: r * blocks].reshape(r, blocks)
    have = -(-cached // page)
    taken = torch.arange(blocks, device=device)[None, :] < have[:, None]
    free = torch.cat([table[~taken], order[r * blocks:]])
    free = free[torch.randperm(free.numel(), generator=gen, device=device)]
    padded = torch.full((pages,), -1, dtype=torch.int32, device=device)  # the list has room for every page; its first entries count
    padded[: free.numel()] = free.int()
    return {"new_lens": new_lens.int(), "cached": cached.int(), "table": torch.where(taken, table, -1).int().contiguous(), "free": padded, "n_free": free.numel(),
            "tokens": tokens, "blocks": blocks, "pages": pages}


def _rope_table(positions, rot, device):
    """[positions, rot]: cos of the rot / 2 angles, then their sin."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / max(rot, 1))
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq[None, :]
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def _inputs(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=device)  # noqa: E731
    if case["op"] == "plan":
        return _requests(case, gen, device)
    dtype = DTYPE[case["dtype"]]
    if case["op"] == "append":
        t, hq, hkv, d, page = case["tokens"], case["hq"], case["hkv"], case["d"], case["page"]
        pages = -(-t // page) + 8
        src = DTYPE[case["src"]]
        slots = torch.randperm(pages * page, generator=gen, device=device)[:t]
        if t > 64:  # prompts: whole pages in an order of their own, filled from front to back
            order = torch.randperm(pages, generator=gen, device=device)
            at = torch.arange(t, device=device)
            slots = order[at // page] * page + at % page
        limit = max(2 * t, 4096)
        first = int(seed) % 97
        positions = (torch.arange(t, device=device) + first) if t > 64 else torch.randint(0, limit, (t,), generator=gen, device=device)
        return {"q": normal(t, hq * d).to(src), "k": normal(t, hkv * d).to(src), "v": normal(t, hkv * d).to(src), "slots": slots.int(), "positions": positions.int(),
                "rope": _rope_table(limit, case["rot"], device), "k_cache": normal(pages, hkv, page, d).to(dtype), "v_cache": normal(pages, hkv, page, d).to(dtype),
                "q_out": torch.zeros(t, hq, d, dtype=dtype, device=device), "pages": pages, "limit": limit}
    s = _requests(case, gen, device)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    s["table"], _, _, s["kv_lens"], _ = _plan(s, page, case["mask"] == "cross")
    s["q"] = normal(s["tokens"], hq, d).to(dtype)
    s["k_cache"] = torch.empty(s["pages"], hkv, page, d, dtype=dtype, device=device).normal_(generator=gen)
    s["v_cache"] = torch.empty(s["pages"], hkv, page, d, dtype=dtype, device=device).normal_(generator=gen)
    s["k_cache"] *= 1.5  # some keys stand out, as they do in trained heads
    s["out"] = torch.zeros(s["tokens"], hq, d, dtype=dtype, device=device)
    s["lse"] = torch.zeros(s["tokens"], hq, dtype=torch.float32, device=device) if case["lse"] else None
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plan(s, page, cross=False):
    """Block table, slots, positions, lengths of the keys, and how many pages the step took."""
    new, cached, table = s["new_lens"].long(), s["cached"].long(), s["table"]
    device, blocks, tokens = table.device, s["blocks"], s["tokens"]
    kv = cached if cross else cached + new
    have, need = -(-cached // page), -(-kv // page)
    first = torch.cumsum(need - have, 0) - (need - have)
    column = torch.arange(blocks, device=device)[None, :]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    at = (first[:, None] + column - have[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][at], table)
    end = torch.cumsum(new, 0)
    token = torch.arange(tokens, device=device)
    request = torch.searchsorted(end, token, right=True)
    real = request < new.numel()
    request = request.clamp(max=new.numel() - 1)
    position = cached[request] + token - (end - new)[request]
    block = (position // page).clamp(max=blocks - 1)
    slot = table[request, block].long() * page + position % page
    stored = real & (not cross)
    return table, torch.where(stored, slot, -1).int(), torch.where(real, position, -1).int(), kv.int(), (need - have).sum().int().reshape(1)


def _rotate(x, cos, sin, rot, pairs):
    if rot == 0:
        return x
    turned, rest = x[..., :rot], x[..., rot:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if pairs == "halves":
        a, b = turned[..., : rot // 2], turned[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _append(s, c):
    t, hq, hkv, d, page, rot = c["tokens"], c["hq"], c["hkv"], c["d"], c["page"], c["rot"]
    dtype = DTYPE[c["dtype"]]
    angles = s["rope"][s["positions"].long()]
    cos, sin = angles[:, : rot // 2], angles[:, rot // 2:]
    q = _rotate(s["q"].float().view(t, hq, d), cos, sin, rot, c["pairs"]).to(dtype)
    k = _rotate(s["k"].float().view(t, hkv, d), cos, sin, rot, c["pairs"]).to(dtype)
    v = s["v"].float().view(t, hkv, d).to(dtype)
    slots = s["slots"].long()
    s["k_cache"][slots // page, :, slots % page] = k
    s["v_cache"][slots // page, :, slots % page] = v
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend(s, c):
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    g = hq // hkv
    new, kv = s["new_lens"].long(), s["kv_lens"].long()
    r, most_new, blocks, device = new.numel(), c["new"], s["blocks"], new.device
    end = torch.cumsum(new, 0)
    row = torch.arange(most_new, device=device)
    real = row[None, :] < new[:, None]                                                 # [r, n]
    at = ((end - new)[:, None] + row[None, :]).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[at].view(r, most_new, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, g * most_new, d)
    pages = s["table"].long().clamp(min=0)                                             # [r, blocks]
    k = s["k_cache"][pages].float().permute(0, 2, 1, 3, 4).reshape(r, hkv, blocks * page, d)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(r, hkv, g, most_new, blocks * page)
    del k
    key = torch.arange(blocks * page, device=device)
    hi = (kv - new)[:, None] + row[None, :] + 1 if c["mask"] == "causal" else kv[:, None].expand(r, most_new)
    lo = (hi - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(hi)
    seen = (key[None, None, :] < hi[:, :, None]) & (key[None, None, :] >= lo[:, :, None])
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
    """What a program sets up once: buffers over its tensors, the shape of its cache, the calls it repeats."""
    from lapid_b200 import DType
    from lapid_b200.paged import Mask, PagedSpec, plan_bytes
    be = _device()
    kinds = {"f32": DType.F32, "f16": DType.F16, "bf16": DType.BF16}
    w = lambda t: be.wrap_tensor(t)  # noqa: E731
    new = lambda n: torch.empty(max(n, 4), dtype=torch.int32, device="cuda")  # noqa: E731
    if c["op"] == "append":
        spec = PagedSpec(dtype=kinds[c["dtype"]], q_heads=c["hq"], kv_heads=c["hkv"], head_dim=c["d"], page_size=c["page"], pages=s["pages"], requests=c["tokens"], tokens=c["tokens"],
                         max_blocks=1, max_new=1)
        s["call"] = be.packed_paged_append(spec, kinds[c["src"]], w(s["q"]), w(s["k"]), w(s["v"]), w(s["slots"]), w(s["positions"]), w(s["k_cache"]), w(s["v_cache"]), w(s["q_out"]),
                                           rope=w(s["rope"]) if c["rot"] else None, rope_rows=s["limit"], rot=c["rot"], neighbours=c["pairs"] == "neighbours")
        s["result"] = {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return
    attend = c["op"] == "attend"
    spec = PagedSpec(dtype=kinds[c.get("dtype", "bf16")], q_heads=c.get("hq", 32), kv_heads=c.get("hkv", 8), head_dim=c.get("d", 128), page_size=c["page"], pages=s["pages"],
                     requests=c["requests"], tokens=s["tokens"], max_blocks=s["blocks"], max_new=c["new"], mask=Mask[c.get("mask", "causal").upper()], window=c.get("window", 0))
    slots, positions, kv_lens, used = new(s["tokens"]), new(s["tokens"]), new(c["requests"]), new(1)
    plan = be.wrap_tensor(torch.zeros(plan_bytes(spec), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    make = be.packed_paged_plan(spec, w(s["new_lens"]), w(s["cached"]), w(s["table"]), w(slots), w(positions), w(kv_lens), w(used), plan, free_pages=w(s["free"]), n_free=s["n_free"])
    s["call"] = make
    s["result"] = {"table": s["table"], "slots": slots[: s["tokens"]], "positions": positions[: s["tokens"]], "kv_lens": kv_lens[: c["requests"]], "used": used[:1]}
    if attend:
        make()  # a step's plan serves all of its layers
        s["call"] = be.packed_paged_attention(spec, plan, w(s["q"]), w(s["k_cache"]), w(s["v_cache"]), w(s["table"]), w(s["out"]), lse=w(s["lse"]) if s["lse"] is not None else None)
        s["result"] = {"out": s["out"], "lse": s["lse"]}


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
    if c["op"] == "plan":
        table, slots, positions, kv_lens, used = _plan(state, c["page"])
        return {"table": table, "slots": slots, "positions": positions, "kv_lens": kv_lens, "used": used}
    return _append(state, c) if c["op"] == "append" else _attend(state, c)


def _mean(most, part):
    return (int(part * most) + most) / 2


def work(case):
    """With the lengths' means: the seed draws them."""
    if case["op"] == "append":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        src = DTYPE[case["src"]].itemsize
        return {"bytes": t * ((hq + 2 * hkv) * d * (src + 2) + 4 * case["rot"] + 8), "flops": 3 * t * (hq + hkv) * case["rot"]}
    r, page = case["requests"], case["page"]
    cached = _mean(case["cached"], case["ragged"])
    lens = [case["new"]] + [1] * (r - 1) if case["spread"] == 0.0 else [max(1.0, _mean(case["new"], case["spread"]))] * r
    tokens = sum(lens)
    if case["op"] == "plan":
        return {"bytes": 12 * r + 8 * tokens + 8 * tokens / page, "flops": 4 * tokens}
    pairs, keys = 0.0, 0.0
    for n in lens:
        kv = cached if case["mask"] == "cross" else cached + n
        if case["mask"] != "causal":
            pairs, keys = pairs + n * kv, keys + kv
        elif not case["window"]:
            pairs, keys = pairs + n * cached + n * (n + 1) / 2, keys + kv
        else:  # row t sees min(cached + t, window) keys
            full = min(n, max(0.0, case["window"] - cached))
            pairs += full * cached + full * (full + 1) / 2 + (n - full) * case["window"]
            keys += min(kv, n + case["window"] - 1)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    return {"bytes": 4 * keys * hkv * d + 4 * tokens * hq * d + (4 * tokens * hq if case["lse"] else 0), "flops": 4 * pairs * hq * d}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers: the plain form's are exact
    if case["op"] == "append":
        t, hq, hkv, d, rot, page = case["tokens"], case["hq"], case["hkv"], case["d"], case["rot"], case["page"]
        index = torch.arange(d, device="cuda")
        half = case["pairs"] == "halves"
        partner, sign, angle = index.clone(), torch.zeros(d, dtype=torch.float64, device="cuda"), torch.zeros(d, dtype=torch.long, device="cuda")
        for i in range(rot // 2):
            a, b = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
            partner[a], partner[b], sign[a], sign[b], angle[a], angle[b] = b, a, -1.0, 1.0, i, i
        table = s["rope"].double()[s["positions"].long()]
        cos, sin = torch.ones(t, d, dtype=torch.float64, device="cuda"), torch.zeros(t, d, dtype=torch.float64, device="cuda")
        if rot:
            cos[:, :rot], sin[:, :rot] = table[:, angle[:rot]], table[:, rot // 2 + angle[:rot]]
        turn = lambda x: x * cos[:, None] + x[..., partner] * (sin * sign)[:, None]  # noqa: E731
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        k, v = turn(s["k"].double().view(t, hkv, d)), s["v"].double().view(t, hkv, d)
        slot = s["slots"].long()
        kc, vc = kc.transpose(1, 2).contiguous(), vc.transpose(1, 2).contiguous()
        kc.view(-1, hkv, d)[slot], vc.view(-1, hkv, d)[slot] = k, v
        return {"q": turn(s["q"].double().view(t, hq, d)), "k_cache": kc.transpose(1, 2).contiguous(), "v_cache": vc.transpose(1, 2).contiguous()}
    hq, hkv, d, page, mask = case["hq"], case["hkv"], case["d"], case["page"], case["mask"]
    g = hq // hkv
    out = torch.zeros(s["tokens"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["tokens"], hq, dtype=torch.float64, device="cuda") if case["lse"] else None
    at = 0
    for r, (n, kv) in enumerate(zip(s["new_lens"].tolist(), s["kv_lens"].tolist())):
        used = s["table"][r, : -(-kv // page)].long()
        for h in range(hkv):
            k = s["k_cache"][used, h].double().reshape(-1, d)[:kv]
            v = s["v_cache"][used, h].double().reshape(-1, d)[:kv]
            for t0 in range(0, n, 1024):
                t1 = min(n, t0 + 1024)
                q = s["q"][at + t0 : at + t1, h * g : (h + 1) * g].double().transpose(0, 1)      # [g, rows, d]
                score = q @ k.T / d ** 0.5
                if mask == "causal":
                    last = kv - n + torch.arange(t0, t1, device="cuda")[:, None]
                    j = torch.arange(kv, device="cuda")[None, :]
                    out_of = (j > last) | ((j <= last - case["window"]) if case["window"] else False)
                    score = score.masked_fill(out_of, -math.inf)
                if kv:
                    out[at + t0 : at + t1, h * g : (h + 1) * g] = (torch.softmax(score, -1) @ v).transpose(0, 1)
                if lse is not None:
                    lse[at + t0 : at + t1, h * g : (h + 1) * g] = torch.logsumexp(score, -1).T if kv else -math.inf
        at += n
    return {"out": out, "lse": lse}
