"""Plain restatements of the paged cache's three operators, in Python integers and 64-bit floats, and the steps that the tests run."""
import math

import numpy as np

import lapid_b200 as lp
from lapid_b200.paged import Mask, PagedSpec, plan_bytes

U = {lp.DType.BF16: 2.0 ** -8, lp.DType.F16: 2.0 ** -11}   # largest relative rounding error of the type


def plan(new, cached, table, free, n_free, page, max_blocks, tokens, cross=False):
    """(table, slots, positions, kv_lens, used) from the definition, request by request."""
    table, slots, positions, kv, used = table.copy(), [], [], [], 0
    for r, (n, c) in enumerate(zip(new, cached)):
        end = c if cross else c + n
        kv.append(end)
        for b in range(-(-c // page), -(-end // page)):
            table[r, b] = free[used] if used < n_free else -1
            used += 1
        for t in range(n):
            positions.append(c + t)
            block = table[r, (c + t) // page] if not cross else -1
            slots.append(block * page + (c + t) % page if block >= 0 else -1)
    pad = [-1] * (tokens - len(slots))
    return table, np.array(slots + pad, np.int32), np.array(positions + pad, np.int32), np.array(kv, np.int32), used


def seen(mask, window, n, kv, t):
    """The keys [lo, hi) that new token t of n sees among kv."""
    hi = max(0, kv - (n - 1 - t)) if mask == Mask.CAUSAL else kv
    return (max(0, hi - window) if window else 0), hi


def attention(q, k, v, g, mask, window, scale, n, kv):
    """One request: q [n, hq, d], k and v [kv, hkv, d] in f64 -> out [n, hq, d], lse [n, hq], and sum p |v| / l [n, hq, d]."""
    hq, d = q.shape[1:]
    out, lse, size = np.zeros((n, hq, d)), np.full((n, hq), -np.inf), np.zeros((n, hq, d))
    for t in range(n):
        lo, hi = seen(mask, window, n, kv, t)
        if hi <= lo:
            continue
        for h in range(hq):
            s = scale * (k[lo:hi, h // g] @ q[t, h])
            m = s.max()
            if m == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                p = np.exp(s - m)
            l = p.sum()
            out[t, h] = p @ v[lo:hi, h // g] / l
            size[t, h] = p @ np.abs(v[lo:hi, h // g]) / l
            lse[t, h] = m + math.log(l) if l == l else np.nan
    return out, lse, size


def bound(dtype, out, size, keys, vmax):
    """How far a result may be off: the softmax's weights are rounded to the cache's type (one unit each, and in f16 2^-25 where they are below its smallest
    normal number) and so is the result; the f32 sums, the scores' rounding and the exponential are given 1e-4 of sum p |v| / l."""
    u = U[dtype]
    tiny = keys * 2.0 ** -25 * vmax if dtype == lp.DType.F16 else 0.0
    return u * np.abs(out) + (u * 1.01 + 1e-4) * size + tiny + 1e-30


def to_half(x, dtype):
    """f64 -> the values of the cache's type, and their bits."""
    import torch
    t = torch.from_numpy(np.asarray(x, np.float64)).float().to(torch.bfloat16 if dtype == lp.DType.BF16 else torch.float16)
    return t.double().numpy(), t.view(torch.int16).numpy()


def from_half(bits, dtype):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(bits).view(np.int16).copy()).view(torch.bfloat16 if dtype == lp.DType.BF16 else torch.float16)
    return t.double().numpy()


class Step:
    """A step of `new` tokens behind `cached` ones: a cache whose pages lie in a random order, with NaN wherever no token is."""

    def __init__(self, be, new, cached, *, dtype=lp.DType.BF16, hq=4, hkv=2, d=64, page=16, mask=Mask.CAUSAL, window=0, scale=0.0, seed=1, pad=0, max_new=None,
                 spread=1.0):
        rng = np.random.default_rng(seed)
        self.be, self.new, self.cached, self.dtype, self.mask, self.window = be, list(new), list(cached), dtype, mask, window
        kv = [c if mask == Mask.CROSS else c + n for n, c in zip(new, cached)]
        self.kv, self.hq, self.hkv, self.g, self.d, self.page = kv, hq, hkv, hq // hkv, d, page
        r, tokens = len(new), sum(new) + pad
        blocks = max([1] + [-(-x // page) for x in kv]) + 1
        pages = sum(-(-x // page) for x in kv) + 3
        order = rng.permutation(pages).astype(np.int32)
        table, at = np.full((r, blocks), -1, np.int32), 0
        for i, c in enumerate(cached):
            have = -(-c // page)
            table[i, :have] = order[at:at + have]
            at += have
        self.table0, self.free, self.tokens, self.blocks, self.pages = table, order[at:].copy(), tokens, blocks, pages
        self.spec = PagedSpec(dtype=dtype, q_heads=hq, kv_heads=hkv, head_dim=d, page_size=page, pages=pages, requests=r, tokens=tokens, max_blocks=blocks,
                              max_new=max_new or max([1] + list(new)), mask=mask, window=window, scale=scale)
        self.scale = scale or 1.0 / math.sqrt(d)
        self.q, self.q_bits = to_half(rng.normal(size=(tokens, hq, d)) * spread, dtype)
        self.k = [to_half(rng.normal(size=(x, hkv, d)) * spread, dtype)[0] for x in kv]
        self.v = [to_half(rng.normal(size=(x, hkv, d)), dtype)[0] for x in kv]

    def upload(self):
        be = self.be
        self.want = plan(self.new, self.cached, self.table0, self.free, len(self.free), self.page, self.blocks, self.tokens, self.mask == Mask.CROSS)
        kc = np.full((self.pages, self.hkv, self.page, self.d), np.nan)
        vc = kc.copy()
        for r, x in enumerate(self.kv):
            for j in range(x):
                p = self.want[0][r, j // self.page]
                kc[p, :, j % self.page], vc[p, :, j % self.page] = self.k[r][j], self.v[r][j]
        z = lambda n: be.upload(np.zeros(max(1, n), np.int32))
        self.b = {"new": be.upload(np.array(self.new, np.int32)), "cached": be.upload(np.array(self.cached, np.int32)), "table": be.upload(self.table0),
                  "free": be.upload(self.free), "slots": z(self.tokens), "positions": z(self.tokens), "kv": z(len(self.new)), "used": z(1),
                  "plan": be.alloc(plan_bytes(self.spec)), "k": be.upload(to_half(kc, self.dtype)[1]), "v": be.upload(to_half(vc, self.dtype)[1]),
                  "q": be.upload(self.q_bits), "out": be.upload(np.full(max(1, self.tokens * self.hq * self.d), 0x7e7e, np.int16)),
                  "lse": be.upload(np.full(max(1, self.tokens * self.hq), 77.0, np.float32))}
        return self

    def make_plan(self):
        b = self.b
        self.be.paged_plan(self.spec, b["new"], b["cached"], b["table"], b["slots"], b["positions"], b["kv"], b["used"], b["plan"], free_pages=b["free"], n_free=len(self.free))

    def attend(self, lse=True, **kw):
        b = self.b
        self.be.paged_attention(self.spec, b["plan"], b["q"], b["k"], b["v"], b["table"], b["out"], lse=b["lse"] if lse else None, **kw)

    def outputs(self):
        n = self.tokens * self.hq
        return (from_half(self.b["out"].download().view(np.int16)[: n * self.d], self.dtype).reshape(self.tokens, self.hq, self.d),
                self.b["lse"].download().view(np.float32)[:n].astype(np.float64).reshape(self.tokens, self.hq))

    def check(self, got=None, lse=True):
        out, got_lse = got or self.outputs()
        at = 0
        for r, n in enumerate(self.new):
            o, l, size = attention(self.q[at:at + n], self.k[r], self.v[r], self.g, self.mask, self.window, self.scale, n, self.kv[r])
            vmax = float(np.abs(self.v[r]).max()) if self.v[r].size else 0.0
            err, most = np.abs(out[at:at + n] - o), bound(self.dtype, o, size, self.kv[r], vmax)
            assert np.all(err <= most), (r, float(err.max()), float((err / most).max()))
            if lse:
                x, y = got_lse[at:at + n], l
                assert np.array_equal(np.isneginf(x), np.isneginf(y)), r
                f = np.isfinite(y)
                assert np.all(np.abs(x[f] - y[f]) <= 1.5e-4 + 1e-6 * np.abs(y[f])), (r, float(np.abs(x[f] - y[f]).max()))
            at += n

    def run(self, lse=True):
        self.upload()
        self.make_plan()
        self.attend(lse)
        self.be.synchronize()
        self.check(lse=lse)
        return self
