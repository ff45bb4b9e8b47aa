"""Plain restatements of what is done with drafted tokens over the paged cache, in Python integers and 64-bit floats, and the steps that the tests run."""
import math

import numpy as np

from lapid_b200.paged import Mask

from . import paged_ref as R


def random_parents(rng, n, branch, roots=0.0):
    """A parent in front of each token, at most ``branch`` places; the first has none, of the others the given part."""
    return [-1 if t == 0 or rng.random() < roots else max(0, t - int(rng.integers(1, branch + 1))) for t in range(n)]


def tree(parents, window=0):
    """Of each token how many ancestors it has, and the set of those that it sees (with itself): those nearer than the window."""
    depth, seen = [], []
    for t, p in enumerate(parents):
        depth.append(0 if p < 0 else depth[p] + 1)
        mine, x = set(), t
        while x >= 0:
            if not window or depth[t] - depth[x] < window:
                mine.add(x)
            x = parents[x]
        seen.append(mine)
    return depth, seen


def tree_words(parents, window, words):
    depth, seen = tree(parents, window)
    out = np.zeros((len(parents), 1 + words), np.uint32)
    for t, mine in enumerate(seen):
        out[t, 0] = depth[t]
        for i in mine:
            out[t, 1 + i // 32] |= np.uint32(1 << (i % 32))
    return out


def tree_attention(q, k, v, g, parents, window, scale, cached):
    """One request: q [n, hq, d], k and v [cached + n, hkv, d] in f64 -> out, lse, and sum p |v| / l, as ``paged_ref.attention``."""
    n, hq, d = q.shape
    depth, seen = tree(parents, window)
    out, lse, size = np.zeros((n, hq, d)), np.full((n, hq), -np.inf), np.zeros((n, hq, d))
    for t in range(n):
        lo = max(0, cached + depth[t] + 1 - window) if window else 0
        keys = list(range(min(lo, cached), cached)) + [cached + i for i in sorted(seen[t])]
        for h in range(hq):
            s = scale * (k[keys, h // g] @ q[t, h])
            m = s.max()
            p = np.exp(s - m)
            l = p.sum()
            out[t, h] = p @ v[keys, h // g] / l
            size[t, h] = p @ np.abs(v[keys, h // g]) / l
            lse[t, h] = m + math.log(l)
    return out, lse, size


class TreeStep(R.Step):
    """A step of drafted tokens: ``paged_ref.Step`` with parents (request by request)."""

    def __init__(self, be, parents, cached, **kw):
        super().__init__(be, [len(p) for p in parents], cached, mask=Mask.CAUSAL, **kw)
        self.parents, self.mask = [list(p) for p in parents], Mask.TREE
        from dataclasses import replace
        self.spec = replace(self.spec, mask=Mask.TREE)

    def upload(self):
        super().upload()
        from lapid_b200.paged import tree_bytes
        flat = [p for q in self.parents for p in q]
        pad = self.tokens - len(flat)
        self.b["parents"] = self.be.upload(np.array(flat + [7] * pad + [0], np.int32))
        self.b["tree"] = self.be.upload(np.full(max(16, tree_bytes(self.spec)), 0x5a, np.uint8))
        return self

    def make_plan(self):
        super().make_plan()
        self.be.paged_tree(self.spec, self.b["plan"], self.b["parents"], self.b["positions"], self.b["tree"])

    def attend(self, lse=True, **kw):
        b = self.b
        self.be.paged_tree_attention(self.spec, b["plan"], b["tree"], b["q"], b["k"], b["v"], b["table"], b["out"], lse=b["lse"] if lse else None, **kw)

    def tree_rows(self):
        words = 1 + -(-self.spec.max_new // 32)
        return self.b["tree"].download().view(np.uint32)[: self.tokens * words].reshape(self.tokens, words)

    def check(self, got=None, lse=True):
        out, got_lse = got or self.outputs()
        at = 0
        for r, n in enumerate(self.new):
            o, l, size = tree_attention(self.q[at:at + n], self.k[r], self.v[r], self.g, self.parents[r], self.window, self.scale, self.cached[r])
            vmax = float(np.abs(self.v[r]).max()) if self.v[r].size else 0.0
            err, most = np.abs(out[at:at + n] - o), R.bound(self.dtype, o, size, self.kv[r], vmax)
            assert np.all(err <= most), (r, float(err.max()), float((err / most).max()))
            if lse:
                assert np.all(np.abs(got_lse[at:at + n] - l) <= 1.5e-4 + 1e-6 * np.abs(l)), r
            at += n
        if self.tokens > at:  # rows behind the last token are left alone
            assert np.all(self.b["out"].download().view(np.int16).reshape(-1)[at * self.hq * self.d: self.tokens * self.hq * self.d] == 0x7e7e)


def verify(logits, parents, tokens, accept, pick, temperature, draft=None):
    """One request's walk: (path, next). ``logits`` f64 [n, vocab], ``draft`` f64 or None."""
    v, path = 0, [0]
    while True:
        z = logits[v]
        if np.isnan(z).any() or z.max() == np.inf or z.max() == -np.inf:
            return path, -1
        if not temperature > 0:
            p = np.zeros(len(z))
            p[int(np.argmax(z))] = 1.0
        else:
            with np.errstate(invalid="ignore"):
                p = np.where(z == -np.inf, 0.0, np.exp((z - z.max()) / temperature))
            p = p / math.fsum(p)
        step = None
        for c in range(v + 1, len(parents)):
            if parents[c] != v or not 0 <= tokens[c] < len(z):
                continue
            x = tokens[c]
            if accept[c] * (draft[v][x] if draft is not None else 1.0) < p[x]:
                step = c
                break
            if draft is not None:
                rest = np.maximum(p - draft[v], 0.0)
            else:
                rest = p.copy()
                rest[x] = 0.0
            total = math.fsum(rest)
            if total > 0:
                p = rest / total
        if step is None:
            run = np.cumsum(p)
            over = np.nonzero(run > pick * run[-1])[0]
            return path, int(over[0]) if len(over) else int(np.nonzero(p)[0][-1])
        path.append(step)
        v = step


def commit(new, cached, table, accepted, path, free, page):
    """(moves [(request, from, to)], kv_lens, used, free list)"""
    moves, kv, kept, back = [], [], [], []
    for r, (n, c) in enumerate(zip(new, cached)):
        a = accepted[r]
        moves += [(r, c + path[r][i], c + i) for i in range(a) if path[r][i] != i]
        kv.append(c + a)
        have, keep, need = -(-c // page), -(-(c + a) // page), -(-(c + n) // page)
        kept += [table[r][b] for b in range(have, keep)]
        back += [table[r][b] for b in range(keep, need)]
    return moves, kv, len(kept), kept + back + list(free[len(kept) + len(back):])
