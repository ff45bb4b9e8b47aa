"""More plain restatements for the paged cache's tests: the plan of a step with requests that take no part, and how far the logarithm of a softmax's sum may be off."""
import math

import numpy as np


def plan_with_refusals(new, cached, table, free, page, max_blocks, max_new, tokens, cross=False):
    """(table, slots, positions, kv_lens, used, which take part) from the definition, request by request. A request's rows begin behind the new lengths before it (those
    from 0 to max_new); one whose lengths are outside the bounds, or whose rows pass `tokens`, keeps its rows, its pages and its length as they are. A free page that is
    -1 is none."""
    table, kv, part, used, start = table.copy(), [], [], 0, 0
    slots, positions = np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32)
    for r, (n, c) in enumerate(zip(new, cached)):
        at, rows = start, n if 0 <= n <= max_new else 0
        start += rows
        end = c if cross else c + n
        ok = n == rows and c >= 0 and -(-end // page) <= max_blocks and (n == 0 or start <= tokens)
        part.append(ok)
        kv.append(end if ok else c)
        if not ok:
            continue
        for b in range(-(-c // page), -(-end // page)):
            table[r, b] = free[used] if used < len(free) else -1
            used += 1
        for t in range(n):
            positions[at + t] = c + t
            block = table[r, (c + t) // page] if not cross else -1
            slots[at + t] = block * page + (c + t) % page if block >= 0 else -1
    return table, slots, positions, np.array(kv, np.int32), used, part


POLYNOMIAL = 2.9e-6   # largest relative error of the exponentials that are a polynomial (of degree 4)


def lse_bound(lse, top, keys):
    """For scores q . k that f32 holds without rounding, `top` the largest of them in size, times the scale. Relative errors of the sum: the exponentials', and a rounding for each of
    the `keys` summands. Absolute ones, in units of 2^-24 of the largest number there: the scale times log2 e, its product with a score, the difference from the maximum, log2 of the sum (two units), the last product;
    each counted twice, for a maximum and a score."""
    return POLYNOMIAL + 2.0 ** -22 + keys * 2.0 ** -24 + 12 * 2.0 ** -24 * (np.abs(lse) + top + 1.0)


def exp2_polynomial(degree):
    """2^x as n + f with |f| <= 1/2 and a polynomial in f: Chebyshev interpolation, within a few percent of the best of its degree."""
    from numpy.polynomial import chebyshev
    c = chebyshev.Chebyshev.interpolate(lambda f: np.exp2(f), degree, domain=[-0.5, 0.5])

    def f(x):
        n = np.rint(x)
        return c(x - n) * np.exp2(n)
    return f


def lse_with(exp2, scores):
    """The logarithm of the sum in 64 bits but for the exponential."""
    m = scores.max()
    return m + math.log(exp2((scores - m) / math.log(2.0)).sum())
