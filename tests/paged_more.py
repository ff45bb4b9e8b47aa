"""More plain restatements for the paged cache's tests: the plan of a step with requests that take no part."""
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
