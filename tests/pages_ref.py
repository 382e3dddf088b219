"""The operators on pages of a cache as loops over the tables, one entry after the other.  All of them change their arguments (lists) in place."""


def fork(table, held, kv, parents, children, free, num_free, shares, page_size):
    """Returns (moves [(from, to, tokens)], num_free, missing)."""
    was = [list(row) for row in table], list(held), list(kv)
    B, P = len(table), len(shares)
    width = len(table[0]) if table else 0
    moves, missing, named = [], 0, set()
    stack, taken = num_free, 0
    for p, c in zip(parents, children):
        if p < 0 or c < 0:
            if 0 <= c < B:
                named.add(c)
            continue
        again = c in named
        if c < B:
            named.add(c)
        if p >= B or c >= B or p == c or again or was[1][c] != 0:
            missing += 1
            continue
        pages = min(max(was[1][p], 0), width)
        n = min(max(was[2][p], 0), pages * page_size)
        full, part = divmod(n, page_size)
        for i in range(full):
            table[c][i] = was[0][p][i]
            if 0 <= was[0][p][i] < P:
                shares[was[0][p][i]] += 1
        held[c], kv[c] = full + (part > 0), n
        if part:
            src = was[0][p][full]
            if not 0 <= src < P:
                table[c][full] = -1
                continue
            taken += 1
            if taken > stack or not 0 <= free[stack - taken] < P:
                missing += 1
                held[c], kv[c] = full, full * page_size
                continue
            table[c][full] = free[stack - taken]
            moves.append((src, table[c][full], part))
    return moves, stack - min(taken, stack), missing


def free_pages(table, held, kv, free, num_free, shares, window, sinks, page_size):
    """Returns (num_free, freed); shares may be None."""
    P = len(shares) if shares is not None else 1 << 31
    width = len(table[0]) if table else 0
    back = []
    for b, row in enumerate(table):
        n, h = max(kv[b], 0), min(max(held[b], 0), width)
        end = min(-(-n // page_size), h)
        hole = range(-(-sinks // page_size), min(end, max(0, n - window + 1) // page_size)) if window > 0 else range(0)
        for c in range(h):
            if c >= end or c in hole:
                if 0 <= row[c] < P:
                    back.append(row[c])
                row[c] = -1
        held[b] = end
    count, seen, freed = {}, set(), 0
    for p in back:
        count[p] = count.get(p, 0) + 1
    for p in back:
        if shares is not None and count[p] <= shares[p] or shares is not None and p in seen:
            continue
        seen.add(p)
        if num_free + freed < len(free):
            free[num_free + freed] = p
        freed += 1
    if shares is not None:
        for p, n in count.items():
            shares[p] = 0 if p in seen else shares[p] - n
    return min(num_free + freed, len(free)), freed


def compact(table, held, free, num_free, shares, pages):
    """Returns (moves [(from, to)], num_free)."""
    live = {p for row, n in zip(table, held) for p in row[:max(n, 0)] if 0 <= p < pages}
    managed = sorted(live | {p for p in free[:num_free] if 0 <= p < pages})
    low, rest = managed[:len(live)], managed[len(live):]
    moves = list(zip(sorted(live - set(low)), sorted(set(low) - live)))
    to = dict(moves)
    for row, n in zip(table, held):
        row[:max(n, 0)] = [to.get(p, p) for p in row[:max(n, 0)]]
    if shares is not None:
        for a, b in moves:
            shares[b], shares[a] = shares[a], 0
    free[:len(rest)] = rest[::-1]
    return moves, len(rest)
