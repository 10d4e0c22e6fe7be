"""The pages of a cache, restated over lists: tables are lists of rows, counts a list, and
what moves is a list of (from page, to page, tokens)."""


def reach(n, page, most):
    return min(-(-max(n, 0) // page), most)


def fork(rows, lengths, counts, source, page):
    counts, most = list(counts), len(rows[0])
    held = [[p for p in row[:reach(n, page, most)]] for row, n in zip(rows, lengths)]
    for h in held:
        for p in h:
            if 0 <= p < len(counts):
                counts[p] -= 1
    out, new = [], []
    for b in source:
        h = held[b] if 0 <= b < len(rows) else []
        for p in h:
            if 0 <= p < len(counts):
                counts[p] += 1
        out.append(h + [-1] * (most - len(h)))
        new.append(lengths[b] if 0 <= b < len(rows) else 0)
    return out, new, counts


def resize(rows, lengths, counts, to, page):
    rows, counts, most, moves = [list(r) for r in rows], list(counts), len(rows[0]), []
    n = [min(max(x, 0), most * page) for x in lengths]
    to = [a if t < 0 else min(t, most * page) for a, t in zip(n, to)]
    for row, a, t in zip(rows, n, to):
        for e in range(reach(t, page, most), reach(a, page, most)):
            if 0 <= row[e] < len(counts):
                counts[row[e]] -= 1
    free = [p for p, c in enumerate(counts) if c == 0]
    before = list(counts)
    asked = 0
    for b, (row, a, t) in enumerate(zip(rows, n, to)):
        has, wants = reach(a, page, most), reach(t, page, most)
        last = row[has - 1] if has else -1
        copy = t > a and a % page != 0 and 0 <= last < len(counts) and before[last] > 1
        need = max(0, wants - has) + copy
        mine = free[asked:asked + need]
        asked += need
        if need and len(mine) < need:
            to[b], wants, mine, copy = a, has, [], False
        for p in mine:
            counts[p] = 1
        if copy:
            counts[last] -= 1
            row[has - 1] = mine.pop(0)
            moves.append((last, row[has - 1], a % page))
        for e in range(most):
            if e >= wants:
                row[e] = -1
            elif e >= has:
                row[e] = mine.pop(0)
    return rows, to, counts, moves


def compact(rows, counts):
    used = sum(c > 0 for c in counts)
    holes = [p for p in range(used) if counts[p] <= 0]
    movers = [p for p in range(used, len(counts)) if counts[p] > 0]
    where, counts = dict(zip(movers, holes)), list(counts)
    for a, b in where.items():
        counts[b], counts[a] = counts[a], 0
    return [[where.get(p, p) for p in row] for row in rows], counts, list(where.items())
