"""Which parts of which row tiles each block of the many-row attention over a cache has where the blocks share the work: the kernel's
own rule, restated, so that a test can say whether its batch has blocks with the sequence of parts that it is about."""

ROWS, POS, LEAST = 256, 128, 4  # query rows of a row tile, positions of a tile, a row tile costs at least a LEAST-th of the longest


def tiles(n, length, group, tile, window=0, sinks=0):
    """(rows, position tiles) of a row tile of an entry without a tree."""
    here = min(ROWS, n * group - tile * ROWS)
    if here <= 0:
        return 0, 0
    first = length - n
    lo, hi = tile * ROWS // group, (tile * ROWS + here - 1) // group
    low = max(first + lo - window, -1) if window else -1
    end = min(length, first + hi + 1)
    head = -(-min(end, sinks if window else 0) // POS) if end > 0 else 0
    main = max((low + 1) // POS, head)
    return here, head + max((-(-end // POS) if end > 0 else 0) - main, 0)


def parts(entries, heads, kvh, blocks, window=0, sinks=0):
    """Per block, in its order: (entry, row tile, head, rows, position tiles of the part, whether it is the whole row tile).
    ``entries``: (rows, length)."""
    group = heads // kvh
    per = -(-max(n for n, _ in entries) * group // ROWS)
    pairs = [(e, t, *tiles(n, length, group, t, window, sinks)) for e, (n, length) in enumerate(entries) for t in range(per)]
    raw = [max(p[3], 1) if p[2] else 0 for p in pairs]
    least = -(-max(raw) // LEAST)
    pre = [0]
    for c in raw:
        pre.append(pre[-1] + (max(c, least) if c else 0))
    total = pre[-1] * kvh
    count = min(blocks, total)
    out = []
    for b in range(count):
        at, end, mine = total * b // count, total * (b + 1) // count, []
        while at < end:
            p = next(i for i in range(len(pairs)) if pre[i + 1] * kvh > at)
            units = pre[p + 1] - pre[p]
            head, start = divmod(at - pre[p] * kvh, units)
            take = min(units - start, end - at)
            e, t, rows, n = pairs[p]
            mine.append((e, t, head, rows, n * (start + take) // units - n * start // units, take == units))
            at += take
        out.append(mine)
    return out
