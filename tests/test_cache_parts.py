"""Batches of single tokens, prompts and empty sequences whose work the blocks of the many-row attention share: sequences of parts in
one block after which a hand-over could be taken for the one before it (a barrier's wait knows only a phase's parity).

Bound per output as in test_gpu_cache_many_rows."""
import math

import pytest
import torch

from cache_parts import parts
from cache_util import Cache, check, i32, queries, run_attention
from test_gpu_cache_many_rows import _both, _entries, oracle

SMS = 148  # blocks that share the work
two = lambda p: p[3] > 128 and p[4] > 0       # noqa: E731  both tiles of 128 rows, position tiles
one = lambda p: 0 < p[3] <= 128 and p[4] > 0  # noqa: E731  the first tile of 128 rows only
none = lambda p: p[3] > 0 and p[4] == 0       # noqa: E731  rows that see nothing


def blocks_with(sizes, heads, kvh, *kinds, whole=True, **kw):
    """How many blocks have parts of these kinds one after the other, whole row tiles all but the last."""
    n = 0
    for mine in parts(sizes, heads, kvh, SMS, **kw):
        for i in range(len(mine) - len(kinds) + 1):
            if all(k(p) and (p[5] or j + 1 == len(kinds) or not whole) for j, (k, p) in enumerate(zip(kinds, mine[i:]))):
                n += 1
                break
    return n


# ---- parts of 256, of at most 128, and of 256 rows ------------------------------------------------------------------------
HALVES = [(32, 200 - i % 20) if i % 2 == 0 else (9 + i % 8, 190) for i in range(500)]  # 8 heads over one: 256 rows, then 72 to 128
# ---- rows that see nothing among others --------------------------------------------------------------------------------------
EMPTY = [(64, 300 + i) if i % 2 == 0 else (64, 0) for i in range(120)]
EARLY = [(300, 20) if i % 2 == 0 else (64, 400) for i in range(60)]  # more tokens than positions: their first rows lie before position 0

TURNS = [(32, 100) if i % 2 == 0 else (32, 0) for i in range(500)]

# ---- single tokens and a prompt ----------------------------------------------------------------------------------------------
MIXED = [[(1, 1500)] * 7 + [(512, 2000)], [(1, 1500)] * 9 + [(256, 3000)]]


def ahead(sizes, heads, kvh):
    """Blocks in which a part of 256 rows follows a whole row tile of at most 128, four position tiles or more before it."""
    return sum(any(one(p) and p[5] and two(mine[i + 1]) and sum(x[4] for x in mine[:i + 1]) >= 4 for i, p in enumerate(mine[:-1]))
               for mine in parts(sizes, heads, kvh, SMS))


def test_the_batches_have_such_blocks():
    assert blocks_with(HALVES, 8, 1, two, one, two) == 102
    assert blocks_with(EMPTY, 8, 1, none, two) == 43
    assert blocks_with(EARLY, 8, 1, none, two) == 20
    assert blocks_with(TURNS, 8, 1, two, none, two) == 102
    for sizes in MIXED:
        assert ahead(sizes, 64, 8) > 0


KINDS16 = [("16", "fp16", 128), ("16", "bf16", 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,rows,hd", KINDS16)
def test_rows_taken_again_before_parts_of_one_and_two_tiles(backend, fmt, rows, hd):
    """An infinite value that only the last token of every fourth entry sees: its other 248 rows are taken again, 102 blocks having a part
    of at most 128 rows and one of 256 behind them."""
    c = Cache(fmt, rows, 1, hd, n_seqs=20, max_len=200, page=16, seed=hd)
    seqs = [i % 20 for i in range(len(HALVES))]
    entries, n = _entries(HALVES, seqs)
    q = queries(n, 8, hd, rows, 1)
    want, tol = oracle(c, q, entries, 8)
    odd = torch.zeros(n, dtype=torch.bool)
    spoiled = {}
    for s, r0, t, length in entries[::4]:
        spoiled.setdefault(s, set()).add(length - 1)
    for s, at in spoiled.items():
        for p in at:
            page, place = c.place(s, p)
            c.pool["v"][page, 0, place, 5] = math.inf
    for s, r0, t, length in entries:
        for i in range(t):
            odd[r0 + i] = any(p <= length - t + i for p in spoiled.get(s, ()))
    got = run_attention(backend, c, q, entries, 8)
    assert odd.any() and not odd.all()
    check(got, want, tol, ~odd)
    assert not torch.isfinite(got[odd][:, :, 5]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [EMPTY, EARLY, TURNS], ids=["empty", "early", "turns"])
@pytest.mark.parametrize("fmt,rows,hd", KINDS16)
def test_rows_that_see_nothing_among_others(backend, fmt, rows, hd, sizes):
    c = Cache(fmt, rows, 1, hd, n_seqs=20, max_len=430, page=32, seed=hd + 1)
    got, again = _both(backend, c, sizes, 8, seqs=[i % 20 for i in range(len(sizes))], seed=2)
    row = 0
    for n, length in sizes:
        assert (got[row:row + max(0, n - length)] == 0).all()
        row += n
    assert torch.equal(got, again())


CODED = [("int8", "fp16", 128), ("e4m3", "bf16", 128), ("int4", "bf16", 128), ("int8", "bf16", 64), ("int4", "fp16", 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", MIXED, ids=["seven", "nine"])
@pytest.mark.parametrize("fmt,rows,hd", CODED)
def test_single_tokens_and_a_prompt_over_codes(backend, fmt, rows, hd, sizes):
    """The values of neighbouring sequences differ 2^6-fold, so that another tile's exponent of the values would show."""
    c = Cache(fmt, rows, 8, hd, n_seqs=len(sizes), max_len=max(x for _, x in sizes), page=64, seed=hd + 2)
    for s in range(len(sizes)):
        c.scale["v"][c.table_cpu[s].long().cuda()] *= 2.0 ** (3 if s % 2 else -3)
    _both(backend, c, sizes, 64, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,rows,hd", CODED)
def test_turns_of_rows_over_codes(backend, fmt, rows, hd):
    """The batches above over codes."""
    for sizes in (HALVES, EMPTY, EARLY, TURNS):
        c = Cache(fmt, rows, 1, hd, n_seqs=20, max_len=430, page=32, seed=hd + 3)
        _both(backend, c, sizes, 8, seqs=[i % 20 for i in range(len(sizes))], seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,rows,hd", [("16", "bf16", 64), ("int8", "fp16", 64), ("16", "fp16", 128)])
def test_many_rows_of_a_long_sequence_taken_again(backend, fmt, rows, hd):
    """An infinite value early in a sequence of 60000 positions, seen by all of its rows or by some: its row tile is taken
    again position by position, which takes far longer than the other row tiles of its blocks, and they are right all the same."""
    sizes = [(32, 300)] * 40 + [(32, 60000)] + [(32, 300)] * 40
    seqs = [int(i != 40) for i in range(81)]
    assert blocks_with(sizes, 8, 1, lambda p: p[0] == 40, lambda p: p[0] == 41, whole=False) == 1
    c = Cache(fmt, rows, 1, hd, n_seqs=2, max_len=60000, page=64, seed=hd + 4)
    entries, n = _entries(sizes, seqs)
    q = queries(n, 8, hd, rows, 5)
    mine = slice(40 * 32, 41 * 32)
    near = [entries[i] for i in (0, 20, 38, 39, 41, 42, 43, 60, 80)]
    others = [r0 + i for _, r0, t, _ in near for i in range(t)]
    want, tol = oracle(c, q, near, 8)
    page, at = c.place(0, 1000)
    if fmt == "16":
        c.pool["v"][page, 0, at, 7] = math.inf
    else:
        c.scale["v"][page, 0, at] = math.inf
    got = run_attention(backend, c, q, entries, 8)
    check(got, want, tol, others)
    assert not torch.isfinite(got[mine].float()).all(-1).any()
    window = 58980  # the last 20 tokens do not see position 1000
    want, tol = oracle(c, q, near, 8, window=window)
    got = run_attention(backend, c, q, entries, 8, window=window)
    check(got, want, tol, others)
    if fmt == "16":
        c.pool["v"][page, 0, at, 7] = 0.0
    else:
        c.scale["v"][page, 0, at] = 0.0
    want, tol = oracle(c, q, [entries[40]], 8, window=window)
    late = [40 * 32 + i for i in range(32) if 59968 + i - window >= 1000]
    assert 0 < len(late) < 32
    check(got, want, tol, late)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("fmt,rows,hd", CODED)
def test_ragged_drafts_over_codes(backend, fmt, rows, hd, seed):
    """Drafts of 2 to 63 tokens behind 200 to 3000 committed ones, and single tokens, neighbouring sequences' values 2^6-fold apart."""
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    sizes = [(1 if r(0, 2) else r(2, 63), 0) for _ in range(9)] + [(63, 0)]
    sizes = [(n, n + r(200, 3000)) for n, _ in sizes]
    c = Cache(fmt, rows, 8, hd, n_seqs=10, max_len=3100, page=64, seed=hd + 5)
    for s in range(10):
        c.scale["v"][c.table_cpu[s].long().cuda()] *= 2.0 ** (3 if s % 2 else -3)
    masks = [1 << j | (1 << max(0, j - 3)) | 1 for n, _ in sizes for j in range(n)]
    _both(backend, c, sizes, 64, seed=seed, masks=masks)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,rows,hd", KINDS16 + CODED[:3])
def test_rows_apart_and_padding_between_entries(backend, fmt, rows, hd):
    """Queries and results with gaps between rows, entries of a negative sequence and without rows among the others: what belongs to no
    entry stays as it was."""
    sizes = [(40 - i, 400 + 9 * i) if i % 7 else (0, 50) for i in range(30)]
    c = Cache(fmt, rows, 2, hd, n_seqs=6, max_len=700, page=64, seed=hd + 6)
    entries, n = _entries(sizes, [i % 6 for i in range(30)])
    q = queries(n + 5, 16, hd, rows, 7)
    padding = [i % 5 == 3 for i in range(30)]
    want, tol = oracle(c, q, [e for e, p in zip(entries, padding) if not p], 16, window=200, sinks=7)
    wide = torch.full((n + 5, 3, 16, hd), 7.0, dtype=q.dtype, device="cuda")
    wide[:, 1] = q.cuda()
    a = [i32([-1 if p else e[0] for e, p in zip(entries, padding)]), i32([e[1] for e in entries] + [n]), i32([e[3] for e in entries])]
    torch.cuda.synchronize()
    step, row = 3 * 16 * hd, 16 * hd * 2
    backend.cache_attention_dev(c.view(), wide.data_ptr() + row, wide.data_ptr() + 2 * row, n_rows=n + 5, n_entries=30, seq=a[0].data_ptr(),
                                q_start=a[1].data_ptr(), length=a[2].data_ptr(), max_tokens=40, max_length=700, num_heads=16, window=200, sinks=7,
                                q_stride=step, out_stride=step)
    backend.synchronize()
    theirs = torch.zeros(n + 5, dtype=torch.bool)
    for (_, r0, t, _), p in zip(entries, padding):
        theirs[r0:r0 + t] = not p
    got = wide.cpu()
    check(got[:, 2], want, tol, theirs)
    assert (got[~theirs][:, 2] == 7).all() and (got[:, 0] == 7).all() and torch.equal(got[:, 1], q)
