"""Many rows over codes whose values differ by powers of two from position to position, near enough for products in fp16 or not,
and large where no row looks.  Bound per output as in test_gpu_cache_many_rows: relative to the values that a row sees."""
import pytest
import torch

from cache_util import Cache, check, queries, run_attention
from test_gpu_cache_many_rows import _both, _entries, oracle

pytestmark = pytest.mark.gpu

CODED = [("int8", "bf16", 128), ("int8", "bf16", 64), ("e4m3", "bf16", 128), ("int4", "bf16", 128), ("int4", "bf16", 64)]


def _spread(c, lo, hi, seed, more=1.0):
    by = torch.exp2(torch.randint(lo, hi + 1, c.scale["v"].shape[:3], generator=torch.Generator().manual_seed(seed)).float()).cuda() * more
    c.scale["v"] *= by if c.fmt != "int4" else by[..., None]


@pytest.mark.parametrize("more", [2.0 ** -90, 2.0 ** -20, 1.0, 2.0 ** 60])
@pytest.mark.parametrize("lo,hi", [(0, 5), (-6, 6), (-12, 13)])
@pytest.mark.parametrize("fmt,rows,hd", CODED)
def test_values_of_any_size(backend, fmt, rows, hd, lo, hi, more):
    c = Cache(fmt, rows, 1, hd, n_seqs=40, max_len=320, page=64, seed=hd)
    _spread(c, lo, hi, hd, more)
    got, again = _both(backend, c, [(20 + i % 7, 20 + i * 7) for i in range(40)], 8, seed=1)
    assert torch.equal(got, again())


@pytest.mark.parametrize("up", [2.0 ** 15, 2.0 ** 22, 2.0 ** 30, 2.0 ** 50])
@pytest.mark.parametrize("fmt,rows,hd", CODED)
def test_large_values_that_no_row_sees(backend, fmt, rows, hd, up):
    """Before the window, and at tokens and drafts that are not in a row's sight."""
    c = Cache(fmt, rows, 1, hd, n_seqs=40, max_len=320, page=64, seed=hd)
    sizes = [(20, 150 + i) for i in range(40)]
    for s, (n, length) in enumerate(sizes):
        for p in (length - n - 70, length - 1, length - 8):
            page, at = c.place(s, p)
            c.scale["v"][page, 0, at] *= up
    entries, rows_n = _entries(sizes, list(range(40)))
    q = queries(rows_n, 8, hd, rows, 2)
    token = torch.arange(rows_n) % 20
    want, tol = oracle(c, q, entries, 8, window=60, sinks=3)
    check(run_attention(backend, c, q, entries, 8, window=60, sinks=3), want, tol)
    assert float(want[token < 12].abs().max()) < 100 < float(want[token == 19].abs().max())
    masks = [((1 << 20) - 1) ^ (1 << 19) ^ (1 << 12) if i % 20 not in (12, 19) else 1 << 12 for i in range(rows_n)]
    pos = [e[3] - 20 + i % 4 for e in entries for i in range(20)]
    want, tol = oracle(c, q, entries, 8, masks=masks, q_pos=pos, window=60, sinks=3)
    check(run_attention(backend, c, q, entries, 8, masks=masks, q_pos=pos, window=60, sinks=3), want, tol)


@pytest.mark.parametrize("first", [0, 8, 15, 24, 40])
@pytest.mark.parametrize("fmt,rows,hd", CODED)
def test_parts_whose_values_lie_apart(backend, fmt, rows, hd, first):
    """The first 500 positions 2^first above the others; cut into parts that are joined, and shared by the blocks."""
    c = Cache(fmt, rows, 1, hd, n_seqs=40, max_len=2000, page=64, seed=hd + 1)
    for s in range(40):
        c.scale["v"][c.table_cpu[s, :500 // 64].long().cuda()] *= 2.0 ** first
    _both(backend, c, [(64, 2000)], 8, seed=3)
    _both(backend, c, [(24, 1000)] * 40, 8, seed=4, window=300)
