"""Tables whose pages are not all there: pages that no row sees are not asked for, and positions of bad pages take no part, whatever
the kernel.  Bound per output as in
test_gpu_cache_many_rows."""
import pytest
import torch

from cache_util import Cache, check, queries, run_attention
from test_gpu_cache_many_rows import _entries, oracle

pytestmark = pytest.mark.gpu

FORMATS = [("16", "fp16"), ("16", "bf16"), ("int8", "fp16"), ("e4m3", "bf16"), ("int4", "bf16")]


def _seen(entries, n_seqs, most, window, sinks, q_pos=None):
    """[sequence, position]: whether some row sees it (drafted positions: all)."""
    see = torch.zeros(n_seqs, most, dtype=torch.bool)
    for s, r0, n, length in entries:
        for i in range(n):
            p = q_pos[r0 + i] if q_pos else length - n + i
            c = torch.arange(most)
            see[s] |= (c < length - n if q_pos else c <= p) & ((c > p - window) | (c < sinks))
        if q_pos:
            see[s, length - n:length] = True
    return see


def _give_back(c, see):
    """Table entries of pages with nothing to see are no pages."""
    gone = ~see.view(c.n_seqs, -1, c.page).any(-1)
    assert gone.any() and not gone.all()
    odd = torch.tensor([-1, c.pages, 1 << 30], dtype=torch.int32)
    c.table.copy_(torch.where(gone, odd[torch.arange(gone.numel()) % 3].view_as(gone), c.table_cpu).cuda())


@pytest.mark.parametrize("window,sinks", [(1, 0), (37, 5), (100, 16), (300, 70)])
@pytest.mark.parametrize("page", [16, 32, 128, 256])
@pytest.mark.parametrize("fmt,rows", FORMATS)
def test_pages_behind_the_window_given_back(backend, fmt, rows, page, window, sinks):
    """Single tokens, small portions and large ones; tokens and drafts."""
    for hd, heads, kvh, sizes in ((64, 6, 2, [(1, 500), (1, 511), (2, 512), (1, 3)]), (256, 4, 1, [(3, 700)]), (32, 4, 1, [(5, 333), (1, 1024)]),
                                  (128, 8, 1, [(40, 600 + 13 * i) for i in range(24)]), (64, 16, 1, [(17 + i, 900 - 31 * i) for i in range(20)]),
                                  (128, 16, 1, [(70, 1000)])):
        most = -(-1024 // page) * page
        c = Cache(fmt, rows, kvh, hd, n_seqs=len(sizes), max_len=most, page=page, seed=hd)
        entries, n = _entries(sizes, list(range(len(sizes))))
        q = queries(n, heads, hd, rows, 1)
        _give_back(c, _seen(entries, len(sizes), most, window, sinks))
        want, tol = oracle(c, q, entries, heads, window=window, sinks=sinks)
        check(run_attention(backend, c, q, entries, heads, window=window, sinks=sinks), want, tol)
        pos = [length - t + i % 3 for t, length in sizes for i in range(t)]
        masks = [(1 << i % 64) | 1 for t, _ in sizes for i in range(t)]
        _give_back(c, _seen(entries, len(sizes), most, window, sinks, pos))
        want, tol = oracle(c, q, entries, heads, window=window, sinks=sinks, masks=masks, q_pos=pos)
        check(run_attention(backend, c, q, entries, heads, window=window, sinks=sinks, masks=masks, q_pos=pos), want, tol)


@pytest.mark.parametrize("number", [-1, 1 << 30])
@pytest.mark.parametrize("fmt,rows", FORMATS)
def test_positions_of_bad_pages_are_skipped_and_reported(backend, fmt, rows, number):
    """Pages that rows see and that are none of the pool's: as if the sequence did not hold their positions."""
    import copy

    from prism_engine_b200 import PrismCudaError

    for hd, heads, kvh, page, sizes in ((64, 6, 2, 16, [(1, 500), (1, 40), (2, 300), (1, 17)]), (256, 2, 1, 32, [(3, 700)]), (32, 4, 1, 16, [(1, 1024), (2, 90)]),
                                        (128, 8, 1, 16, [(9, 300 + 13 * i) for i in range(40)]), (64, 8, 2, 64, [(40, 900 - 31 * i) for i in range(20)]),
                                        (128, 16, 1, 256, [(40, 900)] * 6), (64, 16, 1, 32, [(70, 1000)])):
        c = Cache(fmt, rows, kvh, hd, n_seqs=len(sizes), max_len=1024, page=page, seed=hd + 1)
        entries, n = _entries(sizes, list(range(len(sizes))))
        q = queries(n, heads, hd, rows, 3)
        short = copy.copy(c)
        short.table_cpu = c.table_cpu.clone()
        left = []
        for s, r0, t, length in entries:
            bad = (length - t) // page // (2 if s % 2 else 3) if length - t >= page else None
            if bad is not None and s % 5 != 4:
                c.table[s, bad] = number
                short.table_cpu[s] = torch.cat([c.table_cpu[s, :bad], c.table_cpu[s, bad + 1:], c.table_cpu[s, :1]])
                left.append((s, r0, t, length - page))
            else:
                left.append((s, r0, t, length))
        for masks in (None, [(1 << i % 64) | 1 for t, _ in sizes for i in range(t)]):
            want, tol = oracle(short, q, left, heads, masks=masks)
            out = torch.full((n, heads, hd), 7.0, dtype=q.dtype, device="cuda")
            with pytest.raises(PrismCudaError) as e:
                run_attention(backend, c, q, entries, heads, masks=masks, out=out)
            assert e.value.code == -2
            check(out.cpu(), want, tol)
        c.table[:] = number  # none is left
        with pytest.raises(PrismCudaError):
            run_attention(backend, c, q, entries, heads, out=out)
        assert (out == 0).all()
