"""Scales and values that are not finite in the many-row attention, over codes and 16 bits, where some rows look and others do not;
reading a place outside the pool.  Bound per output as in test_gpu_cache_many_rows."""
import math

import pytest
import torch

from cache_util import DT, Cache, check, i32, queries, run_attention
from test_gpu_cache_many_rows import _entries, oracle

pytestmark = pytest.mark.gpu

FORMATS = [("16", "fp16", 64), ("16", "bf16", 128), ("int8", "fp16", 128), ("int8", "bf16", 64), ("e4m3", "bf16", 64), ("e4m3", "fp16", 128),
           ("int4", "bf16", 128), ("int4", "fp16", 64)]


def _spoil(c, s, p, value, names=("k", "v")):
    page, at = c.place(s, p)
    for n in names:
        if c.fmt == "16":
            c.pool[n][page, :, at, 3] = value
        else:
            c.scale[n][page, :, at] = value
            if c.fmt == "e4m3" and math.isnan(value):
                c.pool[n][page, :, at, 5] = 0x7F  # a code that is NaN by itself


@pytest.mark.parametrize("names", [("k", "v"), ("k",), ("v",)], ids=["both", "keys", "values"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("fmt,rows,hd", FORMATS)
def test_many_rows(backend, fmt, rows, hd, value, names):
    """Behind the last position, outside the window, at a later token and at another branch of the drafts: rows that do not see them are
    as without them, those that do are not finite."""
    c = Cache(fmt, rows, 2, hd, n_seqs=40, max_len=256, page=32, seed=2)
    sizes = [(20, 150 + i % 5) for i in range(40)]
    entries, n = _entries(sizes, list(range(40)))
    q = queries(n, 8, hd, rows, 3)
    token = torch.arange(n) % 20
    masks = [((1 << 20) - 1) ^ (1 << 15) if i % 20 != 3 else 1 << 15 for i in range(n)]
    pos = [e[3] - 10 for e in entries for _ in range(20)]
    plain = oracle(c, q, entries, 8, window=40, sinks=5)
    drafts = oracle(c, q, entries, 8, masks=masks, q_pos=pos, window=40, sinks=5)
    for s, (_, length) in enumerate(sizes):
        for p in [10, 60, length - 5] + list(range(length, 256, 3)):
            _spoil(c, s, p, value, names)
    got = run_attention(backend, c, q, entries, 8, window=40, sinks=5)
    check(got, *plain, token < 15)
    assert not torch.isfinite(got[token >= 15].float()).all(-1).any() or names == ("k",)
    got = run_attention(backend, c, q, entries, 8, masks=masks, q_pos=pos, window=40, sinks=5)
    check(got, *drafts, token != 3)
    assert not torch.isfinite(got[token == 3].float()).all(-1).any() or names == ("k",)
    if names == ("k",) and math.isnan(value):
        assert got[token == 3].isnan().all()


@pytest.mark.parametrize("fmt,rows", [("16", "bf16"), ("int8", "fp16"), ("e4m3", "bf16"), ("int4", "fp16")])
def test_rows_read_from_outside_stay(backend, fmt, rows):
    """A page that is none of the pool's, a sequence and a position outside the cache: their rows stay as they were, the others are read."""
    from prism_engine_b200 import PrismCudaError

    c = Cache(fmt, rows, 2, 64, n_seqs=3, max_len=64, page=16, seed=4)
    for number in (-5, -1, c.pages, 1 << 30):
        c.table.copy_(c.table_cpu)
        c.table[0, 1] = number
        seq, pos = i32([0, 0, 3, 1, 2, 1]), i32([16, 31, 0, 64, 63, 5])
        out = [torch.full((6, 2, 64), 7.0, dtype=DT[rows], device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        backend.cache_read_dev(c.view(), out[0].data_ptr(), out[1].data_ptr(), 6, seq.data_ptr(), pos.data_ptr())
        with pytest.raises(PrismCudaError) as e:
            backend.synchronize()
        assert e.value.code == -2
        for name, got in zip("kv", out):
            assert (got[:4] == 7).all()
            for r, (s, p) in ((4, (2, 63)), (5, (1, 5))):
                a, z, want = (x[p] for x in c.parts(name, s, p + 1))
                # one rounding of the result, one of the product and one of the sum in 32 bits
                bound = torch.finfo(DT[rows]).eps / 2 * want.abs() + 2.0 ** -23 * (a.abs() + z.abs()) + 2.0 ** -25
                assert ((got[r].cpu().double() - want).abs() <= bound).all()
