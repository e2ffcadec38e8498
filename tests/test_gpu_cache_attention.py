"""Attention over a cache of several sequences: windows with first tokens that stay visible, drafted trees, every format and head
layout, against the definition in 64 bits.

Bound per output (cache_util.attention): the result is rounded once; a weight is rounded to 16 bits (those of the row's type for a
16-bit cache, fp16 for codes), which counts twice, in the sum of products and in the sum it is divided by; a score is off by the
rounding of head_dim additions, and of a query's elements that are 2^-14 of its largest or less."""
import pytest
import torch

from cache_util import DT, KINDS, Cache, attention, check, i32, queries, run_attention

pytestmark = pytest.mark.gpu


def _entries(sizes, seqs=None):
    """(sequence, first row, rows, length) of entries of (rows, length)."""
    out, row = [], 0
    for i, (n, length) in enumerate(sizes):
        out.append((seqs[i] if seqs else i, row, n, length))
        row += n
    return out, row


def _both(backend, c, sizes, heads, seqs=None, seed=0, **kw):
    entries, rows = _entries(sizes, seqs)
    q = queries(rows, heads, c.hd, c.rows, seed)
    want, tol = attention(c, q, entries, heads, **kw)
    check(run_attention(backend, c, q, entries, heads, **kw), want, tol)


LAYOUTS = [(32, 5, 1), (32, 8, 8), (64, 14, 2), (128, 28, 4), (128, 24, 2), (256, 4, 2)]


@pytest.mark.parametrize("hd,heads,kvh", LAYOUTS)
@pytest.mark.parametrize("fmt,rows", KINDS)
def test_single_tokens(backend, fmt, rows, hd, heads, kvh):
    """One token of each sequence, lengths about a tile's and a page's ends."""
    c = Cache(fmt, rows, kvh, hd, n_seqs=9, max_len=300, page=16, seed=hd)
    _both(backend, c, [(1, n) for n in (1, 2, 15, 16, 17, 33, 64, 129, 300)], heads)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (16, 16), (33, 4), (100, 70), (500, 4), (64, 0)])
@pytest.mark.parametrize("fmt,rows,hd,heads,kvh,page", [("16", "fp16", 64, 6, 2, 16), ("int8", "bf16", 128, 8, 1, 64), ("int4", "fp16", 32, 3, 3, 0),
                                                       ("16", "bf16", 256, 2, 1, 32), ("e4m3", "fp16", 128, 12, 1, 128)])
def test_windows_with_first_tokens(backend, fmt, rows, hd, heads, kvh, page, window, sinks):
    """Single tokens and portions; the window's end inside a tile, the first tokens in, next to and apart from the window."""
    c = Cache(fmt, rows, kvh, hd, n_seqs=5, max_len=260, page=page, seed=window)
    _both(backend, c, [(1, 1), (1, 260), (40, 40), (21, 200), (3, 90)], heads, window=window, sinks=sinks, seed=window)


@pytest.mark.parametrize("fmt,rows,hd,heads,kvh", [("16", "bf16", 128, 7, 1), ("16", "fp16", 64, 4, 4), ("int8", "fp16", 64, 14, 2), ("int4", "bf16", 128, 16, 2),
                                                   ("e4m3", "bf16", 256, 3, 1), ("16", "fp16", 32, 4, 1)])
def test_portions(backend, fmt, rows, hd, heads, kvh):
    """Prompt portions of any length, one of them the whole sequence, entries in another order than the sequences."""
    c = Cache(fmt, rows, kvh, hd, n_seqs=4, max_len=400, page=32, seed=5)
    _both(backend, c, [(130, 400), (1, 7), (77, 77), (19, 150)], heads, seqs=[2, 0, 3, 1])


def _random_tree(n, g, wide):
    masks, depth = [], []
    for j in range(n):
        p = -1 if j < wide else int(torch.randint(0, j, (1,), generator=g))
        masks.append((masks[p] if p >= 0 else 0) | 1 << j)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return masks, depth


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("fmt,rows,hd,heads,kvh", [("16", "fp16", 64, 14, 2), ("int8", "bf16", 128, 8, 1), ("int4", "fp16", 128, 4, 4), ("e4m3", "fp16", 32, 6, 3),
                                                   ("16", "bf16", 256, 2, 2), ("int8", "fp16", 64, 16, 1)])
def test_trees(backend, fmt, rows, hd, heads, kvh, window, sinks):
    """Drafts of 1 to 100 tokens behind 0 to 200 committed ones."""
    sizes = [(1, 50), (12, 12), (33, 140), (64, 264), (100, 171), (2, 3)]
    c = Cache(fmt, rows, kvh, hd, n_seqs=6, max_len=300, page=16, seed=9)
    g = torch.Generator().manual_seed(1)
    masks, pos = [], []
    for n, length in sizes:
        m, d = _random_tree(n, g, 1 + n // 8)
        masks += m
        pos += [length - n + x for x in d]
    _both(backend, c, sizes, heads, masks=masks, q_pos=pos, window=window, sinks=sinks)


def test_masks_of_any_shape(backend):
    """Rows that see nothing (no committed token, an empty mask), not themselves, or tokens behind them; bits past the draft are ignored."""
    c = Cache("int8", "fp16", 2, 64, n_seqs=3, max_len=64, page=16)
    masks = [0, 1 << 2, 1 << 63 | 7, 0b1010, 0, 2, 1]
    entries, rows = _entries([(3, 3), (2, 20), (2, 40)])
    q = queries(rows, 4, 64, "fp16")
    want, tol = attention(c, q, entries, 4, masks=masks)
    got = run_attention(backend, c, q, entries, 4, masks=masks)
    check(got, want, tol)
    assert (got[0] == 0).all() and (got[1] != 0).any()
    # under a window that leaves nothing of the committed ones either
    masks = [0, 0, 0, 0, 0, 0, 0]
    got = run_attention(backend, c, q, entries, 4, masks=masks, q_pos=[0, 0, 0, 90, 18, 100, 38], window=3)
    want, tol = attention(c, q, entries, 4, masks=masks, q_pos=[0, 0, 0, 90, 18, 100, 38], window=3)
    check(got, want, tol)
    assert (got[3] == 0).all() and (got[4] != 0).any() and (got[5] == 0).all()


def test_rows_of_no_entry_stay(backend):
    """Padding: entries with a negative sequence or no rows, rows behind the last entry; an empty sequence gives zeros."""
    c = Cache("16", "fp16", 1, 64, n_seqs=4, max_len=64, page=16)
    entries, _ = _entries([(2, 9), (3, 30), (0, 5), (1, 0), (2, 1)])
    q = queries(12, 2, 64, "fp16")
    got = run_attention(backend, c, q, entries, 2, seqs=[1, -1, 2, 3, 0])
    want, tol = attention(c, q, [(1, 0, 2, 9)], 2)
    check(got, want, tol, slice(0, 2))
    assert (got[2:5] == 7).all() and (got[8:] == 7).all()
    assert (got[5] == 0).all()          # a token of a sequence that holds nothing
    assert (got[6] == 0).all()          # two tokens, one position: the first lies before it
    want, tol = attention(c, q, [(0, 7, 1, 1)], 2)
    check(got, want, tol, slice(7, 8))


def test_rows_apart_and_scale(backend):
    c = Cache("int4", "bf16", 2, 128, n_seqs=2, max_len=90, page=16)
    wide = queries(5, 3 * 4, 128, "bf16").view(5, 3, 4, 128).cuda()
    q, out = wide[:, 1], torch.zeros(5, 6, 128, dtype=torch.bfloat16, device="cuda")
    entries, _ = _entries([(4, 50), (1, 90)])
    want, tol = attention(c, q.cpu(), entries, 4, scale=0.3)
    qd = wide
    seq, st, ln = i32([0, 1]), i32([0, 4, 5]), i32([50, 90])
    torch.cuda.synchronize()
    backend.cache_attention_dev(c.view(), qd.data_ptr() + 4 * 128 * 2, out.data_ptr(), n_rows=5, n_entries=2, seq=seq.data_ptr(), q_start=st.data_ptr(),
                                length=ln.data_ptr(), max_tokens=4, max_length=90, num_heads=4, scale=0.3, q_stride=12 * 128, out_stride=6 * 128)
    backend.synchronize()
    check(out[:, :4].cpu(), want, tol)
    assert (out[:, 4:] == 0).all()


@pytest.mark.parametrize("fmt,rows,hd", [("16", "fp16", 64), ("16", "bf16", 128), ("int8", "fp16", 128), ("e4m3", "bf16", 64), ("int4", "bf16", 256)])
def test_not_finite_where_nothing_looks(backend, fmt, rows, hd):
    """NaN and infinities behind the last position, outside the window, at a later token of the portion and at a draft's other
    branch stay out of the rows that do not see them, and reach those that do."""
    c = Cache(fmt, rows, 1, hd, n_seqs=1, max_len=256, page=32, seed=2)

    def spoil(p, value):
        page, at = c.place(0, p)
        for n in ("k", "v"):
            if fmt == "16":
                c.pool[n][page, :, at, 3] = value
            else:
                c.scale[n][page, :, at] = value

    for value in (float("nan"), float("inf")):
        fresh = Cache(fmt, rows, 1, hd, n_seqs=1, max_len=256, page=32, seed=2)
        c.pool, c.scale = fresh.pool, fresh.scale
        for p in list(range(150, 256)) + [10, 60, 145]:
            spoil(p, value)
        entries, n = [(0, 0, 20, 150)], 20
        q = queries(n, 4, hd, rows)
        got = run_attention(backend, c, q, entries, 4, window=40, sinks=5)  # rows at 130 .. 149
        want, tol = attention(c, q, entries, 4, window=40, sinks=5)
        check(got, want, tol, slice(0, 15))
        assert torch.isfinite(got[:15].float()).all() and not torch.isfinite(got[15:].float()).all(-1).any()
        assert torch.equal(torch.isnan(got[15:]), torch.isnan(want[15:]))
        # drafted: token 15 of 20 lies at 145
        masks = [((1 << 20) - 1) ^ (1 << 15) if i != 3 else 1 << 15 for i in range(20)]
        got = run_attention(backend, c, q, entries, 4, masks=masks, q_pos=[140] * 20, window=40, sinks=5)
        want, tol = attention(c, q, entries, 4, masks=masks, q_pos=[140] * 20, window=40, sinks=5)
        keep = [i for i in range(20) if i != 3]
        check(got, want, tol, keep)
        assert torch.equal(torch.isnan(got[3]), torch.isnan(want[3].to(DT[rows])))


@pytest.mark.parametrize("fmt,rows", [("16", "fp16"), ("16", "bf16"), ("int8", "bf16"), ("int4", "fp16")])
def test_sharp_and_flat_scores(backend, fmt, rows):
    """Scores hundreds apart, rising along the sequence and falling; all equal; one key that takes everything."""
    c = Cache(fmt, rows, 1, 64, n_seqs=3, max_len=200, page=16, seed=4)
    entries, n = _entries([(2, 200), (2, 131), (1, 64)])
    for mul in (0.0, 30.0, 1000.0):
        q = (queries(n, 2, 64, rows).float() * mul).to(DT[rows])
        want, tol = attention(c, q, entries, 2)
        check(run_attention(backend, c, q, entries, 2), want, tol)


@pytest.mark.parametrize("scale_by", [2.0 ** -90, 2.0 ** -20, 2.0 ** 14, 2.0 ** 60])
@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_scales_of_any_size(backend, fmt, scale_by):
    """Values of codes far from 1, and very different from position to position: no 16-bit number on the way over- or underflows."""
    c = Cache(fmt, "bf16", 1, 128, n_seqs=1, max_len=300, page=64, seed=6)
    g = torch.Generator().manual_seed(7)
    by = torch.exp2(torch.randint(-12, 13, c.scale["v"].shape[:3], generator=g).float()).cuda() * scale_by
    c.scale["v"] *= by if fmt == "int8" else by[..., None]
    entries = [(0, 0, 1, 300), (0, 1, 1, 17)]
    q = queries(2, 8, 128, "bf16")
    want, tol = attention(c, q, entries, 8)
    got = run_attention(backend, c, q, entries, 8)
    check(got, want, tol)


@pytest.mark.parametrize("fmt,rows,hd,heads,kvh,length", [("int4", "bf16", 128, 8, 1, 20011), ("16", "fp16", 64, 7, 1, 9000), ("int8", "fp16", 128, 16, 2, 40000)])
def test_long_sequences(backend, fmt, rows, hd, heads, kvh, length):
    """The work of one token cut over many blocks and joined, the same bits every time; the expected length only says how it is cut."""
    c = Cache(fmt, rows, kvh, hd, n_seqs=1, max_len=length, page=64, seed=8)
    entries = [(0, 0, 1, length)]
    q = queries(1, heads, hd, rows)
    want, tol = attention(c, q, entries, heads)
    a = run_attention(backend, c, q, entries, heads)
    check(a, want, tol)
    assert all(torch.equal(a, run_attention(backend, c, q, entries, heads)) for _ in range(3))
    for most in (0, 100, 1 << 30):
        check(run_attention(backend, c, q, entries, heads, max_length=most), want, tol)


def test_bad_pages_and_entries_are_skipped_and_reported(backend):
    from prism_engine_b200 import PrismCudaError

    c = Cache("int8", "fp16", 1, 64, n_seqs=2, max_len=128, page=16)
    q = queries(4, 2, 64, "fp16")
    for sizes, seqs in (([(2, 129), (2, 60)], [0, 1]), ([(2, 50), (2, 60)], [2, 1]), ([(2, -3), (2, 60)], [0, 1])):
        entries, _ = _entries(sizes)
        out = torch.full((4, 2, 64), 7.0, dtype=torch.float16, device="cuda")
        with pytest.raises(PrismCudaError) as e:
            run_attention(backend, c, q, entries, 2, seqs=seqs, out=out)
        assert e.value.code == -2
        want, tol = attention(c, q, [(1, 2, 2, 60)], 2)
        check(out.cpu(), want, tol, slice(2, 4))
        assert (out[:2] == 7).all()
    c.table[1, 2] = 1 << 20
    entries, _ = _entries([(2, 30), (2, 60)])
    out = torch.full((4, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    with pytest.raises(PrismCudaError):
        run_attention(backend, c, q, entries, 2, out=out)
    want, tol = attention(c, q, [(0, 0, 2, 30)], 2)
    check(out.cpu(), want, tol, slice(0, 2))
    assert torch.isfinite(out.float()).all()
    c.table[1, 2] = c.table_cpu[1, 2]
    want, tol = attention(c, q, entries, 2)
    check(run_attention(backend, c, q, entries, 2), want, tol)


def test_refusals(backend):
    from prism_engine_b200 import PrismCudaError

    c = Cache("int8", "fp16", 2, 64, n_seqs=1, max_len=32, page=16)
    x = torch.zeros(4, 4, 64, dtype=torch.float16, device="cuda")
    s = i32([0, 4, 4])
    p, i = x.data_ptr(), s.data_ptr()
    torch.cuda.synchronize()
    good = dict(q=p, out=p, n_rows=4, n_entries=1, seq=i, q_start=i, length=i + 4, max_tokens=4, max_length=4, num_heads=4)
    for code, over in [(-2, dict(num_heads=3)), (-2, dict(num_heads=0)), (-2, dict(num_heads=1 << 20)), (-2, dict(n_entries=70000)),
                       (-2, dict(q=p + 2)), (-2, dict(out=p + 8)), (-2, dict(q_stride=128)), (-2, dict(out_stride=260)), (-2, dict(scale=float("nan"))),
                       (-2, dict(scale=float("inf"))), (-2, dict(tree=p, tree_words=0)), (-2, dict(tree=p, tree_words=1, max_tokens=65)),
                       (-2, dict(tree=p + 4, tree_words=1)), (-1, dict(tree=p, tree_words=1, window=4)), (-2, dict(max_tokens=1 << 25)),
                       (-1, dict(q=0)), (-1, dict(out=0)), (-1, dict(seq=0)), (-1, dict(q_start=0)), (-1, dict(length=0))]:
        with pytest.raises(PrismCudaError) as e:
            backend.cache_attention_dev(c.view(), **{**good, **over})
        assert e.value.code == code, over
    with pytest.raises(PrismCudaError):
        backend.cache_attention_dev(c.view(head_dim=96), **good)
    for none in (dict(n_entries=0), dict(n_rows=0), dict(max_tokens=0)):
        backend.cache_attention_dev(c.view(), **{**good, **none})
    backend.synchronize()
