"""Attention over a cache where the work is cut up: blocks that share the position tiles of many row tiles, row tiles of a block each,
positions in parts that a second kernel joins, parts of few rows in clusters; against the definition in 64 bits.

Bound per output as in cache_util.attention, with 2^-18 more for a weight's power of two."""
import math

import pytest
import torch

from cache_util import DT, U, Cache, check, i32, queries, run_attention

pytestmark = pytest.mark.gpu


def oracle(cache, q, entries, heads, window=0, sinks=0, scale=None, masks=None, q_pos=None):
    """cache_util.attention, an entry's rows at once, on the GPU."""
    hd, kvh, group = cache.hd, cache.kvh, heads // cache.kvh
    scale = scale or 1 / math.sqrt(hd)
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64)
    tol = torch.zeros_like(out)
    u_p = U[cache.rows] if cache.fmt == "16" else U["fp16"]
    for s, r0, n, length in entries:
        if n == 0 or length == 0:
            continue
        ka, kz, k = [x.cuda() for x in cache.parts("k", s, length)]
        va, vz, v = [x.cuda() for x in cache.parts("v", s, length)]
        c, first = torch.arange(length, device="cuda")[None], length - n
        if masks is None:
            p = first + torch.arange(n, device="cuda")[:, None]
            see = c <= p
        else:
            p = torch.tensor(q_pos[r0:r0 + n] if q_pos is not None else [first] * n, device="cuda")[:, None]
            see = (c < first).expand(n, length)
        if window:
            see = see & ((c > p - window) | (c < sinks))
        if masks is not None:
            see = see.clone()
            bits = torch.tensor([[bool(masks[r0 + i] >> j & 1) for j in range(n)] for i in range(n)], device="cuda")
            lo = max(0, -first)
            see[:, first + lo:] = bits[:, lo:]
        any_, count = see.any(1), see.sum(1)
        rows = see.repeat_interleave(group, 0)
        seen = lambda x: torch.where(rows, x, 0.0).amax(1)  # noqa: E731
        for m in range(kvh):
            x = q[r0:r0 + n, m * group:(m + 1) * group].cuda().double().reshape(n * group, hd)
            sc = torch.where(rows, x @ k[:, m].T * scale, -math.inf)
            w = torch.nan_to_num(torch.softmax(sc, 1)) if not any_.all() else torch.softmax(sc, 1)
            kk, vv = ka[:, m].abs() + kz[:, m].abs(), va[:, m].abs() + vz[:, m].abs()
            off = abs(scale) * (hd * 2.0 ** -24 * seen(x.abs() @ kk.T) + 2.0 ** -24 * x.abs().amax(1) * seen(kk.sum(-1)[None])) + 2.0 ** -20 + 2.0 ** -18
            o = w @ v[:, m]
            least = 2.0 ** -37 * w.amax(1) * count.repeat_interleave(group) * seen(vv.amax(-1)[None])
            t = ((2 * u_p + 2 * off)[:, None] * (w @ vv) + U[cache.rows] * o.abs() + least[:, None] +
                 (2.0 ** -25 if cache.rows == "fp16" else 2.0 ** -134)) * any_.repeat_interleave(group)[:, None]
            out[r0:r0 + n, m * group:(m + 1) * group] = o.view(n, group, hd).cpu()
            tol[r0:r0 + n, m * group:(m + 1) * group] = t.view(n, group, hd).cpu()
    return out, tol


def _entries(sizes, seqs):
    out, row = [], 0
    for i, (n, length) in enumerate(sizes):
        out.append((seqs[i], row, n, length))
        row += n
    return out, row


def _both(backend, c, sizes, heads, seqs=None, seed=0, max_length=None, **kw):
    entries, rows = _entries(sizes, seqs or list(range(len(sizes))))
    q = queries(rows, heads, c.hd, c.rows, seed)
    want, tol = oracle(c, q, entries, heads, **kw)
    got = run_attention(backend, c, q, entries, heads, max_length=max_length, **kw)
    check(got, want, tol)
    return got, lambda: run_attention(backend, c, q, entries, heads, max_length=max_length, **kw)


def _ragged(n, most, longest, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda hi: int(torch.randint(0, hi + 1, (1,), generator=g))  # noqa: E731
    sizes = [(r(most), 0) for _ in range(n)]
    sizes[0] = (most, 0)
    sizes[n // 2] = (0, 0)
    return [(t, t + r(longest) if i % 3 else t + r(20)) for i, (t, _) in enumerate(sizes)]


KINDS = [("16", "fp16", 64), ("16", "bf16", 128), ("int8", "fp16", 128), ("int8", "bf16", 64), ("e4m3", "fp16", 64), ("int4", "bf16", 128), ("int4", "fp16", 64)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
@pytest.mark.parametrize("fmt,rows,hd", KINDS)
def test_shared_work(backend, fmt, rows, hd, window, sinks):
    """Thirty entries of any number of rows and any length, empty ones among them; the same bits every time."""
    sizes = _ragged(30, 61, 900, hd + window)
    c = Cache(fmt, rows, 2, hd, n_seqs=30, max_len=1000, page=32, seed=hd)
    got, again = _both(backend, c, sizes, 16, seed=1, window=window, sinks=sinks)
    for _ in range(3):
        assert torch.equal(got, again())


@pytest.mark.parametrize("fmt,rows,hd", KINDS)
def test_a_sequence_much_longer_than_the_others(backend, fmt, rows, hd):
    """Its row tiles have many blocks each, the others' blocks many row tiles."""
    sizes = [(3, 40)] * 20 + [(50, 5000)] + [(50, 60)] * 20
    seqs = list(range(41))
    c = Cache(fmt, rows, 1, hd, n_seqs=41, max_len=5000, page=64, seed=hd)
    _both(backend, c, sizes, 12, seqs=seqs, seed=2)


@pytest.mark.parametrize("fmt,rows,hd", [("16", "bf16", 64), ("int8", "fp16", 128)])
def test_more_row_tiles_than_are_shared(backend, fmt, rows, hd):
    """A block a row tile: too many entries, and too many row tiles of all heads."""
    c = Cache(fmt, rows, 1, hd, n_seqs=20, max_len=200, page=16, seed=3)
    sizes = [(33 if i == 7 else i % 6, i % 6 + i * 7 % 150 if i != 7 else 180) for i in range(600)]
    _both(backend, c, sizes, 8, seqs=[i % 20 for i in range(600)], seed=3)
    c = Cache(fmt, rows, 8, hd, n_seqs=20, max_len=200, page=16, seed=4)
    sizes = [(i % 6, i % 6 + i * 7 % 150) for i in range(160)]
    _both(backend, c, sizes, 64, seqs=[i % 20 for i in range(160)], seed=4)


@pytest.mark.parametrize("heads,kvh,tokens,length", [(8, 1, 64, 6600), (32, 4, 60, 1900), (64, 8, 120, 1000), (6, 1, 300, 3000)])
@pytest.mark.parametrize("fmt,rows,hd", [("16", "fp16", 128), ("16", "bf16", 64), ("int8", "bf16", 128), ("int4", "fp16", 128)])
def test_parts_that_are_joined(backend, fmt, rows, hd, heads, kvh, tokens, length):
    """Few row tiles, from two to fifty parts; some parts have nothing to see."""
    c = Cache(fmt, rows, kvh, hd, n_seqs=1, max_len=length, page=128, seed=tokens)
    _both(backend, c, [(tokens, length)], heads, seed=5)
    _both(backend, c, [(tokens, tokens + 9)], heads, seed=6, max_length=length * 10)


@pytest.mark.parametrize("hd,heads,kvh", [(32, 6, 1), (64, 14, 2), (128, 16, 2), (256, 5, 1)])
@pytest.mark.parametrize("fmt,rows", [("16", "fp16"), ("int8", "bf16"), ("int4", "fp16")])
def test_parts_of_few_rows(backend, fmt, rows, hd, heads, kvh):
    """Single tokens and small drafts over one to thousands of positions: clusters of any size, blocks of a cluster with nothing to see,
    parts through scratch."""
    c = Cache(fmt, rows, kvh, hd, n_seqs=2, max_len=9000, page=64, seed=hd)
    for n, lengths in ((1, (130, 7)), (1, (700, 300)), (3, (1500, 3)), (1, (4000, 64)), (2, (9000, 1000)), (1, (9000, 2))):
        _both(backend, c, [(n, x) for x in lengths], heads, seed=n)
    _both(backend, c, [(1, 9000), (3, 8000)], heads, seed=9, window=3000, sinks=20)
    _both(backend, c, [(1, 9000)] * 16, heads, seqs=[0, 1] * 8, seed=10)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("fmt,rows,hd", [("16", "fp16", 64), ("16", "bf16", 128), ("int8", "fp16", 128), ("int4", "bf16", 64)])
def test_drafts_of_many_entries(backend, fmt, rows, hd, window, sinks):
    """Masks of any kind, rows among them that see nothing, of drafts that the blocks share."""
    g = torch.Generator().manual_seed(window)
    sizes = [(70 - i, 70 - i + i * 31 % 400) for i in range(24)]
    c = Cache(fmt, rows, 2, hd, n_seqs=24, max_len=520, page=16, seed=11)
    masks, pos = [], []
    for n, length in sizes:
        for i in range(n):
            bits = torch.randint(0, 2, (n,), generator=g).tolist()
            masks.append(0 if i % 9 == 4 else sum(b << j for j, b in enumerate(bits)))
            pos.append(length - n + i % 7)
    _both(backend, c, sizes, 10, seed=7, masks=masks, window=window, sinks=sinks, **(dict(q_pos=pos) if window else {}))


@pytest.mark.parametrize("scale", [-0.11, 2.0])
@pytest.mark.parametrize("fmt,rows,hd", [("16", "bf16", 128), ("int8", "fp16", 64)])
def test_scales_of_scores(backend, fmt, rows, hd, scale):
    """Scores over a negative scale, and sharp ones."""
    c = Cache(fmt, rows, 2, hd, n_seqs=12, max_len=600, page=64, seed=12)
    _both(backend, c, [(40 + i, 40 + i * 50) for i in range(12)], 8, seed=8, scale=scale)


def test_large_values_where_a_row_does_not_look(backend):
    """bf16 values near the type's largest behind a row's position, which meet weight 0, not a weight of 2^-126."""
    c = Cache("16", "bf16", 1, 128, n_seqs=40, max_len=128, page=128, seed=13)
    sizes = [(64, 128)] * 40
    for s in range(40):
        page, _ = c.place(s, 0)
        c.pool["v"][page, 0, 100:] = c.pool["v"][page, 0, 100:].sign() * 3e38
    entries, rows = _entries(sizes, list(range(40)))
    q = queries(rows, 8, 128, "bf16", 14)
    want, tol = oracle(c, q, entries, 8)
    got = run_attention(backend, c, q, entries, 8)
    looks = torch.tensor([i % 64 + 64 >= 100 for i in range(rows)])
    check(got, want, tol, ~looks)
    assert torch.isfinite(got[looks]).all()
    check(got, want, tol, looks)


@pytest.mark.parametrize("rows,hd", [("fp16", 64), ("bf16", 128)])
def test_nan_scores(backend, rows, hd):
    """A query, or a key, that is NaN: NaN where it is seen, and the other rows as they are."""
    c = Cache("16", rows, 1, hd, n_seqs=40, max_len=256, page=64, seed=15)
    entries, n = _entries([(40, 200)] * 40, list(range(40)))
    q = queries(n, 8, hd, rows, 16)
    want, tol = oracle(c, q, entries, 8)
    q[5, 2, 7] = math.nan
    page, at = c.place(3, 190)
    c.pool["k"][page, 0, at, 1] = math.nan
    got = run_attention(backend, c, q, entries, 8)
    odd = torch.zeros(n, 8, dtype=torch.bool)
    odd[5, 2] = True
    odd[3 * 40 + 30:4 * 40] = True  # positions 190 and up
    assert got[odd].isnan().all()
    check(got[~odd], want[~odd], tol[~odd])


def test_shared_work_captured_and_replayed(backend):
    """Two captures of shared work and eager calls of other sizes between their replays: nobody's parts or counters are another's."""
    c = Cache("int8", "bf16", 2, 128, n_seqs=24, max_len=700, page=32, seed=17)
    ext = torch.cuda.ExternalStream(backend.stream())
    sizes = _ragged(24, 50, 600, 5)
    entries, rows = _entries(sizes, list(range(24)))
    q = queries(rows, 16, 128, "bf16", 18)
    want, tol = oracle(c, q, entries, 16)
    qd = q.cuda()
    a = [i32([e[0] for e in entries]), i32([e[1] for e in entries] + [rows]), i32([e[3] for e in entries])]
    outs = [torch.empty_like(qd) for _ in range(3)]

    def call(o, n):
        backend.cache_attention_dev(c.view(), qd.data_ptr(), o.data_ptr(), n_rows=rows, n_entries=n, seq=a[0].data_ptr(), q_start=a[1].data_ptr(),
                                    length=a[2].data_ptr(), max_tokens=50, max_length=700, num_heads=16, q_stride=qd.stride(0), out_stride=o.stride(0))

    graphs = []
    for o in outs[:2]:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=ext):
            call(o, 24)
            call(o, 24)
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(ext):
            graphs[0].replay()
            call(outs[2], 24)
            graphs[1].replay()
            call(outs[2], 20)
        backend.synchronize()
        for o in outs:
            check(o.cpu(), want, tol)


def test_oracle_agrees_with_the_row_by_row_one():
    from cache_util import attention

    c = Cache("int4", "bf16", 2, 32, n_seqs=2, max_len=60, page=16, seed=19)
    entries, rows = _entries([(5, 60), (7, 7)], [1, 0])
    q = queries(rows, 4, 32, "bf16", 20)
    for kw in (dict(), dict(window=9, sinks=2), dict(masks=[0, 1, 3, 5, 9] + [j * 5 for j in range(7)], q_pos=list(range(12)), window=6, sinks=1)):
        for got, want in zip(oracle(c, q, entries, 4, **kw), attention(c, q, entries, 4, **kw)):
            assert torch.allclose(got, want, rtol=1e-6 if got is not None else 0, atol=1e-4)


def test_results_over_the_queries_are_refused(backend):
    from prism_engine_b200 import PrismCudaError

    c = Cache("int8", "fp16", 2, 64, n_seqs=1, max_len=32, page=16)
    x, s = torch.zeros(4, 4, 64, dtype=torch.float16, device="cuda"), i32([0, 4, 4])
    torch.cuda.synchronize()
    with pytest.raises(PrismCudaError, match="overlap") as e:
        backend.cache_attention_dev(c.view(), q=x.data_ptr(), out=x.data_ptr(), n_rows=4, n_entries=1, seq=s.data_ptr(), q_start=s.data_ptr(),
                                    length=s.data_ptr() + 4, max_tokens=4, max_length=4, num_heads=4)
    assert e.value.code == -2
