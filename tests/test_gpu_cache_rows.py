"""Rows of keys and values into a cache of several sequences, back out of it, and accepted drafted tokens moved up: codes and
scales are the same numbers as the definition's, since every step is one rounded 32-bit operation."""
import numpy as np
import pytest
import torch

from cache_util import DT, KINDS, U, Cache, encode, i32, pack

pytestmark = pytest.mark.gpu


def _write(backend, cache, k, v, seq, pos):
    s, p = i32(seq), i32(pos)
    torch.cuda.synchronize()
    backend.cache_write_dev(cache.view(), k.data_ptr(), v.data_ptr(), len(seq), s.data_ptr(), p.data_ptr(), k_stride=k.stride(0), v_stride=v.stride(0))
    backend.synchronize()


def _read(backend, cache, n, seq, pos, fill=7.0):
    k = torch.full((n, cache.kvh, cache.hd), fill, dtype=DT[cache.rows], device="cuda")
    v = torch.full_like(k, fill)
    s, p = i32(seq), i32(pos)
    torch.cuda.synchronize()
    backend.cache_read_dev(cache.view(), k.data_ptr(), v.data_ptr(), n, s.data_ptr(), p.data_ptr())
    backend.synchronize()
    return k.cpu(), v.cpu()


def _expect(cache, rows, seq, pos, before):
    """The pools after the rows were written, on the CPU."""
    pool = {n: before[n][0].clone() for n in ("k", "v")}
    scale = {n: None if before[n][1] is None else before[n][1].clone() for n in ("k", "v")}
    for n in ("k", "v"):
        for r, (s, p) in enumerate(zip(seq, pos)):
            if s < 0 or p < 0:
                continue
            page, at = cache.place(s, p)
            if cache.fmt == "16":
                pool[n][page, :, at] = rows[n][r]
            else:
                c, sc = encode(rows[n][r].float().numpy(), cache.fmt)
                pool[n][page, :, at] = pack(c, cache.fmt)
                scale[n][page, :, at] = torch.from_numpy(sc)
    return pool, scale


def _state(cache):
    return {n: (cache.pool[n].cpu(), None if cache.scale[n] is None else cache.scale[n].cpu()) for n in ("k", "v")}


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) if a.dtype.is_floating_point else torch.equal(a, b)


@pytest.mark.parametrize("hd,kvh", [(32, 5), (64, 2), (128, 4), (256, 1)])
@pytest.mark.parametrize("fmt,rows", KINDS)
def test_written_and_read_back(backend, fmt, rows, hd, kvh):
    """Rows with a gap between them, in any order, some of them padding; the rest of the pool stays as it was."""
    for n, page in ((1, 16), (13, 32), (70, 0)):
        c = Cache(fmt, rows, kvh, hd, n_seqs=3, max_len=100, page=page, seed=n)
        g = torch.Generator().manual_seed(n)
        wide = (torch.randn(n, 2, kvh, hd, generator=g) * torch.exp(2 * torch.randn(n, 2, kvh, 1, generator=g))).to(DT[rows]).cuda()
        new = {"k": wide[:, 0], "v": wide[:, 1]}
        places = torch.randperm(300, generator=g)[:n].tolist()
        seq, pos = [x // 100 for x in places], [x % 100 for x in places]
        if n > 4:
            seq[2], pos[3] = -1, -1
        before = _state(c)
        _write(backend, c, new["k"], new["v"], seq, pos)
        pool, scale = _expect(c, {m: new[m].cpu() for m in new}, seq, pos, before)
        for m in ("k", "v"):
            assert _same(c.pool[m].cpu(), pool[m]), m
            if fmt != "16":
                assert _same(c.scale[m].cpu(), scale[m]), m
        got = dict(zip("kv", _read(backend, c, n, seq, pos)))
        for m in ("k", "v"):
            for r, (s, p) in enumerate(zip(seq, pos)):
                if s < 0 or p < 0:
                    assert (got[m][r] == 7.0).all()
                    continue
                want = c.parts(m, s, p + 1)[2][p]
                # the value in 32 bits (a product, and a sum where there is a zero), then rounded once
                size = sum(x[p].abs() for x in c.parts(m, s, p + 1)[:2])
                assert ((got[m][r].double() - want).abs() <= U[rows] * want.abs() + 2.0 ** -22 * size + 2.0 ** -25).all()


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("rows", ["fp16", "bf16"])
def test_unusual_rows(backend, fmt, rows, hd):
    """Zeros, one value throughout, the type's smallest and largest, one large among small, and values that are not finite."""
    big = torch.finfo(DT[rows]).max
    small = 2.0 ** -24 if rows == "fp16" else 2.0 ** -133
    x = torch.randn(10, 1, hd, generator=torch.Generator().manual_seed(1))
    x[0], x[1], x[2], x[3] = 0, -2.5, small, 0.5 * big
    x[3, 0, 1], x[3, 0, 2] = -0.25 * big, 0
    x[4, 0, 5] = 3e4
    x[5, 0, 7], x[6, 0, 0], x[7, 0, hd - 1] = float("nan"), float("inf"), float("-inf")
    x[8], x[9, 0, 0], x[9, 0, 1] = -0.0, big, -big
    x = x.to(DT[rows]).cuda()
    c = Cache(fmt, rows, 1, hd, n_seqs=1, max_len=16, page=16)
    seq, pos = [0] * 10, list(range(10))
    before = _state(c)
    _write(backend, c, x, x, seq, pos)
    pool, scale = _expect(c, {"k": x.cpu(), "v": x.cpu()}, seq, pos, before)
    for m in ("k", "v"):
        assert _same(c.pool[m].cpu(), pool[m])
        a, b = c.scale[m].cpu(), scale[m]
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, 0.0), torch.nan_to_num(b, 0.0))
    got, _ = _read(backend, c, 10, seq, pos)
    assert torch.isnan(got[[5, 6, 7]].float()).all()
    assert (got[0] == 0).all() and (got[8] == 0).all()


@pytest.mark.parametrize("fmt,rows,hd", [("16", "bf16", 64), ("int8", "fp16", 128), ("e4m3", "bf16", 32), ("int4", "fp16", 256), ("int4", "bf16", 32)])
def test_accepted_tokens_move_up(backend, fmt, rows, hd):
    """Paths of no, one and many tokens, over page boundaries, with tokens that stay where they are; more than are read at once."""
    c = Cache(fmt, rows, 3, hd, n_seqs=5, max_len=200, page=16, seed=3)
    base = [0, 13, 100, 40, 7]
    paths = [[], [0], [1, 2, 5], list(range(0, 40, 2)), [3, 4, 5, 6, 7, 8, 9, 10, 11, 30, 31, 32]]
    stride = max(len(p) for p in paths) + 1
    seq, kept = [4, 0, 2, 1, -1], [len(p) for p in paths]
    flat = torch.tensor([p + [0] * (stride - len(p)) for p in paths], dtype=torch.int32).cuda()
    before = _state(c)
    want = {n: [None if t is None else t.clone() for t in before[n]] for n in before}
    for s, b, p in zip(seq, base, paths):
        for j, d in enumerate(p):
            if s < 0:
                continue
            to, frm = c.place(s, b + j), c.place(s, b + d)
            for n in ("k", "v"):
                for i in (0, 1):
                    if want[n][i] is not None:
                        want[n][i][to[0], :, to[1]] = before[n][i][frm[0], :, frm[1]]
    a = [i32(x) for x in (seq, base, kept)]
    torch.cuda.synchronize()
    backend.cache_keep_dev(c.view(), 5, a[0].data_ptr(), a[1].data_ptr(), flat.data_ptr(), stride, a[2].data_ptr())
    backend.synchronize()
    after = _state(c)
    for n in ("k", "v"):
        assert all(x is None or _same(x, y) for x, y in zip(after[n], want[n]))


def test_pools_of_more_than_2_32_bytes(backend):
    """The last pages of a pool of 5 GB: offsets of codes, scales and pages in 64 bits."""
    pages, kvh, hd, page = 5000, 8, 128, 1024
    pool = {n: torch.zeros(pages, kvh, page, hd, dtype=torch.uint8, device="cuda") for n in "kv"}
    scale = {n: torch.zeros(pages, kvh, page, device="cuda") for n in "kv"}
    import prism_engine_b200 as prism

    table = i32([[pages - 1], [2], [pages - 2]])
    view = prism.kv_cache("int8", "fp16", kvh, hd, page, pages, 3, 1, pool["k"].data_ptr(), pool["v"].data_ptr(), scale["k"].data_ptr(),
                          scale["v"].data_ptr(), table.data_ptr())
    x = torch.randn(6, kvh, hd, generator=torch.Generator().manual_seed(2)).half().cuda()
    y = torch.empty_like(x)
    z = torch.empty_like(x)
    seq, pos = i32([0, 0, 1, 2, 2, 0]), i32([0, 1023, 5, 1023, 512, 600])
    torch.cuda.synchronize()
    backend.cache_write_dev(view, x.data_ptr(), x.data_ptr(), 6, seq.data_ptr(), pos.data_ptr())
    backend.cache_read_dev(view, y.data_ptr(), z.data_ptr(), 6, seq.data_ptr(), pos.data_ptr())
    backend.synchronize()
    amax = x.float().abs().amax(-1, keepdim=True)
    # half a code, and the rounding of the result
    assert ((y.float() - x.float()).abs() <= amax / 127 * 0.5001 + 2.0 ** -11 * x.float().abs()).all() and torch.equal(y, z)
    assert int((scale["k"] != 0).sum()) == 6 * kvh and int((pool["k"][3:pages - 2] != 0).sum()) == 0
    at = torch.tensor([pages - 1, pages - 1, 2, pages - 2, pages - 2, pages - 1], device="cuda")
    assert bool((scale["v"][at, :, pos.long()] == (amax[..., 0] / torch.full_like(amax[..., 0], 127))).all())


def test_places_outside_are_skipped_and_reported(backend):
    from prism_engine_b200 import PrismCudaError

    c = Cache("int8", "fp16", 2, 64, n_seqs=2, max_len=32, page=16)
    before = _state(c)
    x = torch.ones(5, 2, 64, dtype=torch.float16, device="cuda")
    for seq, pos in (([2, 0, 0, 0, 0], [0, 0, 1, 2, 3]), ([0, 1, 1, 1, 1], [32, 0, 1, 2, 3])):
        with pytest.raises(PrismCudaError) as e:
            _write(backend, c, x, x, seq, pos)
        assert e.value.code == -2
        backend.synchronize()  # reported once
        with pytest.raises(PrismCudaError):
            _read(backend, c, 5, seq, pos)
    c.table[0, 1] = c.pages
    with pytest.raises(PrismCudaError):
        _write(backend, c, x, x, [0] * 5, [16, 17, 18, 19, 20])
    c.table[0, 1] = -5
    k, _ = torch.full((1, 2, 64), 7.0), None
    with pytest.raises(PrismCudaError):
        _read(backend, c, 1, [0], [16])
    a = [i32(v) for v in ([0], [0], [[3, 1]], [2])]
    torch.cuda.synchronize()
    backend.cache_keep_dev(c.view(), 1, a[0].data_ptr(), a[1].data_ptr(), a[2].data_ptr(), 2, a[3].data_ptr())  # 1 -> 1 stays, 3 -> 0 moves
    backend.synchronize()
    a[2].copy_(i32([[3, 0]]))
    torch.cuda.synchronize()
    backend.cache_keep_dev(c.view(), 1, a[0].data_ptr(), a[1].data_ptr(), a[2].data_ptr(), 2, a[3].data_ptr())
    with pytest.raises(PrismCudaError):
        backend.synchronize()
    assert not np.array_equal(before["k"][0].numpy(), c.pool["k"].cpu().numpy())  # the places inside were written
    assert k.numel()


def test_refusals(backend):
    from prism_engine_b200 import PrismCudaError

    c = Cache("int4", "bf16", 2, 64, n_seqs=2, max_len=32, page=16)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    s = i32([0, 0, 0, 0])
    torch.cuda.synchronize()

    def refused(code, view, k=x.data_ptr(), v=x.data_ptr(), n=4, seq=s.data_ptr(), pos=s.data_ptr(), **st):
        for call in (backend.cache_write_dev, backend.cache_read_dev):
            with pytest.raises(PrismCudaError) as e:
                call(view, k, v, n, seq, pos, **st)
            assert e.value.code == code

    for over in (dict(head_dim=80), dict(head_dim=0), dict(kv_heads=0), dict(page_size=8), dict(page_size=24), dict(n_pages=0), dict(n_seqs=0),
                 dict(table_stride=0), dict(page_table=0, n_seqs=100), dict(table_stride=1 << 27), dict(k=x.data_ptr() + 2), dict(k_scale=x.data_ptr() + 4),
                 dict(page_table=s.data_ptr() + 1)):
        refused(-2, c.view(**over))
    for over in (dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0)):
        refused(-1, c.view(**over))
    bad = c.view()
    bad.format = 4
    refused(-2, bad)
    bad = c.view()
    bad.rows = 2
    refused(-2, bad)
    refused(-2, c.view(), k=x.data_ptr() + 2)
    refused(-2, c.view(), k_stride=120)
    refused(-2, c.view(), v_stride=132)
    refused(-2, c.view(), n=1 << 30)
    for null in (dict(k=0), dict(v=0), dict(seq=0), dict(pos=0)):
        refused(-1, c.view(), **null)
    backend.cache_write_dev(c.view(), 0, 0, 0, 0, 0)  # no rows: nothing to do
    backend.cache_keep_dev(c.view(), 0, 0, 0, 0, 0, 0)
    for code, a in ((-1, (1, 0, s.data_ptr(), s.data_ptr(), 4, s.data_ptr())), (-2, (70000, s.data_ptr(), s.data_ptr(), s.data_ptr(), 4, s.data_ptr()))):
        with pytest.raises(PrismCudaError) as e:
            backend.cache_keep_dev(c.view(), *a)
        assert e.value.code == code
    import prism_engine_b200 as prism

    with pytest.raises(ValueError):
        prism.kv_cache("int3", "fp16", 1, 64, 16, 1, 1, 1, 0, 0)
    backend.synchronize()
