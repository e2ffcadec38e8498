"""Caches of several sequences for the tests: pools on the GPU, and what they stand for in 64 bits on the CPU."""
import math

import numpy as np
import torch

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of a rounded value, relative to it: bf16 has 8 significant bits
KINDS = [("16", "fp16"), ("16", "bf16"), ("int8", "fp16"), ("int8", "bf16"), ("e4m3", "fp16"), ("int4", "bf16"), ("int4", "fp16")]


def encode(x, fmt):
    """Codes (one a value) and scales of float32 rows [..., head_dim]: one rounded 32-bit operation a step."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        amax = np.abs(x).max(-1, keepdims=True)
        span = (hi - lo).astype(np.float32) if fmt == "int4" else amax
        top = np.float32({"int8": 127, "e4m3": 448, "int4": 15}[fmt])
        real = span >= np.float32(2.0 ** -100)
        scale = np.where(real, span / top, np.float32(0)).astype(np.float32)
        inv = np.where(real, top / span, np.float32(0)).astype(np.float32)
        odd = ~np.isfinite(amax) | ~np.isfinite(span)
        if fmt == "int4":
            c = np.where(real & ~odd, np.rint((x - lo) * inv), np.float32(8))
            sc = np.concatenate([scale, lo + np.float32(8) * scale], -1).astype(np.float32)
        else:
            c = np.where(odd, np.float32(0), x * inv)
            c = np.rint(c) if fmt == "int8" else torch.from_numpy(np.clip(c, -448, 448)).to(torch.float8_e4m3fn).float().numpy()
            sc = scale
        sc = np.where(odd, np.float32(np.nan), sc)
    return c.astype(np.float32), sc[..., 0] if fmt != "int4" else sc


def pack(c, fmt):
    """Codes as the bytes of a pool."""
    c = torch.from_numpy(np.ascontiguousarray(c))
    if fmt == "int8":
        return c.to(torch.int8).view(torch.uint8)
    if fmt == "e4m3":
        return c.to(torch.float8_e4m3fn).view(torch.uint8)
    c = c.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def unpack(b, fmt):
    b = b.cpu().contiguous()
    if fmt == "int4":
        return torch.stack([b & 15, b >> 4], -1).flatten(-2).double() - 8
    return b.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).double()


class Cache:
    """A pool of its own for k and v; ``page`` 0: no table, one page a sequence."""

    def __init__(self, fmt, rows, kvh, hd, n_seqs, max_len, page=16, seed=0, spare=2, fill=True):
        self.fmt, self.rows, self.kvh, self.hd, self.n_seqs = fmt, rows, kvh, hd, n_seqs
        self.page = page or 1 << max(4, (max_len - 1).bit_length())
        self.per = max(1, -(-max_len // self.page))
        g = torch.Generator().manual_seed(seed)
        self.pages = n_seqs * self.per + (spare if page else 0)
        self.table_cpu = torch.randperm(self.pages, generator=g)[:n_seqs * self.per].view(n_seqs, self.per).int() if page else None
        if not page:
            self.table_cpu = torch.arange(n_seqs * self.per).view(n_seqs, self.per).int()
        self.table = self.table_cpu.cuda() if page else None
        shape = (self.pages, kvh, self.page)
        self.pool, self.scale = {}, {}
        for i, n in enumerate(("k", "v")):
            x = torch.randn(*shape, hd, generator=g) * (torch.exp(0.4 * torch.randn(hd, generator=g)) if i == 0 else 1.0) if fill else torch.zeros(*shape, hd)
            x = x.to(DT[rows])
            if fmt == "16":
                self.pool[n], self.scale[n] = x.cuda(), None
            else:
                c, s = encode(x.float().numpy(), fmt)
                self.pool[n], self.scale[n] = pack(c, fmt).cuda(), torch.from_numpy(np.ascontiguousarray(s)).cuda()

    def view(self, **over):
        import prism_engine_b200 as prism

        at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        a = dict(format=self.fmt, rows=self.rows, kv_heads=self.kvh, head_dim=self.hd, page_size=self.page, n_pages=self.pages, n_seqs=self.n_seqs,
                 table_stride=self.per, k=at(self.pool["k"]), v=at(self.pool["v"]), k_scale=at(self.scale["k"]), v_scale=at(self.scale["v"]),
                 page_table=at(self.table))
        a.update(over)
        return prism.kv_cache(**a)

    def place(self, s, p):
        return int(self.table_cpu[s, p // self.page]), p % self.page

    def parts(self, name, s, n):
        """(code * scale, zero, value) of the first n positions of a sequence in 64 bits: [n, kv_heads, head_dim]."""
        pool = self.pool[name].cpu()
        page = self.table_cpu[s].long()[torch.arange(n) // self.page]
        at = torch.arange(n) % self.page
        rows = pool[page, :, at]
        if self.fmt == "16":
            x = rows.double()
            return x, torch.zeros_like(x), x
        sc = self.scale[name].cpu().double()[page, :, at]
        c = unpack(rows, self.fmt)
        if self.fmt == "int4":
            a, z = c * sc[..., :1], sc[..., 1:].expand_as(c)
            return a, z, a + z
        a = c * sc[..., None]
        return a, torch.zeros_like(a), a


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def attention(cache, q, entries, heads, window=0, sinks=0, scale=None, masks=None, q_pos=None):
    """q [rows, heads, hd] (CPU), entries: (sequence, first row, rows, length).  Returns the outputs and, per output, how far they may
    be off: the rounding of the result, that of the weights (16 bits each, in the sums above and below the line), and the scores'."""
    hd, group = cache.hd, heads // cache.kvh
    scale = scale or 1 / math.sqrt(hd)
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64)
    tol = torch.zeros_like(out)
    u_p = U[cache.rows] if cache.fmt == "16" else U["fp16"]
    for s, r0, n, length in entries:
        ka, kz, k = cache.parts("k", s, length)
        va, vz, v = cache.parts("v", s, length)
        first = length - n
        for i in range(n):
            c = torch.arange(length)
            if masks is None:
                p = first + i
                see = c <= p
                if window:
                    see &= (c > p - window) | (c < sinks)
            else:
                p = q_pos[r0 + i] if q_pos is not None else first
                see = c < first
                if window:
                    see &= (c > p - window) | (c < sinks)
                for j in range(n):
                    if first + j >= 0:
                        see[first + j] = bool(masks[r0 + i] >> j & 1)
            if not see.any():
                continue
            for h in range(heads):
                m = h // group
                x = q[r0 + i, h].double()
                sc = k[see, m] @ x * scale
                w = torch.softmax(sc, 0)
                out[r0 + i, h] = w @ v[see, m]
                size = w @ (va[see, m].abs() + vz[see, m].abs())
                # scores: head_dim additions of 2^-24 each, and a query's smallest elements in 16 bits beside its largest
                off = scale * (hd * 2.0 ** -24 * ((ka[see, m].abs() + kz[see, m].abs()) @ x.abs()).max()
                               + 2.0 ** -24 * float(x.abs().max()) * float((ka[see, m].abs() + kz[see, m].abs()).sum(-1).max())) + 2.0 ** -20
                # weights are multiples of 2^-39 of the largest (times the largest scale), results of 2^-24 (fp16) or 2^-133
                least = 2.0 ** -37 * float(w.max()) * len(w) * float((va[see, m].abs() + vz[see, m].abs()).max())
                tol[r0 + i, h] = (2 * u_p + 2 * off) * size + U[cache.rows] * out[r0 + i, h].abs() + least + (2.0 ** -25 if cache.rows == "fp16" else 2.0 ** -134)
    return out, tol


def run_attention(backend, cache, q, entries, heads, window=0, sinks=0, scale=0.0, masks=None, q_pos=None, out=None, seqs=None, max_length=None):
    """The library's result for the same arguments, on the CPU.  Entries' rows follow each other."""
    qd = q.cuda()
    out = torch.full_like(qd, 7.0) if out is None else out
    start = [e[1] for e in entries] + [entries[-1][1] + entries[-1][2]] if entries else [0]
    most = max([e[2] for e in entries] + [0])
    more = {}
    if masks is not None:
        words = max(1, -(-most // 64))
        signed = [[(m >> 64 * w & (1 << 64) - 1) - (1 << 64 if m >> 64 * w + 63 & 1 else 0) for w in range(words)] for m in masks]
        t = torch.tensor(signed, dtype=torch.int64).cuda()
        more = dict(tree=t.data_ptr(), tree_words=words)
        if q_pos is not None:
            qp = i32(q_pos)
            more["q_pos"] = qp.data_ptr()
    seq, st, ln = i32(seqs or [e[0] for e in entries]), i32(start), i32([e[3] for e in entries])
    torch.cuda.synchronize()
    backend.cache_attention_dev(cache.view(), qd.data_ptr(), out.data_ptr(), n_rows=q.shape[0], n_entries=len(entries), seq=seq.data_ptr(),
                                q_start=st.data_ptr(), length=ln.data_ptr(), max_tokens=most,
                                max_length=max_length if max_length is not None else max([e[3] for e in entries] + [0]),
                                num_heads=heads, window=window, sinks=sinks, scale=scale, q_stride=qd.stride(0), out_stride=out.stride(0), **more)
    backend.synchronize()
    return out.cpu()


def check(got, want, tol, rows=None):
    rows = slice(None) if rows is None else rows
    d = (got[rows].double() - want[rows]).abs()
    bad = ~(d <= tol[rows])
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} too far off, worst {float((d / tol[rows].clamp(min=1e-30)).max()):.3g} times the bound"


def queries(rows, heads, hd, dtype, seed=0):
    return (1.5 * torch.randn(rows, heads, hd, generator=torch.Generator().manual_seed(seed))).to(DT[dtype])
