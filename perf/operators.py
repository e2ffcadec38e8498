"""Operators over a quantised key/value cache, on device buffers that the caller owns.

* ``write``   rows of keys and values are quantised into their places of a cache and read back, as the portion that wrote
              them reads them (``cache_write_dev`` + ``cache_read_dev``);
* ``read``    whole sequences of a cache read back into rows (``cache_read_dev``);
* ``attend``  attention over a cache for the last tokens of each sequence, with a sliding window and first tokens that
              stay visible (``cache_attention_dev``);
* ``tree``    attention over a cache for a tree of drafted tokens of each sequence (``cache_attention_dev`` with masks);
* ``keep``    the drafted tokens that were accepted move up behind the committed ones and are read back
              (``cache_keep_dev`` + ``cache_read_dev``).

A cache is a pool of pages, ``[page][kv head][position in page][head]``, of 16-bit values or of codes:

* ``int8``   code = rint(x * (127 / amax)),             value = code * scale,            scale = amax / 127;
* ``e4m3``   code = the nearest e4m3 to x * (448 / amax), value = code * scale,          scale = amax / 448;
* ``int4``   code = rint((x - lo) * (15 / (hi - lo))),  value = (code - 8) * scale + zero, scale = (hi - lo) / 15,
             zero = lo + 8 * scale; element 2i in the low half of byte i;

amax, lo and hi over one head of one position, all of it in 32 bits.

Head layouts are those of the framework's model configurations; ``draw`` adds others.
"""
import math
import random

import torch

own = False

SHAPES = {"0p5b": (14, 2, 64), "7b": (28, 4, 128), "72b": (64, 8, 128)}  # heads, kv_heads, head_dim
TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}
WIDTH = {"16": 2.0, "int8": 1.0, "e4m3": 1.0, "int4": 0.5}  # bytes of a value
SCALES = {"16": 0, "int8": 1, "e4m3": 1, "int4": 2}  # 32-bit numbers per head and position


def _case(kind, shape, fmt, rows, seqs, tokens, length, page=64, window=0, sinks=0, ragged=False, name=None):
    h, kvh, hd = SHAPES[shape] if isinstance(shape, str) else shape
    c = dict(kind=kind, heads=h, kv_heads=kvh, head_dim=hd, fmt=fmt, rows=rows, seqs=seqs, tokens=tokens, length=length, page=page,
             window=window, sinks=sinks, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decode step's new keys and values of a small batch: launch and latency bound
        _case("write", "7b", "int8", "fp16", seqs=8, tokens=1, length=1203, name="write_step_int8"),
        # the keys and values of a long prompt portion of several sequences
        _case("write", "72b", "int4", "bf16", seqs=4, tokens=2048, length=2900, ragged=True, name="write_prompt_int4"),
        # one short sequence handed to a path that takes 16-bit rows
        _case("read", "0p5b", "int4", "fp16", seqs=1, tokens=0, length=517, page=16, name="read_short_int4"),
        # several long sequences handed over, to another cache say
        _case("read", "72b", "e4m3", "bf16", seqs=6, tokens=0, length=8000, ragged=True, name="read_long_e4m3"),
        # chat with a small model: one sequence, one token, 16-bit cache
        _case("attend", "0p5b", "16", "fp16", seqs=1, tokens=1, length=1301, window=512, sinks=4, name="attend_0p5b_step"),
        # a serving batch in decode: sequences of very different lengths, long window
        _case("attend", "72b", "int8", "fp16", seqs=32, tokens=1, length=16000, window=4096, sinks=4, ragged=True, name="attend_72b_batch"),
        # one long document, everything visible: the work of one token is spread over the GPU
        _case("attend", "72b", "int4", "bf16", seqs=1, tokens=1, length=131071, name="attend_72b_long"),
        # a prompt portion of two sequences behind what they have already
        _case("attend", "7b", "16", "bf16", seqs=2, tokens=2048, length=6001, window=1024, sinks=4, name="attend_7b_portion"),
        # a small draft for one sequence of a small model
        _case("tree", "0p5b", "int8", "fp16", seqs=1, tokens=12, length=711, page=16, name="tree_0p5b"),
        # wide drafts for a serving batch
        _case("tree", "72b", "int8", "bf16", seqs=8, tokens=63, length=4100, ragged=True, name="tree_72b_batch"),
        # what the drafts above leave: a few accepted tokens per sequence, one sequence and a batch
        _case("keep", "0p5b", "int8", "fp16", seqs=1, tokens=12, length=711, page=16, name="keep_0p5b"),
        _case("keep", "72b", "16", "bf16", seqs=64, tokens=63, length=1900, ragged=True, name="keep_72b_batch"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["write", "read", "attend", "tree", "keep"], [2, 2, 6, 4, 1])[0]
    hd = rng.choice([32, 64, 64, 128, 128, 128, 256])
    kvh = rng.choice([1, 2, 3, 4, 8])
    shape = SHAPES[rng.choice(sorted(SHAPES))] if rng.random() < 0.5 else (kvh * rng.choice([1, 2, 4, 5, 7, 8, 12]), kvh, hd)
    fmt, rows = rng.choice(["16", "int8", "e4m3", "int4"]), rng.choice(["fp16", "bf16"])
    page = rng.choice([0, 16, 32, 64, 128])
    ragged = rng.random() < 0.6
    row = shape[1] * shape[2]  # values of a cached row
    if kind == "write":
        seqs = _log(rng, 1, 32)
        tokens = _log(rng, 1, max(1, min(8192, (8 << 20) // row) // seqs))
        return _case(kind, shape, fmt, rows, seqs, tokens, tokens + rng.randint(0, 500), page, ragged=ragged)
    if kind == "read":
        seqs = _log(rng, 1, 16)
        return _case(kind, shape, fmt, rows, seqs, 0, _log(rng, 1, max(1, min(32000, (40 << 20) // (row * seqs)))), page, ragged=ragged)
    if kind == "keep":
        tokens = rng.randint(2, 64)
        return _case(kind, shape, fmt, rows, _log(rng, 1, 64), tokens, tokens + _log(rng, 1, 2000), page, ragged=ragged)
    window = rng.choice([0, 0, _log(rng, 16, 4096), _log(rng, 16, 4096)])
    sinks = rng.choice([0, 1, 4, 4, 17, 64]) if window else 0
    if kind == "tree":
        seqs, tokens = _log(rng, 1, 16), _log(rng, 2, 128)
        most = min(16000, (32 << 20) // (row * seqs), (200 << 20) // (shape[0] * seqs * tokens))
        return _case(kind, shape, fmt, rows, seqs, tokens, tokens + _log(rng, 1, max(1, most)), page, window, sinks, ragged)
    if rng.random() < 0.65:  # decode
        seqs = _log(rng, 1, 64)
        length = _log(rng, 1, max(1, min(131072, (300 << 20) // (row * seqs))))
        return _case(kind, shape, fmt, rows, seqs, rng.choice([1, 1, 1, 2, 3]), length + 2, page, window, sinks, ragged)
    seqs = _log(rng, 1, 8)  # portions of prompts
    tokens = _log(rng, 4, max(4, 4096 // seqs))
    most = min(8000, (400 << 20) // (shape[0] * seqs * tokens))
    return _case(kind, shape, fmt, rows, seqs, tokens, tokens + _log(rng, 1, max(1, most)), page, window, sinks, ragged)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lens(case):
    """Cached positions of each sequence and how many of them are its new tokens: the case's own, whatever the seed."""
    s, top, t = case["seqs"], case["length"], case["tokens"]
    lens, toks = [top] * s, [t] * s
    if case["ragged"]:
        r = random.Random(s * top + t)
        u = [[r.random() for _ in range(s)] for _ in range(2)]
        toks = [t if i == 0 or t < 2 else max(2, int(t * (0.4 + 0.6 * u[0][i]))) for i in range(s)]
        lens = [top if i == 0 else max(toks[i], 1, int(top * (0.2 + 0.8 * u[1][i]))) for i in range(s)]
    return lens, toks


def _quantise(x, fmt):
    """Codes and scales of rows [..., head_dim] in 32 bits; 16-bit caches hold the rows themselves."""
    if fmt == "16":
        return x, None
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = hi - lo if fmt == "int4" else torch.maximum(-lo, hi)
    top = torch.full_like(span, {"int4": 15.0, "int8": 127.0, "e4m3": 448.0}[fmt])  # a tensor: a number would be a product with its reciprocal
    real = span >= 2.0 ** -100
    scale = torch.where(real, span / top, torch.zeros_like(span))
    inv = torch.where(real, top / span, torch.zeros_like(span))
    if fmt == "int4":
        c = torch.where(real, torch.round((x - lo) * inv), torch.full_like(x, 8.0)).to(torch.uint8)
        return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([scale, lo + 8 * scale], -1)
    c = x * inv
    c = torch.round(c).to(torch.int8) if fmt == "int8" else c.clamp(-448, 448).to(torch.float8_e4m3fn)
    return c.view(torch.uint8), scale.squeeze(-1)


def _values(codes, scale, fmt):
    """The 32-bit values that codes and scales stand for."""
    if fmt == "16":
        return codes.float()
    if fmt == "int4":
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8
        return c * scale[..., :1] + scale[..., 1:]
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float() * scale[..., None]


def _places(lens, toks, which, device):
    """(sequence, position) of the new tokens, or of every cached one, as 32-bit arrays."""
    pairs = [(torch.full((n,), s, dtype=torch.int32), torch.arange(length - n, length, dtype=torch.int32))
             for s, (length, n) in enumerate(zip(lens, toks if which == "new" else lens))]
    return torch.cat([p[0] for p in pairs]).to(device), torch.cat([p[1] for p in pairs]).to(device)


def _tree(tokens, g):
    """Parents of a draft in the order of its levels: every token hangs on an earlier one or on the last committed token (-1)."""
    u = torch.rand(tokens, generator=g, device="cuda").tolist()
    parent, level, first = [], [], {}
    for j in range(tokens):
        p = -1 if j < max(1, tokens // 8) else max(-1, int(j * (0.3 + 0.7 * u[j])) - 2)
        parent.append(p)
        level.append(0 if p < 0 else level[p] + 1)
        first.setdefault(level[j], j)
    return parent, level


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, hd, kvh, h, fmt = TORCH[case["rows"]], case["head_dim"], case["kv_heads"], case["heads"], case["fmt"]
    lens, toks = _lens(case)
    seqs, n = case["seqs"], sum(toks)
    page = case["page"] or -(-max(lens) // 16) * 16
    page = 1 << (page - 1).bit_length()  # a cache without a table has one page per sequence
    per = -(-max(lens) // page)
    pages = seqs * per + (3 if case["page"] else 0)
    i32 = dict(dtype=torch.int32, device="cuda")
    s = dict(case=case, page=page, pages=pages, per=per, lens=torch.tensor(lens, **i32), max_len=max(lens), max_tokens=max(toks))
    s["table"] = torch.randperm(pages, generator=g, device="cuda")[:seqs * per].view(seqs, per).to(torch.int32) if case["page"] else None
    s["seq"] = torch.arange(seqs, **i32)
    # channels of keys differ in size, as projections' do
    spread = torch.exp(0.4 * torch.randn(kvh, 1, hd, generator=g, device="cuda"))

    def pool(by):
        if case["kind"] == "write":
            x = torch.zeros(pages, kvh, page, hd, device="cuda", dtype=dt)
            codes, scale = _quantise(x, fmt)
            return codes.contiguous(), scale
        parts, step = [], max(1, (64 << 20) // (kvh * page * hd))
        for at in range(0, pages, step):  # a large pool's 32-bit rows are never there at once
            x = torch.randn(min(step, pages - at), kvh, page, hd, generator=g, device="cuda") * by
            parts.append(_quantise(x.to(dt), fmt))
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]) if fmt != "16" else None

    s["k"], s["k_scale"] = pool(spread)
    s["v"], s["v_scale"] = pool(1.0)
    if case["kind"] in ("write", "read"):
        s["at_seq"], s["at_pos"] = _places(lens, toks, "new" if case["kind"] == "write" else "all", "cuda")
        rows = s["at_seq"].numel()
        if case["kind"] == "write":
            s["new_k"] = (torch.randn(rows, kvh, hd, generator=g, device="cuda") * spread.transpose(0, 1)).to(dt)
            s["new_v"] = torch.randn(rows, kvh, hd, generator=g, device="cuda").to(dt)
    elif case["kind"] == "keep":
        # accepted: one token of each level from the first on, none of them where another is moved to
        path, kept = torch.zeros(seqs, case["tokens"], dtype=torch.int32), []
        u = torch.rand(seqs, generator=g, device="cuda").tolist()
        for i, t in enumerate(toks):
            k = max(1, min(t // 2, 1 + (5 * i + 3) % 6))
            kept.append(k)
            for j in range(k):
                path[i, j] = k + j + int((t - 2 * k + 1) * u[i] * 0.99)
        s["path"], s["kept"] = path.cuda(), torch.tensor(kept, **i32)
        s["base"] = torch.tensor([a - b for a, b in zip(lens, toks)], **i32)
        s["at_seq"] = torch.repeat_interleave(s["seq"], s["kept"].long()).to(torch.int32)
        s["at_pos"] = torch.cat([torch.arange(a - b, a - b + k) for a, b, k in zip(lens, toks, kept)]).to(**i32)
        rows = sum(kept)
    else:
        s["q"] = (1.5 * torch.randn(n, h, hd, generator=g, device="cuda")).to(dt)
        start = [0]
        for t in toks:
            start.append(start[-1] + t)
        s["start"] = torch.tensor(start, **i32)
        # the place of token j of sequence i among the rows, for a dense form; behind the last one: row 0
        s["dense"] = torch.tensor([[a + min(j, t - 1) for j in range(max(toks))] for a, t in zip(start, toks)], device="cuda")
        s["toks"] = torch.tensor(toks, device="cuda")
        s["out"] = torch.empty(n, h, hd, dtype=dt, device="cuda")
        if case["kind"] == "tree":
            words = -(-max(toks) // 64)
            bits, place = [], []
            for length, t in zip(lens, toks):
                parent, level = _tree(t, g)
                masks = []
                for j, p in enumerate(parent):
                    masks.append((masks[p] if p >= 0 else 0) | 1 << j)
                bits += [[(m >> 64 * w) & (1 << 64) - 1 for w in range(words)] for m in masks]
                place += [length - t + v for v in level]
            s["tree"] = torch.tensor([[b - (1 << 64) if b >> 63 else b for b in m] for m in bits], dtype=torch.int64, device="cuda")
            s["place"] = torch.tensor(place, **i32)
        return s
    s["out_k"] = torch.empty(rows, kvh, hd, dtype=dt, device="cuda")
    s["out_v"] = torch.empty_like(s["out_k"])
    return s


# ---- the framework's calls ---------------------------------------------------------------------------------------------

_backends = {}


def _handle(s):
    """The context of this device, and the description of this cache that a program keeps beside it."""
    if "cache" not in s:
        import prism_engine_b200 as prism

        device = s["k"].device.index or 0
        if device not in _backends:
            _backends[device] = prism.CudaBackend(device=device)
        c = s["case"]
        at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        s["be"] = _backends[device]
        s["cache"] = prism.kv_cache(format=c["fmt"], rows=c["rows"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], page_size=s["page"],
                                    n_pages=s["pages"], n_seqs=c["seqs"], table_stride=s["per"], k=at(s["k"]), v=at(s["v"]),
                                    k_scale=at(s["k_scale"]), v_scale=at(s["v_scale"]), page_table=at(s["table"]))
    return s["be"], s["cache"]


def _run_own(s):
    be, cache = _handle(s)
    c = s["case"]
    if c["kind"] in ("attend", "tree"):
        tree = {} if c["kind"] == "attend" else dict(tree=s["tree"].data_ptr(), tree_words=s["tree"].shape[1], q_pos=s["place"].data_ptr())
        be.cache_attention_dev(cache, s["q"].data_ptr(), s["out"].data_ptr(), n_rows=s["q"].shape[0], n_entries=c["seqs"], seq=s["seq"].data_ptr(),
                               q_start=s["start"].data_ptr(), length=s["lens"].data_ptr(), max_tokens=s["max_tokens"], max_length=s["max_len"],
                               num_heads=c["heads"], window=c["window"], sinks=c["sinks"], **tree)
        return s["out"]
    n, at_seq, at_pos = s["at_seq"].numel(), s["at_seq"].data_ptr(), s["at_pos"].data_ptr()
    if c["kind"] == "write":
        be.cache_write_dev(cache, s["new_k"].data_ptr(), s["new_v"].data_ptr(), n, at_seq, at_pos)
    elif c["kind"] == "keep":
        be.cache_keep_dev(cache, c["seqs"], s["seq"].data_ptr(), s["base"].data_ptr(), s["path"].data_ptr(), s["path"].shape[1], s["kept"].data_ptr())
    be.cache_read_dev(cache, s["out_k"].data_ptr(), s["out_v"].data_ptr(), n, at_seq, at_pos)
    return _answer(s, s["out_k"], s["out_v"])


def _answer(s, k, v):
    out = {"k": k, "v": v}
    if s["case"]["kind"] == "write" and s["k_scale"] is not None:
        out["k_scale"], out["v_scale"] = s["k_scale"], s["v_scale"]
    return out


# ---- the plain form ----------------------------------------------------------------------------------------------------

def _rows_at(s, seq, pos):
    """Page and place in it of positions of sequences, as 64-bit indices."""
    seq, pos = seq.long(), pos.long()
    at = torch.div(pos, s["page"], rounding_mode="floor")
    page = seq * s["per"] + at if s["table"] is None else s["table"][seq, at].long()
    return page, pos % s["page"]


def _cached(s, name, page, place):
    """32-bit values of a pool at pages and places: [..., kv_heads, head_dim]."""
    scale = s[name + "_scale"]
    return _values(s[name][page, :, place], None if scale is None else scale[page, :, place], s["case"]["fmt"])


def _attend(s):
    c = s["case"]
    dev, kvh, hd = s["q"].device, c["kv_heads"], c["head_dim"]
    pos = torch.arange(s["max_len"], device=dev)
    lens = s["lens"].long()
    seq = s["seq"].long()[:, None].expand(-1, s["max_len"])
    page, place = _rows_at(s, seq, pos[None].expand_as(seq))
    k, v = _cached(s, "k", page, place), _cached(s, "v", page, place)  # [seqs, length, kv_heads, head_dim]
    q = s["q"].float()[s["dense"]].unflatten(2, (kvh, -1))             # [seqs, tokens, kv_heads, group, head_dim]
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.permute(0, 2, 3, 1)) / math.sqrt(hd)
    scores = scores.unflatten(2, (-1, s["dense"].shape[1]))             # [seqs, kv_heads, group, tokens, length]
    committed = (lens - s["toks"])[:, None]
    token = torch.arange(s["dense"].shape[1], device=dev)[None]
    if c["kind"] == "tree":
        at = s["place"].long()[s["dense"]][..., None]
        drafted = pos[None] - committed                                # [seqs, length]: which drafted token a position is
        word = drafted.clamp(0, 64 * s["tree"].shape[1] - 1)
        bits = torch.gather(s["tree"][s["dense"]], 2, (word >> 6)[:, None].expand(-1, s["dense"].shape[1], -1))
        bits = (bits >> (word & 63)[:, None]) & 1
        seen = torch.where(drafted[:, None] >= 0, bits != 0, (pos < c["sinks"]) | (pos > at - c["window"]) | (c["window"] == 0))
    else:
        at = (committed + token)[..., None]
        seen = (pos <= at) & ((pos < c["sinks"]) | (pos > at - c["window"]) | (c["window"] == 0))
    seen = seen & (pos < lens[:, None, None])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v.transpose(1, 2)).unflatten(2, (-1, s["dense"].shape[1])) / total
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)                      # [seqs, tokens, heads, head_dim]
    return out[token.expand_as(s["dense"]) < s["toks"][:, None]].to(s["q"].dtype)


def _run_plain(s):
    c = s["case"]
    if c["kind"] in ("attend", "tree"):
        return _attend(s)
    if c["kind"] == "write":
        page, place = _rows_at(s, s["at_seq"], s["at_pos"])
        codes, scale = _quantise(s["new_k"], c["fmt"])
        s["k"][page, :, place] = codes
        codes, more = _quantise(s["new_v"], c["fmt"])
        s["v"][page, :, place] = codes
        if scale is not None:
            s["k_scale"][page, :, place], s["v_scale"][page, :, place] = scale, more
    elif c["kind"] == "keep":
        j = torch.arange(s["path"].shape[1], device="cuda")
        moved = j[None] < s["kept"][:, None]
        seq = s["seq"][:, None].expand_as(moved)[moved]
        base = s["base"][:, None].expand_as(moved)[moved]
        p0, at0 = _rows_at(s, seq, base + s["path"][moved])
        p1, at1 = _rows_at(s, seq, base + j[None].expand_as(moved)[moved])
        s["k"][p1, :, at1], s["v"][p1, :, at1] = s["k"][p0, :, at0], s["v"][p0, :, at0]
        if c["fmt"] != "16":
            s["k_scale"][p1, :, at1], s["v_scale"][p1, :, at1] = s["k_scale"][p0, :, at0], s["v_scale"][p0, :, at0]
    page, place = _rows_at(s, s["at_seq"], s["at_pos"])
    dt = TORCH[c["rows"]]
    return _answer(s, _cached(s, "k", page, place).to(dt), _cached(s, "v", page, place).to(dt))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def _seen(case, length, tokens):
    """Positions of a sequence that some new token sees, and pairs of token and position, all of them causal."""
    w, first = case["window"], length - tokens
    if case["kind"] == "tree":
        return (length, tokens * (first + 8)) if not w else (min(length, w + case["sinks"] + tokens), tokens * (min(first, w + case["sinks"]) + 8))
    lo = max(0, first - w + 1) if w else 0
    union = length if lo <= case["sinks"] else length - lo + case["sinks"]
    per = [min(p + 1, w + min(case["sinks"], max(0, p - w + 1))) if w else p + 1 for p in (first, (first + length) // 2, length - 1)]
    return union, tokens * sum(per) / 3


def work(case):
    hd, kvh, h = case["head_dim"], case["kv_heads"], case["heads"]
    share_l, share_t = (0.6, 0.7) if case["ragged"] and case["seqs"] > 1 else (1.0, 1.0)
    length, tokens = max(1, int(case["length"] * share_l)), max(1, int(case["tokens"] * share_t))
    row = 2 * kvh * (hd * WIDTH[case["fmt"]] + 4 * SCALES[case["fmt"]])  # a cached position, keys and values
    wide = 2 * kvh * hd * 2                                              # the same as rows
    n = case["seqs"] * tokens
    if case["kind"] == "write":
        return {"bytes": n * 2 * (wide + row + 4), "flops": 6 * n * 2 * kvh * hd}
    if case["kind"] == "read":
        return {"bytes": case["seqs"] * length * (wide + row + 8), "flops": 2 * case["seqs"] * length * 2 * kvh * hd}
    if case["kind"] == "keep":
        kept = case["seqs"] * max(1, min(tokens // 2, 4))
        return {"bytes": kept * (3 * row + wide), "flops": 2 * kept * 2 * kvh * hd}
    seen, pairs = _seen(case, max(length, tokens), tokens)
    return {"bytes": case["seqs"] * seen * row + 2 * n * h * hd * 2, "flops": 4 * case["seqs"] * pairs * h * hd}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f64, hd, kvh, fmt = torch.float64, case["head_dim"], case["kv_heads"], case["fmt"]
    lens = s["lens"].tolist()

    def place(seq, pos):
        b = pos // s["page"]
        return (seq * s["per"] + b if s["table"] is None else s["table"][seq, b].long()), pos % s["page"]

    def stands_for(name, page, at):
        codes = s[name][page, :, at]
        if fmt == "16":
            return codes.to(f64)
        scale = s[name + "_scale"].to(f64)[page, :, at]
        if fmt == "int4":
            c = torch.empty(*codes.shape[:-1], hd, dtype=f64, device=codes.device)
            c[..., 0::2], c[..., 1::2] = (codes % 16).to(f64), torch.div(codes, 16, rounding_mode="floor").to(f64)
            return (c - 8) * scale[..., 0:1] + scale[..., 1:2]
        return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).to(f64) * scale.unsqueeze(-1)

    if case["kind"] in ("write", "keep", "read"):
        out = {}
        page, at = place(s["at_seq"].long(), s["at_pos"].long())
        for name in ("k", "v"):
            if case["kind"] == "keep":
                base, path = s["base"].tolist(), s["path"].tolist()
                src = torch.tensor([base[i] + path[i][j] for i, k in enumerate(s["kept"].tolist()) for j in range(k)], device="cuda")
                out[name] = stands_for(name, *place(s["at_seq"].long(), src))
            elif case["kind"] == "read" or fmt == "16":
                out[name] = stands_for(name, page, at) if case["kind"] == "read" else s["new_" + name].to(f64)
            else:
                x = s["new_" + name].to(f64)
                scales = s[name + "_scale"].to(f64)
                r = lambda y: y.to(torch.float32).to(f64)  # noqa: E731  a code is chosen by 32-bit steps: each rounded by itself
                if fmt == "int4":
                    lo, span = x.amin(-1), x.amax(-1) - x.amin(-1)
                    scales[page, :, at] = torch.stack([span / 15, lo + 8 * (span / 15)], -1)
                    c = torch.round(r(r(x - lo[..., None]) * r(15 / r(span))[..., None]))
                    out[name] = lo[..., None] + c * (span / 15)[..., None]
                else:
                    amax, top = x.abs().amax(-1), 127 if fmt == "int8" else 448
                    scales[page, :, at] = amax / top
                    y = r(x * r(top / amax)[..., None]).clamp(-top, top)
                    # three bits behind the leading one down to 2^-6, multiples of 2^-9 below that
                    grain = torch.ones_like(y) if fmt == "int8" else torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                    out[name] = torch.round(y / grain) * grain * (amax / top)[..., None]
                out[name + "_scale"] = scales
        if case["kind"] == "write" and fmt != "16":
            return {"k": out["k"], "v": out["v"], "k_scale": out["k_scale"], "v_scale": out["v_scale"]}
        return {"k": out["k"], "v": out["v"]}
    q, group = s["q"].to(f64), case["heads"] // kvh
    toks, start, parts = s["toks"].tolist(), s["start"].tolist(), []
    for i, (length, n) in enumerate(zip(lens, toks)):
        pos = torch.arange(length, device="cuda")
        page, at = place(torch.full_like(pos, i), pos)
        k, v = stands_for("k", page, at), stands_for("v", page, at)
        mine = torch.empty(n, case["heads"], hd, dtype=f64, device="cuda")
        step = max(1, (1 << 28) // (length * group))
        for t0 in range(0, n, step):
            t = torch.arange(t0, min(n, t0 + step), device="cuda")
            where = length - n + t if case["kind"] == "attend" else s["place"].long()[start[i] + t]
            see = pos[None, :] <= where[:, None] if case["kind"] == "attend" else (pos[None, :] < length - n).expand(len(t), -1).clone()
            if case["window"]:
                see = see & ((pos[None, :] < case["sinks"]) | (where[:, None] - pos[None, :] < case["window"]))
            if case["kind"] == "tree":
                for j in range(n):
                    see[:, length - n + j] = (s["tree"][start[i] + t, j // 64] >> (j % 64)) & 1 != 0
            for m in range(kvh):
                rows = q[start[i] + t, m * group:(m + 1) * group]
                x = torch.einsum("tgd,pd->tgp", rows, k[:, m]) / math.sqrt(hd)
                x = torch.softmax(x.masked_fill(~see[:, None], -math.inf), -1)
                mine[t0:t0 + step, m * group:(m + 1) * group] = torch.einsum("tgp,pd->tgd", x, v[:, m])
        parts.append(mine)
    return torch.cat(parts)
