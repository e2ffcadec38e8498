"""The operators over a cache of several sequences as a server uses them: prompts written and attended to in portions, steps, drafts,
accepted tokens moved up; on the context's stream behind the work of others, captured and replayed, two captures in turn."""
import pytest
import torch

from cache_util import DT, Cache, attention, check, i32, queries

pytestmark = pytest.mark.gpu


def _attend(backend, c, q, out, seq, start, length, most, longest, heads, **kw):
    backend.cache_attention_dev(c.view(), q.data_ptr(), out.data_ptr(), n_rows=q.shape[0], n_entries=seq.numel(), seq=seq.data_ptr(), q_start=start.data_ptr(),
                                length=length.data_ptr(), max_tokens=most, max_length=longest, num_heads=heads, **kw)


@pytest.mark.parametrize("fmt,rows,window,sinks", [("int8", "fp16", 0, 0), ("int4", "bf16", 24, 4), ("16", "bf16", 0, 0), ("e4m3", "fp16", 24, 4)])
def test_prompt_steps_and_drafts(backend, fmt, rows, window, sinks):
    kvh, heads, hd = 2, 8, 64
    c = Cache(fmt, rows, kvh, hd, n_seqs=2, max_len=160, page=16, fill=False)
    g = torch.Generator().manual_seed(0)
    kv = lambda n: [torch.randn(n, kvh, hd, generator=g).to(DT[rows]).cuda() for _ in range(2)]  # noqa: E731
    lens = [0, 0]

    def step(new, tree=None):
        """Writes new[i] tokens of sequence i and attends for them; with a tree they are drafted."""
        rows_n = sum(new)
        k, v = kv(rows_n)
        q = queries(rows_n, heads, hd, rows, seed=sum(lens)).cuda()
        seq = [i for i, n in enumerate(new) for _ in range(n)]
        pos = [lens[i] + j for i, n in enumerate(new) for j in range(n)]
        out = torch.empty_like(q)
        a = [i32(x) for x in (seq, pos, [0, 1], [0, new[0], rows_n], [lens[i] + n for i, n in enumerate(new)])]
        more = dict(window=window, sinks=sinks)
        if tree:
            masks, depth = tree
            at = [lens[i] + depth[j] for i, n in enumerate(new) for j in range(n)]
            bits, qp = torch.tensor([masks[j] for n in new for j in range(n)]).cuda(), i32(at)
            more.update(tree=bits.data_ptr(), tree_words=1, q_pos=qp.data_ptr())
        torch.cuda.synchronize()
        backend.cache_write_dev(c.view(), k.data_ptr(), v.data_ptr(), rows_n, a[0].data_ptr(), a[1].data_ptr())
        _attend(backend, c, q, out, a[2], a[3], a[4], max(new), max(lens) + max(new), heads, **more)
        backend.synchronize()
        entries = [(i, sum(new[:i]), n, lens[i] + n) for i, n in enumerate(new)]
        extra = dict(masks=[masks[j] for n in new for j in range(n)], q_pos=at) if tree else {}
        want, tol = attention(c, q.cpu(), entries, heads, window=window, sinks=sinks, **extra)
        check(out.cpu(), want, tol)

    step([37, 50])
    lens = [37, 50]
    step([41, 3])
    lens = [78, 53]
    step([1, 1])
    lens = [79, 54]
    masks, depth = [1, 2, 5, 2 | 8, 5 | 16, 2 | 8 | 32], [0, 0, 1, 1, 2, 2]
    step([6, 6], (masks, depth))
    # tokens 1, 3, 5 of the first sequence, 0 and 2 of the second
    want = [c.parts("k", 0, 85)[2][[80, 82, 84]], c.parts("k", 1, 60)[2][[54, 56]]]
    a = [i32(x) for x in ([0, 1], lens, [[1, 3, 5], [0, 2, 0]], [3, 2])]
    torch.cuda.synchronize()
    backend.cache_keep_dev(c.view(), 2, a[0].data_ptr(), a[1].data_ptr(), a[2].data_ptr(), 3, a[3].data_ptr())
    backend.synchronize()
    assert torch.equal(c.parts("k", 0, 82)[2][79:], want[0]) and torch.equal(c.parts("k", 1, 56)[2][54:], want[1])
    lens = [82, 56]
    step([1, 1])
    lens = [83, 57]
    step([1, 2])


def test_behind_other_work_on_the_contexts_stream(backend):
    """Inputs made by kernels of the context's stream, outputs read by later ones, nothing waited for in between."""
    c = Cache("int8", "fp16", 2, 128, n_seqs=2, max_len=512, page=64)
    heads = 8
    ext = torch.cuda.ExternalStream(backend.stream())
    seq, start, length = i32([0, 1]), i32([0, 1, 2]), i32([512, 333])
    q0 = queries(2, heads, 128, "fp16").cuda()
    out = torch.empty_like(q0)
    torch.cuda.synchronize()
    with torch.cuda.stream(ext):
        q = q0 * 1
        for _ in range(20):
            q = q * 2
            q = q * 0.5
        _attend(backend, c, q, out, seq, start, length, 1, 512, heads)
        twice = out * 2
    backend.synchronize()
    want, tol = attention(c, q0.cpu(), [(0, 0, 1, 512), (1, 1, 1, 333)], heads)
    check(twice.cpu() / 2, want, tol)


@pytest.mark.parametrize("tokens", [1, 40])
def test_captured_and_replayed(backend, tokens):
    """A captured write and attention, replayed with other places and lengths; a second capture and larger eager calls between them."""
    kvh, heads, hd, most = 2, 16, 128, 6000
    c = Cache("int4", "bf16", kvh, hd, n_seqs=2, max_len=most, page=64)
    ext = torch.cuda.ExternalStream(backend.stream())
    q = queries(2 * tokens, heads, hd, "bf16").cuda()
    new = torch.randn(2 * tokens, kvh, hd, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    out, out2 = torch.empty_like(q), torch.empty_like(q)
    seq, start, length = i32([0, 1]), i32([0, tokens, 2 * tokens]), i32([tokens, tokens])
    rows_seq, rows_pos = i32([0] * tokens + [1] * tokens), i32(list(range(tokens)) * 2)

    def call(o):
        backend.cache_write_dev(c.view(), new.data_ptr(), new.data_ptr(), 2 * tokens, rows_seq.data_ptr(), rows_pos.data_ptr())
        _attend(backend, c, q, o, seq, start, length, tokens, most, heads)

    graphs = []
    for o in (out, out2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=ext):
            call(o)
        graphs.append(graph)
    big = Cache("int8", "fp16", 2, 128, n_seqs=8, max_len=2000, page=64)
    bq = queries(8, 32, 128, "fp16").cuda()
    bo = torch.empty_like(bq)
    ba = [i32(x) for x in (list(range(8)), list(range(9)), [2000] * 8)]
    torch.cuda.synchronize()
    for at in ((5000, 1234), (tokens, 77), (most, 4000)):
        lens = [max(x, tokens) for x in at]
        length.copy_(i32(lens))
        rows_pos.copy_(i32([x - tokens + j for x in lens for j in range(tokens)]))
        torch.cuda.synchronize()
        with torch.cuda.stream(ext):
            graphs[0].replay()
            _attend(backend, big, bq, bo, ba[0], ba[1], ba[2], 1, 2000, 32)
            graphs[1].replay()
        backend.synchronize()
        want, tol = attention(c, q.cpu(), [(0, 0, tokens, lens[0]), (1, tokens, tokens, lens[1])], heads)
        check(out.cpu(), want, tol)
        assert torch.equal(out, out2)
    want, tol = attention(big, bq.cpu(), [(s, s, 1, 2000) for s in range(8)], 32)
    check(bo.cpu(), want, tol)
