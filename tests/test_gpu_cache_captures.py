"""Attention over a cache captured again and again, as a server does that keeps a graph for each batch size and drops some: scratch
of graphs that are gone serves later captures, that of living ones nobody else's."""
import gc
import time

import pytest
import torch

from cache_util import Cache, check, i32, queries
from test_gpu_cache_many_rows import _entries, oracle

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, backend, c, sizes, heads, seed):
        self.backend, self.c, self.heads, self.sizes = backend, c, heads, sizes
        entries, self.n = _entries(sizes, [i % c.n_seqs for i in range(len(sizes))])
        q = queries(self.n, heads, c.hd, c.rows, seed)
        self.want, self.tol = oracle(c, q, entries, heads)
        self.q, self.out = q.cuda(), torch.zeros(self.n, heads, c.hd, dtype=q.dtype, device="cuda")
        self.a = [i32([e[0] for e in entries]), i32([e[1] for e in entries] + [self.n]), i32([e[3] for e in entries])]

    def __call__(self):
        seq, start, length = self.a
        self.backend.cache_attention_dev(self.c.view(), self.q.data_ptr(), self.out.data_ptr(), n_rows=self.n, n_entries=len(self.sizes),
                                         seq=seq.data_ptr(), q_start=start.data_ptr(), length=length.data_ptr(), max_tokens=max(n for n, _ in self.sizes),
                                         max_length=max(x for _, x in self.sizes), num_heads=self.heads)

    def captured(self):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(self.backend.stream())):
            self()
        return graph

    def right(self, graph=None):
        self.out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.ExternalStream(self.backend.stream())):
            graph.replay() if graph else self()
        self.backend.synchronize()
        check(self.out.cpu(), self.want, self.tol)


def _free():
    """Bytes that are free once what was dropped is."""
    gc.collect()
    torch.cuda.synchronize()
    time.sleep(0.3)
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("fmt,rows", [("int8", "bf16"), ("16", "fp16")])
def test_scratch_of_dropped_graphs_is_used_again(backend, fmt, rows):
    """Twelve captures of shared work, each dropped before the next: 39 MB each if they were kept."""
    c = Cache(fmt, rows, 2, 128, n_seqs=20, max_len=400, page=32, seed=1)
    call = Call(backend, c, [(20 + i % 9, 30 + 17 * i) for i in range(20)], 16, 2)
    graph = call.captured()
    call.right(graph)
    del graph
    before = _free()
    for _ in range(12):
        graph = call.captured()
        call.right(graph)
        graph.replay()  # dropped with its launch under way
        del graph
        left = _free()
    assert before - left < 2 * 40 << 20


def test_living_graphs_keep_their_own(backend):
    """Graphs of several sizes, dropped and captured in turn beside one that stays and eager calls that grow."""
    c = Cache("int8", "fp16", 2, 64, n_seqs=20, max_len=2100, page=64, seed=3)
    calls = [Call(backend, c, sizes, 16, 4) for sizes in ([(20, 100 + i) for i in range(20)], [(1, 2000), (2, 700)], [(30, 60 + 20 * i) for i in range(25)],
                                                          [(40, 2000)], [(33, 50 + i) for i in range(60)])]
    stays = calls[0].captured()
    for turn in range(3):
        graphs = [x.captured() for x in calls[turn:]]
        for x, g in list(zip(calls[turn:], graphs))[::-1]:
            x.right(g)
            calls[0].right(stays)
            calls[(turn + 3) % 5].right()
        del graphs, g
        _free()
        calls[0].right(stays)


def test_a_capture_that_is_given_up(backend):
    """A capture that ends with an error leaves a context that captures and runs."""
    c = Cache("int8", "fp16", 2, 64, n_seqs=20, max_len=500, page=64, seed=5)
    call = Call(backend, c, [(20, 100 + i) for i in range(20)], 16, 6)
    with pytest.raises(ZeroDivisionError):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(backend.stream())):
            call()
            raise ZeroDivisionError
    graph = None
    _free()
    call.right()
    call.right(call.captured())
