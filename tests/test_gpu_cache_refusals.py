"""Arrays of places, entries and positions that lie off their 4-byte boundaries are refused before anything is launched."""
import pytest
import torch

from cache_util import Cache, i32

pytestmark = pytest.mark.gpu


def test_arrays_off_their_boundaries(backend):
    from prism_engine_b200 import PrismCudaError

    c = Cache("int8", "fp16", 2, 64, n_seqs=1, max_len=32, page=16)
    x, y = (torch.zeros(4, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    s = i32([0, 4, 4, 0, 0, 0, 0, 0])
    p, o, i = x.data_ptr(), y.data_ptr(), s.data_ptr()
    torch.cuda.synchronize()

    def refused(call, *args, **kw):
        with pytest.raises(PrismCudaError, match="4-byte aligned") as e:
            call(c.view(), *args, **kw)
        assert e.value.code == -2

    for off in (1, 2, 3):
        for call in (backend.cache_write_dev, backend.cache_read_dev):
            refused(call, p, o, 4, i + off, i)
            refused(call, p, o, 4, i, i + off)
        for k in range(4):
            a = [i + (off if j == k else 0) for j in range(4)]
            refused(backend.cache_keep_dev, 1, a[0], a[1], a[2], 2, a[3])
        good = dict(q=p, out=o, n_rows=4, n_entries=1, seq=i, q_start=i, length=i + 4, max_tokens=4, max_length=4, num_heads=4, tree=p, tree_words=1,
                    window=2, q_pos=i)
        for name in ("seq", "q_start", "length", "q_pos"):
            refused(backend.cache_attention_dev, **{**good, name: good[name] + off})
    backend.synchronize()
