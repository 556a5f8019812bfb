"""gg_kv_attention stays within the workspace that its size function names, also where fewer rows need more."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from kv_ref import TYPES, seqs_of
from test_gpu_kv_attention import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("e4m3", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows,lengths,max_rows", [([1], [9000], None), ([3, 1, 0, 5], [9000, 40, 700, 6000], None), ([150], [9000], None), ([700], [9000], None),
                                                   ([150, 1, 30], [9000, 5000, 64], None), ([150], [9000], 1), ([2, 1], [9000, 3], 5000)])
def test_nothing_is_written_outside(gpu, rows, lengths, max_rows, cache, x):
    say("workspace", rows, lengths, max_rows, cache, x)
    c = Case(rows, lengths, 4, 2, 64, 16, cache, x)
    seqs, keep = seqs_of(c.pool, rows, lengths, max_rows=max_rows)
    pages = c.pool.pages()
    out = torch.empty(c.n, c.heads * 64, dtype=TYPES[x][1], device="cuda:0")
    lse = torch.empty(c.n, c.heads, device="cuda:0")
    for window, sinks in ((0, 0), (3000, 70)):
        n = capi.kv_attention_workspace_size(pages, seqs, c.heads, window, sinks)
        guard = 1 << 16
        buf = torch.full((n + 2 * guard,), 0xa5, dtype=torch.uint8, device="cuda:0")
        results = []
        for fill in (0xa5, 0xff):
            buf[guard:guard + n] = fill
            capi.kv_attention(pages, seqs, c.buf.data_ptr(), TYPES[x][0], c.ld, c.heads, 0.125, window, sinks, out.data_ptr(), c.heads * 64,
                              lse.data_ptr(), buf.data_ptr() + guard if n else None, stream())
            torch.cuda.synchronize()
            assert (buf[:guard] == 0xa5).all() and (buf[guard + n:] == 0xa5).all()
            results.append((out.double().cpu().numpy(), lse.double().cpu().numpy()))
        assert np.array_equal(results[0][0], results[1][0]) and np.array_equal(results[0][1], results[1][1])
        assert np.isfinite(results[0][0]).all()


def test_one_buffer_for_calls_of_all_sizes(gpu):
    """The largest size over the calls serves each of them."""
    cases = [Case(rows, lengths, 4, 1, 64, 16, "bf16", "bf16", seed=i) for i, (rows, lengths) in
             enumerate([([8192], [8192]), ([200], [6000]), ([20], [6000]), ([1], [6000]), ([1] * 20, [3000] * 20)])]
    work = []
    for c in cases:
        seqs, keep = seqs_of(c.pool, c.rows, c.lengths)
        pages = c.pool.pages()
        work.append((c, seqs, keep, pages, capi.kv_attention_workspace_size(pages, seqs, c.heads)))
    most = max(w[4] for w in work)
    assert work[0][4] < most          # not the call with the most rows
    ws = torch.empty(most, dtype=torch.uint8, device="cuda:0")
    for c, seqs, keep, pages, n in work + work[::-1]:
        want = c.run()[0]
        out = torch.empty(c.n, c.heads * 64, dtype=torch.bfloat16, device="cuda:0")
        capi.kv_attention(pages, seqs, c.buf.data_ptr(), capi.GG_TYPE_BF16, c.ld, c.heads, 0.125, 0, 0, out.data_ptr(), c.heads * 64, None,
                          ws.data_ptr(), stream())
        torch.cuda.synchronize()
        assert np.array_equal(out.double().cpu().numpy().reshape(want.shape), want)
