"""The workspace of gg_kv_attention: its size belongs to one call's structures, and may grow as rows shrink."""
import pytest

from gemma_amd import capi
from test_kv_refusals import structures


def size(n_rows, max_len, heads, kv, dim, n_seqs=1, max_rows=None, window=0, sinks=0):
    p, s = structures(pages=dict(n_kv_heads=kv, head_dim=dim, pos_stride=kv * dim, head_stride=dim, page_stride=16 * kv * dim),
                      seqs=dict(n_seqs=n_seqs, n_rows=n_rows, max_rows=max_rows or n_rows, max_len=max_len, table_ld=max_len))
    return capi.kv_attention_workspace_size(p, s, heads, window, sinks)


def test_fewer_rows_may_need_more():
    assert size(8192, 32768, 4, 1, 256) == 0 < size(1024, 32768, 4, 1, 256)
    assert size(4096, 32768, 32, 8, 128) == 0 < size(512, 32768, 32, 8, 128)


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 256), (32, 8, 128), (8, 8, 64), (16, 1, 80)])
@pytest.mark.parametrize("n_seqs", [1, 3, 64])
def test_the_bound_that_callers_are_told(heads, kv, dim, n_seqs):
    group = heads // kv
    for rows in (1, 2, 7, 16, 17, 64, 100, 1000, 5000):
        for max_len in (1, 100, 2049, 32768, 1 << 20, 1 << 30):
            for max_rows in (1, 16, rows, 100000):
                for window, sinks in ((0, 0), (512, 4), (1 << 30, 1 << 30)):
                    n = size(rows * n_seqs, max_len, heads, kv, dim, n_seqs, max_rows, window, sinks)
                    unit = rows * n_seqs * heads * (dim + 4) * 4
                    assert n % unit == 0 and n // unit != 1 and n // unit <= (256 if max_rows * group <= 64 else 64)
