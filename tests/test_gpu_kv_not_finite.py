"""Attention over K/V pages with infinities and NaN in q, K and V, by the
formula: a score of +inf or a NaN leaves nothing of its row, one of -inf has
weight 0, and what the kernels do with such rows depends neither on the number
of rows nor on that of chunks."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from kv_ref import TYPES, attention, seqs_of
from test_gpu_kv_attention import Case, KINDS

pytestmark = pytest.mark.gpu
INF_KINDS = [(c, x) for c, x in KINDS if c != "e4m3"]   # 8-bit rows hold no infinity


def row_expected(q, k, v, pos, scale, cache, x):
    """One row of one head over keys 0..pos -> None where nothing is left of it, else out, lse and their bounds (V finite)."""
    with np.errstate(invalid="ignore"):
        s = np.array([np.sum(q * k[j]) for j in range(pos + 1)]) * scale
    if not (s < np.inf).all():
        return None
    some = np.flatnonzero(np.isfinite(s))
    return [t[0] for t in attention(q[None], k[some], v[some], [1 << 30], scale, 0, 0, cache, x)]


def set_key(c, s, p, d, value):
    c.pool.views()[0][c.pool.table[s, p // c.pool.page], p % c.pool.page, 0, d] = value
    c.k[s][p, 0, d] = value


def compare(c, out, lse, rows, lengths, scale=0.125, every=1):
    """-> how many (row, head) have nothing left, and how many have a score of -inf"""
    none = low = at = 0
    for s, n in enumerate(rows):
        for i in range(0, n, every):
            pos = lengths[s] - n + i
            for h in range(c.heads):
                q, k, v = c.q[at + i, h], c.k[s][:, 0], c.v[s][:, 0]
                ref = row_expected(q, k, v, pos, scale, c.cache, c.x)
                got, gl = out[at + i, h], lse[at + i, h]
                if ref is None:
                    none += 1
                    assert np.isnan(got).all() and np.isnan(gl), (s, i, h, got[:4], gl)
                else:
                    low += not np.isfinite(k[:pos + 1]).all()
                    ro, rl, bo, bl = ref
                    assert (np.abs(got - ro) <= bo).all() and abs(gl - rl) <= bl, (s, i, h, got[:4], ro[:4], gl, rl)
        at += n
    return none, low


@pytest.mark.parametrize("cache,x", INF_KINDS)
@pytest.mark.parametrize("rows,lengths", [([4, 2], [70, 100]), ([140], [200])])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_an_infinity_in_a_key(gpu, bad, dim, rows, lengths, cache, x):
    """K alone, V finite: among the first values of a head (which narrow heads are filled up with) and further back."""
    say("key", bad, dim, rows, cache, x)
    c = Case(rows, lengths, 4, 1, dim, 16, cache, x)
    set_key(c, 0, 20, 3, bad)
    set_key(c, 0, lengths[0] - max(rows[0] // 2, 1), dim - 9, bad)
    if len(rows) > 1:
        set_key(c, 1, 99, 0, bad)
    scale = np.float64(np.float32(dim ** -0.5))
    out, lse = c.run()
    none, low = compare(c, out, lse, rows, lengths, scale, every=1 if rows[0] < 100 else 7)
    assert none and low


@pytest.mark.parametrize("cache,x", INF_KINDS)
@pytest.mark.parametrize("rows", [[3], [140]])
def test_an_infinity_in_a_key_of_several_chunks(gpu, rows, cache, x):
    """Each chunk but one is finite; the join keeps what is left of the rows."""
    lengths = [12000]
    c = Case(rows, lengths, 4, 1, 64, 16, cache, x)
    seqs, keep = seqs_of(c.pool, rows, lengths)
    assert capi.kv_attention_workspace_size(c.pool.pages(), seqs, 4) > 0
    for p, bad in ((700, -np.inf), (11000, np.inf)):
        set_key(c, 0, p, 11, bad)
        out, lse = c.run(seqs=seqs)
        none, low = compare(c, out, lse, rows, lengths, every=1 if rows[0] < 100 else 23)
        assert none and (low or p > 1000)
        set_key(c, 0, p, 11, 0.5)


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows,length", [(4, 300), (150, 450), (3, 12000), (140, 12000)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_query_that_is_not_finite(gpu, bad, rows, length, cache, x):
    """Keys of both signs meet it: nothing is left of its row and head."""
    say("query", bad, rows, length, cache, x)
    c = Case([rows], [length], 3, 1, 64, 16, cache, x)
    r = rows // 2
    c.buf.view(-1, c.ld)[r, 64 + 5] = bad
    out, lse = c.run()
    assert np.isnan(out[r, 1]).all() and np.isnan(lse[r, 1])
    assert np.isfinite(np.delete(out.reshape(rows * 3, 64), 3 * r + 1, 0)).all() and np.isfinite(lse).sum() == lse.size - 1


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("rows,length", [(4, 300), (150, 450), (3, 12000), (140, 12000)])
def test_weights_that_round_to_zero_beside_an_infinity(gpu, rows, length, x):
    """A weight of e^-375 is 0 for a finite value, however large; an infinity has any weight but none."""
    c = Case([rows], [length], 2, 1, 64, 16, "bf16", x)
    q = c.buf.view(-1, c.ld)
    for h in range(2):
        q[:, 64 * h] = 30.0
        c.q[:, h, 0] = 30.0
    k_view, v_view = c.pool.views()
    place = lambda p: (c.pool.table[0, p // 16], p % 16, 0)
    for p in range(length):
        c.k[0][p, 0, 0] = 0.0
    k_view[..., 0] = 0.0
    far, near, both = 60, 100, 140
    for p in (far, both):
        set_key(c, 0, p, 0, -100.0)           # 30 * 100 / 8 = 375 below the others
    large = float(torch.tensor(1e38).bfloat16())
    v_view[place(far)][7], v_view[place(near)][9], v_view[place(both)][11] = large, np.inf, -np.inf
    c.v[0][far, 0, 7] = large
    out, lse = c.run()
    for i in range(0, rows, 1 if rows < 100 else 13):
        for h in range(2):
            ro, rl, bo, bl = (t[0] for t in attention(c.q[i:i + 1, h], c.k[0][:, 0], c.v[0][:, 0], [length - rows + i], 0.125, 0, 0, "bf16", x))
            # e^-375 times 1e38 is 10^-125
            good = ~np.isin(np.arange(64), (9, 11))
            assert (np.abs(out[i, h] - ro) <= bo)[good].all(), (i, h, out[i, h, 7], ro[7])
            assert abs(lse[i, h] - rl) <= bl and out[i, h, 9] == np.inf and out[i, h, 11] == -np.inf


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows", [4, 300])
def test_nothing_but_nan(gpu, rows, cache, x):
    """Every key and value a NaN: NaN for every row; with a page that the table lacks in their place: 0 and -inf."""
    c = Case([rows], [rows + 500], 2, 1, 64, 16, cache, x)
    for t in c.pool.views():
        t.fill_(0x7f if cache == "e4m3" else np.nan)
    out, lse = c.run()
    assert np.isnan(out).all() and np.isnan(lse).all()
    c.pool.table[:] = -1
    c.pool.table_dev.copy_(torch.from_numpy(c.pool.table))
    out, lse = c.run()
    assert (out == 0).all() and np.isneginf(lse).all()


@pytest.mark.parametrize("rows,length,heads,dim", [([256], [4096], 4, 256), ([300, 40], [3000, 2500], 8, 128), ([1] * 16, [3000] * 16, 8, 128)])
def test_one_nan_does_not_stop_a_call(gpu, rows, length, heads, dim):
    """A NaN in V that all rows see: some ten times the call's time, not hundreds of times."""
    c = Case(rows, length, heads, 1, dim, 64, "bf16", "bf16")
    seqs, keep = seqs_of(c.pool, rows, length)
    pages = c.pool.pages()
    out = torch.empty(c.n, heads * dim, dtype=torch.bfloat16, device="cuda:0")
    ws = torch.empty(max(capi.kv_attention_workspace_size(pages, seqs, heads), 16), dtype=torch.uint8, device="cuda:0")

    def best():
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            capi.kv_attention(pages, seqs, c.buf.data_ptr(), capi.GG_TYPE_BF16, c.ld, heads, dim ** -0.5, 0, 0, out.data_ptr(), heads * dim, None,
                              ws.data_ptr(), stream())
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    clean = best()
    for s in range(len(rows)):
        c.pool.views()[1][c.pool.table[s, 0], 10, 0, 7] = np.nan
    dirty = best()
    say("one NaN", rows[0], length[0], clean, dirty)
    assert torch.isnan(out.view(c.n, heads, dim)[:, :, 7]).all() and torch.isfinite(out.view(c.n, heads, dim)[:, :, 8]).all()
    assert dirty < 40 * clean


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows,length", [(6, 9000), (200, 9000)])
def test_many_keys_that_are_not_finite(gpu, rows, length, cache, x):
    """NaN, infinities and large finite values in V all along a long axis: each in a column of its own, the others as they are."""
    c = Case([rows], [length], 2, 1, 64, 16, cache, x)
    rng = np.random.default_rng(rows)
    view = c.pool.views()[1]
    cols = {3: 0x7f} if cache == "e4m3" else {3: np.nan, 20: np.inf, 41: -np.inf}
    if cache == "e4m3":
        # a NaN scale takes the whole row with it: only codes here
        for p in rng.integers(0, length - rows, 40):
            view[c.pool.table[0, p // 16], p % 16, 0, 3] = 0x7f
    else:
        for d, value in cols.items():
            for p in rng.integers(0, length - rows, 40):
                view[c.pool.table[0, p // 16], p % 16, 0, d] = value
    out, lse = c.run()
    good = ~np.isin(np.arange(64), list(cols))
    for i in range(0, rows, 1 if rows < 100 else 17):
        for h in range(2):
            ro, rl, bo, bl = (t[0] for t in attention(c.q[i:i + 1, h], c.k[0][:, 0], c.v[0][:, 0], [length - rows + i], 0.125, 0, 0, cache, x))
            assert (np.abs(out[i, h] - ro) <= bo)[good].all() and abs(lse[i, h] - rl) <= bl
            assert np.isnan(out[i, h, 3])
            assert cache == "e4m3" or out[i, h, 20] == np.inf and out[i, h, 41] == -np.inf


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows,length", [(5, 400), (5, 9000), (140, 500), (140, 9000)])
@pytest.mark.parametrize("dim", [48, 144, 192, 240, 256])
def test_every_part_of_a_head(gpu, dim, rows, length, cache, x):
    """NaN in V in the first, the middle and the last values of heads of all widths, for rows from the middle of the chunk on."""
    c = Case([rows], [length], 3, 1, dim, 16, cache, x)
    p = length - rows // 2
    cols = [0, dim // 2 - 1, dim // 2, dim - 1]
    row = c.pool.views()[1][c.pool.table[0, p // 16], p % 16, 0]
    row[cols] = 0x7f if cache == "e4m3" else np.nan
    out, lse = c.run()
    good = ~np.isin(np.arange(dim), cols)
    scale = np.float64(np.float32(dim ** -0.5))
    for i in range(0, rows, 1 if rows < 100 else 13):
        pos = length - rows + i
        for h in range(3):
            ro, rl, bo, bl = (t[0] for t in attention(c.q[i:i + 1, h], c.k[0][:, 0], c.v[0][:, 0], [pos], scale, 0, 0, cache, x))
            assert (np.abs(out[i, h] - ro) <= bo)[good | (pos < p)].all() and abs(lse[i, h] - rl) <= bl
            assert (np.isnan(out[i, h][cols]) == (pos >= p)).all()
