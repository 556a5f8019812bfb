"""Attention over K/V pages against a 64-bit plain form."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from kv_ref import LEAST, Pool, TYPES, attention, seqs_of, typed

pytestmark = pytest.mark.gpu
KINDS = [("bf16", "f32"), ("bf16", "bf16"), ("bf16", "f16"), ("f16", "f16"), ("e4m3", "f32"), ("e4m3", "bf16"), ("e4m3", "f16")]


class Case:
    """Sequences with their pools' contents; q on the device."""

    def __init__(self, rows, lengths, group, n_kv, dim, page, cache, x, layout="phd", seed=0, gap=0, offset=0, q_scale=2.0, spare=3):
        rng = np.random.default_rng(seed + 17 * sum(lengths) + dim)
        self.rows, self.lengths, self.group, self.n_kv, self.dim, self.cache, self.x = rows, lengths, group, n_kv, dim, cache, x
        self.heads, self.n = n_kv * group, sum(rows)
        self.pool = Pool(lengths, page, n_kv, dim, cache, seed=seed, layout=layout, spare=spare)
        self.k, self.v = [], []
        for s, n in enumerate(lengths):
            k, v = rng.standard_normal((2, n, n_kv, dim))
            e = rng.integers(-8, -5, (2, n, n_kv)).astype(np.float64)
            if cache == "e4m3":
                k, v = k * 100 * np.exp2(e[0])[:, :, None], v * 100 * np.exp2(e[1])[:, :, None]
            k, v = self.pool.put(s, k, v, e)
            self.k.append(k)
            self.v.append(v)
        self.offset, self.ld = offset, self.heads * dim + gap
        self.buf = torch.full((offset + max(self.n, 1) * self.ld,), 55.0, dtype=TYPES[x][1], device="cuda:0")
        t, q = typed(rng.standard_normal((self.n, self.heads * dim)) * q_scale, x)
        self.buf[offset:].view(-1, self.ld)[:self.n, :self.heads * dim] = t
        self.q = q.reshape(self.n, self.heads, dim)

    def run(self, scale=None, window=0, sinks=0, seqs=None, lse=True, max_len=None, max_rows=None):
        """-> out [n, heads, dim], lse [n, heads]"""
        scale = self.dim ** -0.5 if scale is None else scale
        if seqs is None:
            seqs, self.keep = seqs_of(self.pool, self.rows, self.lengths, max_len=max_len, max_rows=max_rows)
        ldo = self.heads * self.dim + 3
        out = torch.full((seqs.n_rows, ldo), -9.0, dtype=TYPES[self.x][1], device="cuda:0")
        l = torch.full((seqs.n_rows, self.heads), -9.0, device="cuda:0")
        pages = self.pool.pages()
        ws = torch.full((max(capi.kv_attention_workspace_size(pages, seqs, self.heads, window, sinks), 16),), 255, dtype=torch.uint8,
                        device="cuda:0")
        capi.kv_attention(pages, seqs, self.buf.data_ptr() + self.offset * self.buf.element_size(), TYPES[self.x][0], self.ld, self.heads,
                          scale, window, sinks, out.data_ptr(), ldo, l.data_ptr() if lse else None, ws.data_ptr(), stream())
        torch.cuda.synchronize()
        assert (out[:, self.heads * self.dim:] == -9).all()
        return out[:, :self.heads * self.dim].double().cpu().numpy().reshape(seqs.n_rows, self.heads, self.dim), l.double().cpu().numpy()

    def check(self, scale=None, window=0, sinks=0, every=1, lengths=None, hidden=(), **more):
        """Against 64 bits, every `every`-th row of a sequence; hidden: (sequence, page index) that the table lacks."""
        scale = self.dim ** -0.5 if scale is None else scale
        out, lse = self.run(scale, window, sinks, **more)
        at = 0
        for s, n in enumerate(self.rows):
            length = self.lengths[s] if lengths is None else lengths[s]
            pick = sorted(set(range(0, n, every)) | set(range(max(n - 2, 0), n)))
            pos = length - n + np.array(pick, int)
            keys = np.arange(min(length, len(self.k[s])))
            for sq, pg in hidden:
                if sq == s:
                    keys = keys[keys // self.pool.page != pg]
            for h in range(self.heads) if pick else ():
                kh = h // self.group
                q = self.q[at + np.array(pick), h]
                k, v = self.k[s][keys, kh], self.v[s][keys, kh]
                # keys that are not there: positions the reference function never sees
                full_k, full_v = np.zeros((length, self.dim)), np.zeros((length, self.dim))
                full_k[keys], full_v[keys] = k, v
                ro, rl, bo, bl = reference(q, full_k, full_v, keys, pos, np.float32(scale).astype(np.float64), window, sinks, self.cache, self.x)
                got, gl = out[at + np.array(pick), h], lse[at + np.array(pick), h]
                assert (np.abs(got - ro) <= bo).all(), (s, h, np.abs(got - ro).max(), (np.abs(got - ro) / bo).max())
                none = np.isneginf(rl)
                assert (np.isneginf(gl) == none).all()
                off = np.abs(gl[~none] - rl[~none])
                assert (off <= bl[~none]).all(), (s, h, (off / bl[~none]).max())
                assert (got[none] == 0).all()
            at += n
        return out, lse


def reference(q, k, v, keys, pos, scale, window, sinks, cache, x):
    if len(keys) == len(k):
        return attention(q, k, v, pos, scale, window, sinks, cache, x)
    # with holes: each row on the keys that it sees, as if they were all
    out = [attention(q[i:i + 1], *(t[[j for j in keys if j <= p and (not window or j > p - window or j < sinks)]] for t in (k, v)),
                     [1 << 30], scale, 0, 0, cache, x) for i, p in enumerate(pos)]
    return tuple(np.concatenate([o[i] for o in out]) for i in range(4))


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 192, 256])
def test_single_tokens(gpu, dim, cache, x):
    say("tokens", dim, cache, x)
    Case([1] * 6, [1, 2, 33, 129, 700, 2500], 4, 2, dim, 16, cache, x).check()


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows,lengths,group,n_kv,dim,page,layout,gap,offset", [
    ([3, 1, 0, 8, 5], [3, 64, 9, 300, 1000], 1, 3, 64, 16, "hpd", 3, 1),
    ([6, 2], [6, 513], 3, 2, 96, 24, "both", 8, 8),
    ([9, 30, 17], [100, 31, 2000], 8, 1, 128, 1, "pad", 1, 0),
    ([5, 33], [1500, 90], 5, 2, 256, 100, "phd", 0, 4),
    ([40], [40], 2, 2, 32, 1000, "phd", 0, 0),
    ([1, 16], [4097, 16], 16, 1, 192, 64, "hpd", 0, 0),
])
def test_chunks(gpu, rows, lengths, group, n_kv, dim, page, layout, gap, offset, cache, x):
    say("chunks", rows, lengths, group, n_kv, dim, page, layout, cache, x)
    Case(rows, lengths, group, n_kv, dim, page, cache, x, layout, gap=gap, offset=offset).check()


@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("bf16", "f32"), ("e4m3", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("rows,lengths,group,n_kv,dim,page", [
    ([300, 129, 1], [300, 1000, 500], 4, 1, 256, 64),
    ([500, 64], [500, 900], 1, 2, 128, 16),
    ([257, 255, 3], [700, 255, 700], 3, 2, 80, 24),
    ([1025], [3000], 2, 1, 64, 100),
])
def test_long_chunks(gpu, rows, lengths, group, n_kv, dim, page, cache, x):
    say("long chunks", rows, lengths, group, n_kv, dim, page, cache, x)
    Case(rows, lengths, group, n_kv, dim, page, cache, x).check(every=7)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 70), (16, 4), (33, 33), (512, 4), (700, 1000), (5000, 2), (1 << 30, 1 << 30)])
@pytest.mark.parametrize("rows,cache,x", [([1, 1, 1], "bf16", "f32"), ([7, 1, 20], "e4m3", "bf16"), ([200, 30, 400], "bf16", "bf16"),
                                          ([130, 7, 600], "f16", "f16")])
def test_windows_and_first_positions(gpu, rows, cache, x, window, sinks):
    say("window", window, sinks, rows, cache, x)
    Case(rows, [max(rows[0], 40), 900, 1800], 4, 1, 64, 24, cache, x).check(window=window, sinks=sinks, every=5)


@pytest.mark.parametrize("rows", [[1, 2, 5], [3, 40, 200]])
@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("e4m3", "f32"), ("f16", "f16")])
def test_rows_that_see_nothing(gpu, rows, cache, x):
    """Positions below zero, empty sequences, lengths past max_len, tables without pages."""
    c = Case(rows, [max(rows) + 60] * 3, 2, 2, 64, 8, cache, x)
    c.pool.table[2, :] = -1
    c.pool.table_dev.copy_(torch.from_numpy(c.pool.table))
    lengths = [0, rows[1] - 1, rows[2] + 50]
    seqs, keep = seqs_of(c.pool, rows, lengths, max_len=max(lengths))
    hidden = [(2, i) for i in range(c.pool.table.shape[1])]
    out, lse = c.check(seqs=seqs, lengths=lengths, hidden=hidden)
    assert (out[:rows[0]] == 0).all() and np.isneginf(lse[:rows[0]]).all()
    assert (out[rows[0]] == 0).all() and np.isneginf(lse[rows[0]]).all()       # the row at position -1
    assert (out[sum(rows[:2]):] == 0).all()


@pytest.mark.parametrize("rows", [[2, 1, 9], [150, 4, 300]])
def test_holes_and_bounds(gpu, rows):
    """Unmapped and foreign pages within a sequence, a length above max_len, a table that ends before it."""
    c = Case(rows, [400, 400, 400], 4, 1, 128, 16, "bf16", "bf16")
    hidden = [(0, 3), (0, 24), (1, 0), (2, 20)]
    for (s, i), to in zip(hidden, (-1, c.pool.n_pages, 1 << 30, -(1 << 30))):
        c.pool.table[s, i] = to
    c.pool.table_dev.copy_(torch.from_numpy(c.pool.table))
    c.check(hidden=hidden, every=5)
    c.check(hidden=hidden, max_len=390, lengths=[390] * 3, every=5)
    seqs, keep = seqs_of(c.pool, rows, [400] * 3)
    short = torch.from_numpy(c.pool.table[:, :20].copy()).cuda()
    seqs.table, seqs.table_ld = short.data_ptr(), 20
    c.check(seqs=seqs, hidden=hidden + [(s, i) for s in range(3) for i in range(20, 25)], every=5)


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [[1, 1], [6, 5], [200, 130]])
def test_other_rows_are_left_alone(gpu, rows, x):
    c = Case(rows, [300, 200], 2, 1, 64, 16, "bf16", x)
    n = sum(rows)
    seqs, keep = seqs_of(c.pool, rows, [300, 200], n_rows=3 + n + 4, first=3)
    big = torch.zeros((n + 7) * c.ld, dtype=c.buf.dtype, device="cuda:0")
    big[3 * c.ld:(3 + n) * c.ld] = c.buf[:n * c.ld]
    plain = c.run()
    c.buf = big
    out, lse = c.run(seqs=seqs)
    assert (out[:3] == -9).all() and (out[3 + n:] == -9).all() and (lse[:3] == -9).all() and (lse[3 + n:] == -9).all()
    assert np.array_equal(out[3:3 + n], plain[0]) and np.array_equal(lse[3:3 + n], plain[1])


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows", [[4, 2], [150, 40]])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_has_no_effect(gpu, rows, cache, x, bad):
    """NaN and infinities in K and V of later rows of the chunk and of positions before the window."""
    lengths = [rows[0] + 70, rows[1] + 300]
    window, sinks = 64, 3
    c = Case(rows, lengths, 4, 1, 64, 16, cache, x)
    clean, clean_lse = c.run(window=window, sinks=sinks)
    views = c.pool.views()
    # (sequence, position, value index) in K and V
    places = [(0, lengths[0] - 1, 5), (1, lengths[1] - rows[1] // 2, 63), (1, 100, 0), (0, lengths[0] - rows[0] // 2 - 1, 40)]
    for i, (s, p, d) in enumerate(places):
        for t in range(2):
            view = views[t][c.pool.table[s, p // 16], p % 16, 0]
            if cache == "e4m3":
                view[d] = 0x7f
            else:
                view[d] = bad
    out, lse = c.run(window=window, sinks=sinks)
    at, touched = 0, 0
    for s, n in enumerate(rows):
        for i in range(n):
            pos = lengths[s] - n + i
            meets = any(sq == s and p <= pos and (p > pos - window or p < sinks) for sq, p, _ in places)
            touched += meets
            if not meets:
                # rows beside ones that need care may be summed in another order: within the bounds of the clean values
                for h in range(4) if not np.array_equal(out[at + i], clean[at + i]) or not np.array_equal(lse[at + i], clean_lse[at + i]) else ():
                    ro, rl, bo, bl = attention(c.q[at + i:at + i + 1, h], c.k[s][:, 0], c.v[s][:, 0], [pos], 0.125, window, sinks, cache, x)
                    assert (np.abs(out[at + i, h] - ro[0]) <= bo[0]).all() and abs(lse[at + i, h] - rl[0]) <= bl[0]
            else:
                # a score of -inf has weight 0: an infinity in K that every head's q meets with one sign may leave lse finite
                assert np.isnan(lse[at + i]).all() if cache == "e4m3" or np.isnan(bad) else not np.isfinite(out[at + i]).all()
        at += n
    assert 0 < touched < sum(rows)


@pytest.mark.parametrize("x,cache", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("rows", [[4], [140]])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_infinite_values_of_seen_keys(gpu, rows, x, cache, bad):
    """An infinity or NaN in V alone reaches its own column of the rows that see it, as the formula has it, and nothing else."""
    n = rows[0]
    c = Case(rows, [n + 40], 2, 1, 64, 16, cache, x)
    clean, clean_lse = c.run()
    p = n + 40 - max(n // 2, 1)
    c.pool.views()[1][c.pool.table[0, p // 16], p % 16, 0, 17] = bad
    out, lse = c.run()
    see = (40 + np.arange(n)) >= p
    # rows that need care may be summed in another order
    for i in range(n):
        for h in range(2):
            ro, rl, bo, bl = attention(c.q[i:i + 1, h], c.k[0][:, 0], c.v[0][:, 0], [40 + i], 0.125, 0, 0, cache, x)
            good = (np.arange(64) != 17) | (not see[i])
            assert (np.abs(out[i, h] - ro[0]) <= bo[0])[good].all() and abs(lse[i, h] - rl[0]) <= bl[0]
    assert (np.isnan(out[see][:, :, 17]) if np.isnan(bad) else out[see][:, :, 17] == bad).all()


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows", [[1, 3], [90, 130]])
def test_peaked_and_far_scores(gpu, rows, cache, x):
    """Scores in the hundreds that rise and fall along the axis, weights that round to 0, equal scores, scale 0 and below it."""
    c = Case(rows, [400, 700], 2, 1, 64, 32, cache, x, q_scale=30.0)
    for scale in (1.0, -0.5, 0.0, 1e-3):
        say("scale", scale, cache, x, rows)
        c.check(scale=scale, every=5)


@pytest.mark.parametrize("cache,x", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("rows", [1, 6, 150])
def test_one_key_comes_out_as_it_is(gpu, rows, cache, x):
    """A window of one: out is v of the row's own position, to the type's last bit."""
    c = Case([rows], [rows + 200], 2, 2, 64, 16, cache, x)
    out, lse = c.run(window=1)
    v = np.repeat(c.v[0][200:], 2, axis=1)
    ref = typed(v, x)[1]
    assert np.array_equal(out, ref)


@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("e4m3", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows", [[1, 1, 1], [5, 1, 3], [140, 1, 60]])
def test_repeats_bit_for_bit_and_bounds_do_not_matter(gpu, rows, cache, x):
    """The same call again, without lse, and with a wrong max_rows."""
    c = Case(rows, [3000, 200, 1000], 4, 1, 128, 16, cache, x)
    out, lse = c.run()
    again, _ = c.run(lse=False)
    assert np.array_equal(out, again)
    for mr in (1, 4000):
        c.check(max_rows=mr, every=11)


def test_shared_pages(gpu):
    """Two sequences whose tables begin with the same pages."""
    c = Case([2, 3], [200, 100], 2, 1, 64, 16, "bf16", "bf16")
    c.pool.table[1, :3] = c.pool.table[0, :3]
    c.pool.table_dev.copy_(torch.from_numpy(c.pool.table))
    c.k[1][:48], c.v[1][:48] = c.k[0][:48], c.v[0][:48]
    c.check()


@pytest.mark.parametrize("rows", [[1, 1, 1], [4, 1, 2], [130, 1, 40]])
def test_attention_in_a_graph(gpu, rows):
    """Captured; between replays the lengths, tables and queries change and other calls run."""
    c = Case(rows, [1500, 600, 900], 4, 1, 64, 16, "bf16", "bf16")
    seqs, (start, length) = seqs_of(c.pool, rows, c.lengths, max_len=1500)
    out = torch.zeros(c.n, c.heads * 64, dtype=torch.bfloat16, device="cuda:0")
    lse = torch.zeros(c.n, c.heads, device="cuda:0")
    pages = c.pool.pages()
    ws = torch.full((max(capi.kv_attention_workspace_size(pages, seqs, c.heads, 100, 4), 16),), 255, dtype=torch.uint8, device="cuda:0")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        capi.kv_attention(pages, seqs, c.buf.data_ptr(), capi.GG_TYPE_BF16, c.ld, c.heads, 0.125, 100, 4, out.data_ptr(), c.heads * 64,
                          lse.data_ptr(), ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for rep in range(4):
        c.buf.copy_(torch.randn(c.buf.numel()) * 2)
        lens = [1500 - 300 * rep, 600 - 100 * rep, 900 - 7 * rep]
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        eager, eager_lse = c.run(0.125, 100, 4, seqs=seqs)
        assert np.array_equal(out.double().cpu().numpy().reshape(eager.shape), eager)
        assert np.array_equal(lse.double().cpu().numpy(), eager_lse)


def test_two_calls_at_once(gpu):
    """Two streams, a workspace each."""
    cases = [Case([1] * 8, [2000 + 100 * i for i in range(8)], 4, 2, 128, 16, "bf16", "bf16", seed=i) for i in range(2)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    work = []
    for c in cases:
        seqs, keep = seqs_of(c.pool, c.rows, c.lengths)
        pages = c.pool.pages()
        work.append((c, pages, seqs, keep, torch.zeros(c.n, c.heads * 128, dtype=torch.bfloat16, device="cuda:0"),
                     torch.zeros(max(capi.kv_attention_workspace_size(pages, seqs, c.heads), 16), dtype=torch.uint8, device="cuda:0")))
    torch.cuda.synchronize()
    for _ in range(20):
        for (c, pages, seqs, keep, out, ws), s in zip(work, streams):
            capi.kv_attention(pages, seqs, c.buf.data_ptr(), capi.GG_TYPE_BF16, c.ld, c.heads, 128 ** -0.5, 0, 0, out.data_ptr(),
                              c.heads * 128, None, ws.data_ptr(), s.cuda_stream)
    torch.cuda.synchronize()
    for (c, *_, out, ws), (ref, _) in zip(work, want):
        assert np.array_equal(out.double().cpu().numpy().reshape(ref.shape), ref)


def test_long_sequence(gpu):
    """130000 positions, most of them in one page: many chunks and their join."""
    c = Case([1, 2], [130000, 90001], 2, 1, 64, 50000, "e4m3", "f32", spare=0)
    c.check()


def test_pool_past_32_bits(gpu):
    """Rows whose offset in the pool passes 2^32 elements."""
    d, n_kv, page = 256, 8, 1024
    n_pages = (1 << 32) // (page * n_kv * d) + 4
    k, v = (torch.zeros(n_pages * page * n_kv * d, dtype=torch.uint8, device="cuda:0") for _ in range(2))
    ks, vs = (torch.ones(n_pages, page, n_kv, device="cuda:0") for _ in range(2))
    pages = capi.kv_pages(k.data_ptr(), v.data_ptr(), capi.GG_TYPE_E4M3, n_pages, page, n_kv, d, k_scale=ks.data_ptr(), v_scale=vs.data_ptr())
    table = torch.tensor([[0, n_pages - 1]], dtype=torch.int32, device="cuda:0")
    for rows in (2, 60):
        far = v.view(n_pages, page, n_kv, d)[n_pages - 1]
        far[:100] = torch.randint(0, 0x70, (100, n_kv, d), dtype=torch.uint8, device="cuda:0")
        start, length = torch.tensor([0, rows], dtype=torch.int32, device="cuda:0"), torch.tensor([1124], dtype=torch.int32, device="cuda:0")
        seqs = capi.kv_seqs(start.data_ptr(), length.data_ptr(), table.data_ptr(), 1, rows, rows, 2048, 2)
        q, out = torch.randn(rows, n_kv * d, device="cuda:0"), torch.zeros(rows, n_kv * d, device="cuda:0")
        ws = torch.zeros(max(capi.kv_attention_workspace_size(pages, seqs, n_kv, 100, 0), 16), dtype=torch.uint8, device="cuda:0")
        capi.kv_attention(pages, seqs, q.data_ptr(), capi.GG_TYPE_F32, n_kv * d, n_kv, 1.0, 100, 0, out.data_ptr(), n_kv * d, None,
                          ws.data_ptr(), stream())
        torch.cuda.synchronize()
        # K is 0: equal weights; a row's window is the last 100 positions up to its own
        vals = torch.cat([torch.zeros(1024, n_kv, d, device="cuda:0", dtype=torch.float64), far[:100].view(torch.float8_e4m3fn).double()])
        ref = torch.stack([vals[1124 - rows + i - 99:1124 - rows + i + 1].mean(0) for i in range(rows)])
        # equal weights of 1: sums of 100 values and one division, all in f32
        assert ((out.view(rows, n_kv, d) - ref).abs() <= ref * 110 * 2.0 ** -24 + LEAST["f32"]).all()


@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("e4m3", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows", [[1] * 70, [2] * 40 + [300] + [0] * 5 + [1] * 40 + [70, 17], [0] * 30 + [130] * 3 + [0] * 70 + [5]])
def test_more_than_64_sequences(gpu, rows, cache, x):
    """Sequences found by search; long and short ones and such without rows in one call."""
    lengths = [n + 37 * i % 210 for i, n in enumerate(rows)]
    say("sequences", len(rows), sum(rows), cache, x)
    c = Case(rows, lengths, 4, 1, 64, 24, cache, x)
    c.check(every=7)
    c.check(window=50, sinks=3, every=13)


def test_thousands_of_sequences(gpu):
    rows = [i % 3 for i in range(4200)]
    c = Case(rows, [max(n, 1) + i % 5 for i, n in enumerate(rows)], 1, 1, 16, 4, "bf16", "bf16")
    c.check()


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("dim", [48, 112, 208, 240])
def test_odd_heads(gpu, dim, cache, x):
    """Heads between the kernels' widths, groups that no tile divides by: few rows, many, and both."""
    for rows in ([3, 1], [60, 8], [50, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1]):
        say("heads of", dim, cache, x, rows)
        Case(rows, [n + 333 for n in rows], 17, 1, dim, 10, cache, x).check(every=5)


@pytest.mark.parametrize("cache,x", KINDS)
@pytest.mark.parametrize("rows", [4, 150])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_queries_that_are_not_finite(gpu, rows, cache, x, bad):
    """One head of one row has a NaN or an infinity: no other row or head changes but within its bounds."""
    say("query", bad, rows, cache, x)
    c = Case([rows], [rows + 300], 3, 1, 64, 16, cache, x)
    r = rows // 2
    c.buf.view(-1, c.ld)[r, 5] = bad
    out, lse = c.run()
    for h in range(3):
        keep = np.array([i for i in range(rows) if (i, h) != (r, 0)])
        ro, rl, bo, bl = attention(c.q[keep, h], c.k[0][:, 0], c.v[0][:, 0], 300 + keep, np.float32(0.125).astype(np.float64), 0, 0, cache, x)
        assert (np.abs(out[keep, h] - ro) <= bo).all() and (np.abs(lse[keep, h] - rl) <= bl).all()
    if np.isnan(bad):
        assert np.isnan(out[r, 0]).all() and np.isnan(lse[r, 0])
