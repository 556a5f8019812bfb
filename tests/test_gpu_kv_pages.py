"""Rows into K/V pages and back: norm, rotation, 16 and 8 bits, against 64-bit plain forms."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from kv_ref import HALF_STEP, LEAST, Pool, TYPES, e4m3_row, norm_rope, seqs_of, typed

pytestmark = pytest.mark.gpu
EPS, THETA = 1e-6, 1e6


def close(got, ref, name):
    """Rounded once from a value that is off by 2^-36 of the row's size at most, on both sides together: an f64 angle below
    2^15 is a power and a product, off by 2^15 2^-52."""
    ref = np.asarray(ref, np.float64)
    slack = 2.0 ** -36 * np.abs(ref).max(-1, keepdims=True)
    assert (np.abs(np.asarray(got, np.float64) - ref) <= np.abs(ref) * HALF_STEP[name] + LEAST[name] + slack).all()


def store(pool, seqs, x, name, n_q, ld, offset, qw, kw, theta, q_name, q_gap=0):
    """x [rows, heads, d] -> (q_out, x as kept)"""
    rows, heads, d = x.shape
    buf = torch.full((offset + rows * ld,), 77.0, dtype=TYPES[name][1], device="cuda:0")
    t, kept = typed(x.reshape(rows, -1), name)
    buf[offset:].view(rows, ld)[:, :heads * d] = t
    ptr, es = buf.data_ptr() + offset * buf.element_size(), buf.element_size()
    n_kv = (heads - n_q) // 2
    ldq = n_q * d + q_gap
    q_out = torch.full((rows, max(ldq, 1)), -5.0, dtype=TYPES[q_name][1], device="cuda:0")
    w = [None if a is None else torch.from_numpy(a.astype(np.float32)).cuda() for a in (qw, kw)]
    capi.kv_store(pool.pages(), seqs, TYPES[name][0], ptr if n_q else None, ld, ptr + n_q * d * es, ld, ptr + (n_q + n_kv) * d * es, ld, n_q,
                  None if w[0] is None else w[0].data_ptr(), None if w[1] is None else w[1].data_ptr(), EPS, theta,
                  q_out.data_ptr() if n_q else None, TYPES[q_name][0], ldq, stream())
    torch.cuda.synchronize()
    return q_out.double().cpu().numpy(), kept.reshape(rows, heads, d)


def load(pool, seqs, rows, name="f32", gap=0):
    ld = pool.n_kv * pool.dim + gap
    k, v = (torch.full((rows, ld), -5.0, dtype=TYPES[name][1], device="cuda:0") for _ in range(2))
    capi.kv_load(pool.pages(), seqs, k.data_ptr(), ld, v.data_ptr(), ld, TYPES[name][0], stream())
    torch.cuda.synchronize()
    return k.double().cpu().numpy(), v.double().cpu().numpy()


CASES = [
    # rows, lengths, page, n_q, n_kv, dim, layout, ld gap, offset
    ([1], [1], 16, 4, 1, 256, "phd", 0, 0),
    ([1], [32767], 64, 4, 1, 256, "phd", 0, 0),
    ([5, 1, 0, 9], [5, 17, 3, 1000], 16, 3, 3, 64, "hpd", 3, 1),
    ([7, 2], [30, 2], 1, 8, 2, 128, "both", 4, 4),
    ([33, 20], [33, 90], 24, 6, 2, 80, "pad", 1, 3),
    ([600], [700], 100, 2, 1, 16, "phd", 0, 0),
    ([40, 1], [40, 77], 1000, 0, 4, 192, "pad", 8, 8),
    ([70] * 70, [75 + i for i in range(70)], 16, 1, 1, 32, "phd", 0, 0),
]


@pytest.mark.parametrize("name,q_name,cache", [("f32", "f32", "bf16"), ("bf16", "bf16", "e4m3"), ("f16", "f32", "f16"), ("f32", "bf16", "e4m3"),
                                               ("f16", "f16", "bf16")])
@pytest.mark.parametrize("rows,lengths,page,n_q,n_kv,dim,layout,gap,offset", CASES)
def test_store_and_load(gpu, rows, lengths, page, n_q, n_kv, dim, layout, gap, offset, name, q_name, cache):
    rng = np.random.default_rng(sum(lengths) + dim)
    say("store", name, q_name, cache, rows[:4], lengths[:4], page, n_q, n_kv, dim, layout)
    pool = Pool(lengths, page, n_kv, dim, cache, seed=1, layout=layout)
    seqs, keep = seqs_of(pool, rows, lengths)
    n, heads = sum(rows), n_q + 2 * n_kv
    x = rng.standard_normal((n, heads, dim)) * np.exp2(rng.integers(-6, 7, (n, heads, 1)).astype(np.float64))
    qw, kw = rng.random(dim) + 0.5, rng.random(dim) + 0.5
    q_out, kept = store(pool, seqs, x, name, n_q, heads * dim + gap, offset, qw, kw, THETA, q_name, q_gap=gap)
    pos = np.concatenate([np.arange(b - a, b) for a, b in zip(rows, lengths)])
    qw, kw = qw.astype(np.float32).astype(np.float64), kw.astype(np.float32).astype(np.float64)
    if n_q:
        close(q_out[:, :n_q * dim].reshape(n, n_q, dim), norm_rope(kept[:, :n_q], qw, pos, EPS, THETA), q_name)
        assert (q_out[:, n_q * dim:] == -5).all()
    k, v = norm_rope(kept[:, n_q:n_q + n_kv], kw, pos, EPS, THETA), kept[:, n_q + n_kv:]
    gk, gv = (t[:, :n_kv * dim].reshape(n, n_kv, dim) for t in load(pool, seqs, n, gap=3))
    if cache == "e4m3":
        assert np.array_equal(gk, e4m3_row(k)) and np.array_equal(gv, e4m3_row(v))
    else:
        close(gk, k, cache)
        close(gv, v, cache)
    # only the rows' places were written
    written = sum(rows) * n_kv
    for view in pool.views():
        empty = (view.view(torch.uint8) == 255) if cache == "e4m3" else torch.isnan(view)
        assert int((~empty.all(-1)).sum()) == written
    # what was stored comes back in other types, rounded once
    for other in ("bf16", "f16"):
        ok, ov = load(pool, seqs, n, other)
        ref = torch.from_numpy(gk.reshape(n, -1)).float().to(TYPES[other][1]).double().numpy()
        assert np.array_equal(ok, ref)


@pytest.mark.parametrize("theta,norm", [(0.0, True), (1e4, False), (0.0, False)])
def test_store_without_norm_or_rotation(gpu, theta, norm):
    rng = np.random.default_rng(5)
    pool = Pool([50, 9], 16, 2, 96, "bf16")
    seqs, keep = seqs_of(pool, [20, 9], [50, 9])
    x = rng.standard_normal((29, 6 + 4, 96))
    w = (rng.random(96) + 0.5).astype(np.float32).astype(np.float64) if norm else None
    q_out, kept = store(pool, seqs, x, "f32", 6, 960, 0, w, w, theta, "f32")
    pos = np.concatenate([np.arange(30, 50), np.arange(9)])
    close(q_out.reshape(29, 6, 96), norm_rope(kept[:, :6], w, pos, EPS, theta), "f32")
    gk, gv = load(pool, seqs, 29)
    close(gk.reshape(29, 2, 96), norm_rope(kept[:, 6:8], w, pos, EPS, theta), "bf16")
    close(gv.reshape(29, 2, 96), kept[:, 8:], "bf16")


def test_values_next_to_a_border(gpu):
    """Ties of every type, the largest magnitudes of an 8-bit row on both sides of 448 2^e, subnormal and huge rows, zeros, infinities."""
    d = 32
    base = np.zeros((12, d))
    base[0, :8] = [448, 1.0625, 1.1875, 2 ** -9 * 0.5, 2 ** -9 * 1.5, 2 ** -9 * 0.500001, -1.0625, 3.25]
    base[1, 0], base[1, 1] = np.nextafter(np.float32(448), np.float32(500)), 100   # just above: the next scale
    base[2, 0] = 449
    base[3] = 0
    base[4, 0], base[4, 1] = 2.0 ** -140, 2.0 ** -149
    base[5, 0], base[5, 1] = 3e38, 1
    base[6, 0] = np.inf
    base[7, 3] = np.nan
    base[8, :3] = [2.0 ** -126, 2.0 ** -120, -(2.0 ** -130)]
    base[9, 0], base[9, 1] = 1.75, 1.75 * (1 + 2.0 ** -23)
    base[10] = np.linspace(-448, 448, d)
    base[11] = 1.0
    for cache in ("e4m3", "bf16", "f16"):
        pool = Pool([12], 5, 1, d, cache)
        seqs, keep = seqs_of(pool, [12], [12])
        x = np.stack([base, base], 1)
        _, kept = store(pool, seqs, x, "f32", 0, 2 * d, 0, None, None, 0.0, "f32")
        gk, gv = load(pool, seqs, 12)
        rows = [i for i in range(12) if i not in (6, 7)]
        if cache == "e4m3":
            ref = e4m3_row(kept[rows, 0])
            assert np.isnan(gk[[6, 7]]).all() and np.isnan(gv[[6, 7]]).all()
            assert np.array_equal(gk[rows], ref) and np.array_equal(gv[rows], ref)
        else:
            ref = torch.from_numpy(kept[:, 0]).float().to(TYPES[cache][1]).double().numpy()
            assert np.array_equal(gk, ref, equal_nan=True) and np.array_equal(gv, ref, equal_nan=True)


def test_rounding_once_from_64_bits(gpu):
    """Norms that land a value next to a tie: rounding to f32 first would give the other neighbour."""
    d, n = 64, 4096
    rng = np.random.default_rng(2)
    x = rng.standard_normal((n, 2, d))
    w = np.ones(d)
    for cache in ("bf16", "f16"):
        pool = Pool([n], 64, 1, d, cache)
        seqs, keep = seqs_of(pool, [n], [n])
        _, kept = store(pool, seqs, x, "f32", 0, 2 * d, 0, None, w, 0.0, "f32")
        k = norm_rope(kept[:, :1], w, np.arange(n), EPS, 0.0)[:, 0]
        got, _ = load(pool, seqs, n)
        m, e = np.frexp(k)
        bits = 8 if cache == "bf16" else 11
        scaled = np.ldexp(m, bits)
        lands = np.where(np.abs(scaled - np.floor(scaled) - 0.5) < 2.0 ** -36, np.nan, np.ldexp(np.round(scaled), e - bits))
        same = (got == lands) | np.isnan(lands) | (e < -12)
        assert same.all()


def test_rows_without_a_place(gpu):
    """Positions below zero, unmapped and foreign pages, lengths past max_len, rows outside of all sequences."""
    d, n_kv = 64, 2
    pool = Pool([40, 40, 40], 8, n_kv, d, "bf16")
    pool.table[1, 4] = -1
    pool.table[2, 4] = pool.n_pages
    pool.table_dev.copy_(torch.from_numpy(pool.table))
    rows = [6, 12, 12]
    seqs, keep = seqs_of(pool, rows, [4, 40, 40], n_rows=2 + 30 + 5, max_len=38, first=2)   # len 40 counts as 38
    n = 37
    x = np.random.default_rng(3).standard_normal((n, 1 + 2 * n_kv, d))
    q_out, kept = store(pool, seqs, x, "bf16", 1, 5 * d, 0, None, None, 0.0, "f32")
    assert (q_out[:2] == -5).all() and (q_out[32:] == -5).all()
    assert np.array_equal(q_out[2:32], kept[2:32, 0])
    pos = np.concatenate([np.arange(-2, 4), np.arange(26, 38), np.arange(26, 38)])
    seq = np.repeat([0, 1, 2], rows)
    placed = (pos >= 0) & ~((seq > 0) & (pos // 8 == 4))
    gk, gv = load(pool, seqs, n)
    ref = np.where(placed[:, None], kept[2:32, 1:3].reshape(30, -1), 0.0)
    assert np.array_equal(gk[2:32], ref)
    assert np.array_equal(gv[2:32], np.where(placed[:, None], kept[2:32, 3:].reshape(30, -1), 0.0))
    assert (gk[:2] == -5).all() and (gv[32:] == -5).all()
    assert sum(int((~torch.isnan(v).all(-1)).sum()) for v in pool.views()) == 2 * int(placed.sum()) * n_kv


def test_store_in_a_graph(gpu):
    """A captured store follows the device's lengths and tables; its pool is used by eager calls in between."""
    pool = Pool([64, 64], 16, 1, 128, "e4m3")
    seqs, (start, length) = seqs_of(pool, [1, 1], [10, 20], max_len=64)
    x = torch.zeros(2, 6 * 128, dtype=torch.bfloat16, device="cuda:0")
    q_out = torch.zeros(2, 4 * 128, dtype=torch.bfloat16, device="cuda:0")
    w = torch.ones(128, device="cuda:0")
    k, v = (torch.zeros(2, 128, device="cuda:0") for _ in range(2))

    def call(s):
        capi.kv_store(pool.pages(), seqs, capi.GG_TYPE_BF16, x.data_ptr(), 768, x.data_ptr() + 1024, 768, x.data_ptr() + 1280, 768, 4,
                      w.data_ptr(), w.data_ptr(), EPS, THETA, q_out.data_ptr(), capi.GG_TYPE_BF16, 512, s)
        capi.kv_load(pool.pages(), seqs, k.data_ptr(), 128, v.data_ptr(), 128, capi.GG_TYPE_F32, s)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        call(torch.cuda.current_stream().cuda_stream)
    for rep in range(4):
        x.copy_(torch.randn(2, 768))
        length.add_(rep)
        g.replay()
        torch.cuda.synchronize()
        kept = x.double().cpu().numpy().reshape(2, 6, 128)
        pos = length.cpu().numpy() - 1
        close(q_out.double().cpu().numpy().reshape(2, 4, 128), norm_rope(kept[:, :4], np.ones(128), pos, EPS, THETA), "bf16")
        ref_k, ref_v = e4m3_row(norm_rope(kept[:, 4:5], np.ones(128), pos, EPS, THETA))[:, 0], e4m3_row(kept[:, 5:])[:, 0]
        assert np.array_equal(k.cpu().numpy(), ref_k) and np.array_equal(v.cpu().numpy(), ref_v)
        before = k.clone()
        call(stream())
        torch.cuda.synchronize()
        assert torch.equal(before, k)


def test_offsets_past_32_bits(gpu):
    """A pool of more than 2^32 elements: rows in its first and last pages."""
    d, n_kv, page = 256, 8, 1024
    n_pages = (1 << 32) // (page * n_kv * d) + 4
    k, v = (torch.zeros(n_pages * page * n_kv * d, dtype=torch.uint8, device="cuda:0") for _ in range(2))
    ks, vs = (torch.zeros(n_pages, page, n_kv, device="cuda:0") for _ in range(2))
    pages = capi.kv_pages(k.data_ptr(), v.data_ptr(), capi.GG_TYPE_E4M3, n_pages, page, n_kv, d, k_scale=ks.data_ptr(), v_scale=vs.data_ptr())
    table = torch.tensor([[0, n_pages - 1]], dtype=torch.int32, device="cuda:0")
    start, length = torch.tensor([0, 4], dtype=torch.int32, device="cuda:0"), torch.tensor([1026], dtype=torch.int32, device="cuda:0")
    seqs = capi.kv_seqs(start.data_ptr(), length.data_ptr(), table.data_ptr(), 1, 4, 4, 2048, 2)
    x = torch.randn(4, 2 * n_kv * d, device="cuda:0")
    capi.kv_store(pages, seqs, capi.GG_TYPE_F32, None, 0, x.data_ptr(), 2 * n_kv * d, x.data_ptr() + 4 * n_kv * d, 2 * n_kv * d, 0, None, None,
                  0.0, 0.0, None, 0, 0, stream())
    ko, vo = (torch.empty(4, n_kv * d, device="cuda:0") for _ in range(2))
    capi.kv_load(pages, seqs, ko.data_ptr(), n_kv * d, vo.data_ptr(), n_kv * d, capi.GG_TYPE_F32, stream())
    torch.cuda.synchronize()
    ref = e4m3_row(x.double().cpu().numpy().reshape(4, 2, n_kv, d))
    assert np.array_equal(ko.double().cpu().numpy().reshape(4, n_kv, d), ref[:, 0])
    assert np.array_equal(vo.double().cpu().numpy().reshape(4, n_kv, d), ref[:, 1])
    assert int((ks.view(-1, n_kv)[[1022, 1023]] != 0).sum()) == 16 and int((ks[-1, :2] != 0).sum()) == 16
    assert int((ks != 0).sum()) == 32
