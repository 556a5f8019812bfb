"""MXFP4 quantisation, expansion and products against 64-bit plain forms."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from mx_ref import TYPES, product_bound, quantised

pytestmark = pytest.mark.gpu
MX = capi.GG_TYPE_MXFP4


def packed(n):
    """A buffer of n bytes whose old contents show: 0xff is NaN as a scale byte."""
    return torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda:0")


def rows_of(values, name, ld, offset=0):
    """A device buffer that holds the rows of `values` (numpy) `ld` elements apart, after `offset` elements."""
    t = TYPES[name][1]
    m, k = values.shape
    buf = torch.full((offset + m * ld,), 123.0, dtype=t, device="cuda:0")
    buf[offset:].view(m, ld)[:, :k] = torch.from_numpy(values).to("cuda:0").to(t)
    return buf, buf.data_ptr() + offset * buf.element_size(), buf[offset:].view(m, ld)[:, :k].double().cpu().numpy()


def pack(values, name="f32", ld=None, offset=0):
    m, k = values.shape
    buf, ptr, kept = rows_of(values, name, ld or k, offset)
    p = packed(capi.mxfp4_packed_size(m, k))
    capi.mxfp4_quantize(ptr, TYPES[name][0], m, k, ld or k, p.data_ptr(), stream())
    torch.cuda.synchronize()
    return p, kept


def unpack(p, m, k, ld=None, offset=0):
    out = torch.full((offset + m * (ld or k) + 4,), -7.0, device="cuda:0")
    capi.mxfp4_dequant(p.data_ptr(), out.data_ptr() + 4 * offset, m, k, ld or k, stream())
    torch.cuda.synchronize()
    return out.cpu().numpy()


def sample(rng, m, k):
    x = rng.standard_normal((m, k)) * np.where(rng.random(k) < 0.05, 20.0, 1.0)
    return x * np.exp2(rng.integers(-8, 9, (m, 1)).astype(np.float64))


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("m,k,ld,offset", [(1, 1, 1, 0), (1, 32, 32, 0), (3, 33, 33, 0), (32, 64, 64, 0), (33, 255, 259, 1),
                                           (31, 256, 256, 4), (65, 257, 260, 0), (7, 1152, 1152, 0), (40, 700, 704, 2)])
def test_round_trip(gpu, name, m, k, ld, offset):
    rng = np.random.default_rng(m * 1000 + k)
    say("round trip", name, m, k, ld, offset)
    p, kept = pack(sample(rng, m, k), name, ld, offset)
    got = unpack(p, m, k, ld, offset)
    body = got[offset:offset + m * ld].reshape(m, ld)
    assert np.array_equal(body[:, :k].astype(np.float64), quantised(kept))
    assert (got[:offset] == -7).all() and (got[offset + m * ld:] == -7).all() and (body[:, k:] == -7).all()


def test_every_border_and_magnitude(gpu):
    """Every midpoint and its neighbours, saturation, and blocks from the smallest f32 to the largest."""
    a = np.concatenate([np.arange(0, 8, 1 / 16), np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) + 2.0 ** -20,
                        np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) - 2.0 ** -20]).astype(np.float32)
    rows = []
    for v in a:
        row = np.zeros(32, np.float32)
        row[0], row[1], row[2] = 4.0 if v < 4 else v, v, -v
        rows.append(row)
    x = np.stack(rows)
    scaled = [x]
    for e in (-150, -149, -140, -128, -127, -126, -125, -60, 60, 120, 124, 125):
        with np.errstate(over="ignore", under="ignore"):
            y = (x.astype(np.float64) * 2.0 ** e).astype(np.float32)
        scaled.append(y[np.isfinite(y).all(1)])
    x = np.concatenate(scaled)
    say("borders", x.shape)
    p, kept = pack(x.astype(np.float64))
    assert np.array_equal(kept, x.astype(np.float64))
    assert np.array_equal(unpack(p, *x.shape)[:-4].reshape(x.shape).astype(np.float64), quantised(kept))


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_block_with_inf_or_nan(gpu, bad):
    x = np.random.default_rng(5).standard_normal((40, 100))
    x[3, 40] = bad
    x[39, 99] = bad
    p, kept = pack(x)
    got = unpack(p, 40, 100)[:-4].reshape(40, 100)
    want = quantised(kept)
    assert np.isnan(got[3, 32:64]).all() and np.isnan(got[39, 96:]).all() and np.isnan(got).sum() == 36
    assert np.array_equal(got.astype(np.float64), want, equal_nan=True)


def linear(wp, xptr, x_type, ldx, m, n, k, y_name, ldy=None, offset=0, ws=None):
    """y with a margin around and between its rows that must keep its values."""
    ldy = ldy or n
    y = torch.full((offset + m * ldy + 8,), 55.0, dtype=TYPES[y_name][1], device="cuda:0")
    if ws is None:
        ws = packed(capi.mxfp4_linear_workspace_size(x_type, m, n, k))
    capi.mxfp4_linear(wp.data_ptr(), xptr, x_type, ldx, y.data_ptr() + offset * y.element_size(), TYPES[y_name][0], ldy, m, n,
                      k, ws.data_ptr(), stream())
    torch.cuda.synchronize()
    y = y.double().cpu().numpy()
    body = y[offset:offset + m * ldy].reshape(m, ldy)
    assert (y[:offset] == 55).all() and (y[offset + m * ldy:] == 55).all() and (body[:, n:] == 55).all()
    return body[:, :n]


SHAPES = [(1, 1, 1), (1, 16, 32), (1, 17, 33), (2, 33, 100), (3, 64, 64), (3, 40, 700), (4, 100, 129), (5, 40, 300),
          (16, 65, 257), (17, 31, 1152), (31, 129, 65), (33, 130, 64), (64, 257, 520), (130, 300, 777), (1, 1536, 1152),
          (2, 1152, 6912), (260, 1000, 1152)]


@pytest.mark.parametrize("y_name", list(TYPES))
@pytest.mark.parametrize("x_name", list(TYPES) + ["mxfp4"])
def test_linear(gpu, x_name, y_name):
    for m, n, k in SHAPES:
        rng = np.random.default_rng(m * 7919 + n * 31 + k)
        say("linear", x_name, y_name, m, n, k)
        w = rng.standard_normal((n, k)) * 0.05
        x = sample(rng, m, k)
        if y_name == "f16":
            x = np.clip(x, -500, 500)
        wp, wk = pack(w)
        wq = quantised(wk)
        if x_name == "mxfp4":
            xp, xk = pack(x)
            xk = quantised(xk)
            got = linear(wp, xp.data_ptr(), MX, 0, m, n, k, y_name)
        else:
            buf, ptr, xk = rows_of(x, x_name, k)
            got = linear(wp, ptr, TYPES[x_name][0], k, m, n, k, y_name)
        want = xk @ wq.T
        err = np.abs(got - want) / product_bound(xk, wq, want, None if x_name == "mxfp4" else x_name, y_name)
        assert err.max() <= 1, (m, n, k, err.max())


@pytest.mark.parametrize("m,ldx,xoff,ldy,yoff", [(1, 515, 1, 301, 3), (3, 520, 0, 304, 0), (9, 515, 1, 301, 1), (70, 513, 3, 300, 2),
                                                 (70, 516, 4, 308, 4)])
@pytest.mark.parametrize("x_name,y_name", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16")])
def test_linear_strides_and_alignment(gpu, m, ldx, xoff, ldy, yoff, x_name, y_name):
    n, k = 300, 513
    rng = np.random.default_rng(m + ldx)
    say("linear strides", m, ldx, xoff, ldy, yoff, x_name, y_name)
    wp, wk = pack(rng.standard_normal((n, k)) * 0.1)
    buf, ptr, xk = rows_of(rng.standard_normal((m, k)), x_name, ldx, xoff)
    got = linear(wp, ptr, TYPES[x_name][0], ldx, m, n, k, y_name, ldy, yoff)
    wq = quantised(wk)
    want = xk @ wq.T
    assert (np.abs(got - want) <= product_bound(xk, wq, want, x_name, y_name)).all()


@pytest.mark.parametrize("m", [1, 3, 50])
def test_linear_infinities_and_nans_stay_in_their_rows(gpu, m):
    n, k = 70, 200
    rng = np.random.default_rng(m)
    w, x = rng.standard_normal((n, k)), rng.standard_normal((m, k))
    w[5, 33] = np.nan     # block 1 of weight row 5
    x[m - 1, 190] = np.inf
    wp, wk = pack(w)
    buf, ptr, xk = rows_of(x, "f32", k)
    got = linear(wp, ptr, capi.GG_TYPE_F32, k, m, n, k, "f32")
    nan = np.zeros((m, n), bool)
    nan[:, 5] = True
    nan[m - 1] = True
    assert np.array_equal(np.isnan(got), nan)
    xp, xk4 = pack(x)
    got4 = linear(wp, xp.data_ptr(), MX, 0, m, n, k, "f32")
    assert np.array_equal(np.isnan(got4), nan)
    wq = np.where(np.isnan(quantised(wk)), 0, quantised(wk))
    xk = np.where(np.isfinite(xk), xk, 0)
    want = xk @ wq.T
    assert (np.abs(got - want) <= product_bound(xk, wq, want, "f32", "f32"))[~nan].all()


@pytest.mark.parametrize("m", [2, 40])
@pytest.mark.parametrize("ex,ew", [(-130, 0), (-100, -20), (100, 20), (126, -10), (-149, 120)])
def test_linear_far_magnitudes(gpu, m, ex, ew):
    n, k = 40, 96
    rng = np.random.default_rng(3)
    x = (rng.uniform(-1.9, 1.9, (m, k)) * 2.0 ** ex).astype(np.float32).astype(np.float64)
    wp, wk = pack(rng.uniform(-1.9, 1.9, (n, k)) * 2.0 ** ew)
    buf, ptr, xk = rows_of(x, "f32", k)
    assert np.array_equal(xk, x)
    got = linear(wp, ptr, capi.GG_TYPE_F32, k, m, n, k, "f32")
    wq = quantised(wk)
    want = x @ wq.T
    # results and running sums below 2^-126 may lose their last bits
    assert (np.abs(got - want) <= product_bound(x, wq, want, "f32", "f32") + 2.0 ** -126).all()


def test_linear_offsets_past_32_bits(gpu):
    """The last rows of weights and of results whose byte offsets pass 2^32."""
    n, k, m = 1 << 20, 8192, 1
    gen = torch.Generator(device=gpu).manual_seed(1)
    p = packed(capi.mxfp4_packed_size(n, k))
    assert p.numel() > 1 << 32
    w = torch.randn(64, k, generator=gen, device=gpu)
    tile = packed(capi.mxfp4_packed_size(64, k))
    capi.mxfp4_quantize(w.data_ptr(), capi.GG_TYPE_F32, 64, k, k, tile.data_ptr(), stream())
    codes, scales = 64 // 32 * 128 * 1024, 64 // 32 * 32 * 256
    p[:n // 64 * codes].view(n // 64, codes)[:] = tile[:codes]
    p[n // 64 * codes:].view(n // 64, scales)[:] = tile[codes:codes + scales]
    say("far offsets")
    x = torch.randn(m, k, generator=gen, device=gpu)
    y = torch.zeros(m, n, device=gpu)
    capi.mxfp4_linear(p.data_ptr(), x.data_ptr(), capi.GG_TYPE_F32, k, y.data_ptr(), capi.GG_TYPE_F32, n, m, n, k, None, stream())
    torch.cuda.synchronize()
    assert torch.equal(y.view(n // 64, 64), y[0, :64].expand(n // 64, 64))
    wq, xk = quantised(w.double().cpu().numpy()), x.double().cpu().numpy()
    want = xk @ wq.T
    assert (np.abs(y[:, :64].double().cpu().numpy() - want) <= product_bound(xk, wq, want, "f32", "f32")).all()


def test_linear_in_a_graph_and_on_another_stream(gpu):
    """Captured once, replayed with new inputs and eager calls between, each with a workspace of its own."""
    n, k = 200, 640
    rng = np.random.default_rng(9)
    wp, wk = pack(rng.standard_normal((n, k)) * 0.1)
    wq = quantised(wk)
    for m in (1, 37):
        say("graph", m)
        x = torch.zeros(m, k, device=gpu)
        xp = packed(capi.mxfp4_packed_size(m, k))
        ya, yb = torch.zeros(m, n, device=gpu), torch.zeros(m, n, device=gpu)
        ws = packed(capi.mxfp4_linear_workspace_size(capi.GG_TYPE_F32, m, n, k))
        s = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cs = torch.cuda.current_stream().cuda_stream
            capi.mxfp4_linear(wp.data_ptr(), x.data_ptr(), capi.GG_TYPE_F32, k, ya.data_ptr(), capi.GG_TYPE_F32, n, m, n, k,
                              ws.data_ptr(), cs)
            capi.mxfp4_quantize(x.data_ptr(), capi.GG_TYPE_F32, m, k, k, xp.data_ptr(), cs)
            capi.mxfp4_linear(wp.data_ptr(), xp.data_ptr(), MX, 0, yb.data_ptr(), capi.GG_TYPE_F32, n, m, n, k, None, cs)
        for rep in range(4):
            xv = rng.standard_normal((m, k))
            x.copy_(torch.from_numpy(xv))
            g.replay()
            torch.cuda.synchronize()
            xk = x.double().cpu().numpy()
            want = xk @ wq.T
            assert (np.abs(ya.double().cpu().numpy() - want) <= product_bound(xk, wq, want, "f32", "f32")).all()
            eager = torch.from_numpy(linear(wp, x.data_ptr(), capi.GG_TYPE_F32, k, m, n, k, "f32"))
            assert torch.equal(eager.float(), ya.cpu())
            eager = torch.from_numpy(linear(wp, xp.data_ptr(), MX, 0, m, n, k, "f32"))
            assert torch.equal(eager.float(), yb.cpu())


@pytest.mark.parametrize("m", [1, 5, 100])
def test_linear_repeats_bit_for_bit(gpu, m):
    n, k = 1000, 2048
    rng = np.random.default_rng(2)
    wp, _ = pack(rng.standard_normal((n, k)))
    buf, ptr, _ = rows_of(rng.standard_normal((m, k)), "f32", k)
    first = linear(wp, ptr, capi.GG_TYPE_F32, k, m, n, k, "f32")
    for _ in range(3):
        assert np.array_equal(first, linear(wp, ptr, capi.GG_TYPE_F32, k, m, n, k, "f32"))


@pytest.mark.parametrize("x_name", ["f32", "f16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(12, 100, 16400), (40, 96, 8200), (70, 200, 5000), (300, 260, 3100)])
def test_linear_long_k(gpu, x_name, m, n, k):
    """Many stages of each tile, with and without slices of k."""
    say("long k", x_name, m, n, k)
    rng = np.random.default_rng(k + m)
    x = sample(rng, m, k)
    wp, wk = pack(rng.standard_normal((n, k)) * 0.05)
    wq = quantised(wk)
    if x_name == "mxfp4":
        xp, xk = pack(x)
        xk = quantised(xk)
        got = linear(wp, xp.data_ptr(), MX, 0, m, n, k, "f32")
    else:
        buf, ptr, xk = rows_of(np.clip(x, -500, 500), x_name, k)
        got = linear(wp, ptr, TYPES[x_name][0], k, m, n, k, "f32")
    want = xk @ wq.T
    assert (np.abs(got - want) <= product_bound(xk, wq, want, None if x_name == "mxfp4" else x_name, "f32")).all()


def test_round_trip_of_many_rows(gpu):
    """More rows than one grid's threads allow: 2^28 and a few, of one element."""
    rows = (1 << 28) + 70
    say("round trip", rows)
    src = (torch.arange(rows, dtype=torch.int32, device="cuda:0") % 13).to(torch.bfloat16)
    p = torch.empty(capi.mxfp4_packed_size(rows, 1), dtype=torch.uint8, device="cuda:0")
    out = torch.empty(rows, device="cuda:0")
    capi.mxfp4_quantize(src.data_ptr(), capi.GG_TYPE_BF16, rows, 1, 1, p.data_ptr(), stream())
    capi.mxfp4_dequant(p.data_ptr(), out.data_ptr(), rows, 1, 1, stream())
    kept = torch.from_numpy(quantised(np.arange(13.0)[:, None])[:, 0]).to("cuda:0", torch.float32)
    for lo in range(0, rows, 1 << 26):
        part = out[lo:lo + (1 << 26)]
        assert torch.equal(part, kept[src[lo:lo + (1 << 26)].long()])


@pytest.mark.parametrize("x_name,y_name", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("mxfp4", "f32")])
def test_linear_large(gpu, x_name, y_name):
    """Sizes of the largest blocks, ragged at each edge; rows of the first, inner and last blocks are checked."""
    m, n, k = 2500, 8300, 6020
    say("large", x_name, y_name)
    rng = np.random.default_rng(77)
    wp, _ = pack(rng.standard_normal((n, k)) * 0.02)
    w = unpack(wp, n, k)[:-4].reshape(n, k).astype(np.float64)
    x = np.clip(sample(rng, m, k), -200, 200)
    pick = np.r_[0:24, 244:268, 1500:1510, m - 40:m]
    if x_name == "mxfp4":
        xp, xk = pack(x)
        xk = quantised(xk[pick])
        got = linear(wp, xp.data_ptr(), MX, 0, m, n, k, y_name)
    else:
        buf, ptr, xk = rows_of(x, x_name, k)
        xk = xk[pick]
        got = linear(wp, ptr, TYPES[x_name][0], k, m, n, k, y_name)
    want = xk @ w.T
    assert (np.abs(got[pick] - want) <= product_bound(xk, w, want, None if x_name == "mxfp4" else x_name, y_name)).all()
