"""Verification of drafted tokens against a 64-bit plain form."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from kv_ref import TYPES, i32, typed, verify

pytestmark = pytest.mark.gpu


def run(z, y, draft, start, heat, u, v, name="f32", gap=0, offset=0, n_rows=None, logprobs=True):
    """-> accepted, tokens, logprobs and the kept logits"""
    rows, n = z.shape
    ld = n + gap

    def place(a):
        buf = torch.full((offset + rows * ld,), float("nan"), dtype=TYPES[name][1], device="cuda:0")
        t, kept = typed(a, name)
        buf[offset:].view(rows, ld)[:, :n] = t
        return buf, buf.data_ptr() + offset * buf.element_size(), kept
    zb, zp, z = place(z)
    yb, yp, y = place(y) if y is not None else (None, None, None)
    seqs = len(start) - 1
    dt, st = i32(draft), i32(start)
    ht = torch.tensor(np.asarray(heat, np.float32), device="cuda:0")
    ut, vt = (torch.tensor(np.asarray(a, np.float64), device="cuda:0") for a in (u, v))
    acc = torch.full((seqs,), 99, dtype=torch.int32, device="cuda:0")
    tok = torch.full((rows,), 99, dtype=torch.int32, device="cuda:0")
    lp = torch.full((rows,), 99.0, device="cuda:0")
    ws = torch.full((capi.verify_drafts_workspace_size(rows, seqs, n),), 255, dtype=torch.uint8, device="cuda:0")
    for _ in range(2):   # a workspace that holds the last call's results
        capi.verify_drafts(zp, yp, TYPES[name][0], rows, n, ld, ld, dt.data_ptr(), st.data_ptr(), seqs, ht.data_ptr(), ut.data_ptr(),
                           vt.data_ptr(), acc.data_ptr(), tok.data_ptr(), lp.data_ptr() if logprobs else None, ws.data_ptr(), stream())
    torch.cuda.synchronize()
    return acc.cpu().numpy(), tok.cpu().numpy(), lp.double().cpu().numpy(), z, y


def check(z, y, draft, start, heat, u, v, name="f32", margin=1e-9, **more):
    """Decisions whose 64-bit margin is below `margin` may fall either way; there are none in most cases."""
    acc, tok, lp, zk, yk = run(z, y, draft, start, heat, u, v, name, **more)
    ra, rt, rl, m = verify(zk, yk, draft, start, np.asarray(heat, np.float32), u, v)
    clear = m > margin
    # p(d) is compared with its sums in f32 exponentials, 2^-20 of it
    seq = np.repeat(np.arange(len(start) - 1), np.diff(start))
    assert np.array_equal(acc[clear], ra[clear]), (acc, ra)
    body, rows = tok[start[0]:start[-1]], clear[seq]
    assert np.array_equal(body[rows], rt[start[0]:start[-1]][rows])
    a, b = lp[start[0]:start[-1]][rows], rl[start[0]:start[-1]][rows]
    heat_of = np.where(np.asarray(heat) > 0, heat, 1.0)[seq][rows]
    with np.errstate(invalid="ignore"):
        # f32 exponentials of (z - m) / T: 2^-22 of their exponent, which is at most that where they count (40), and the result's rounding
        ok = np.abs(a - b) <= 40 * 2.0 ** -22 + 2.0 ** -22 * np.abs(b)
    assert (ok | (np.isnan(a) & np.isnan(b)) | (np.isneginf(a) & np.isneginf(b))).all()
    assert heat_of.min(initial=1) > 0
    return acc, tok, lp, clear


def sample(rng, counts, n, peak=True, agree=0.5):
    start = np.concatenate([[0], np.cumsum(np.asarray(counts) + 1)])
    rows = start[-1]
    z = rng.standard_normal((rows, n)) * 2
    if peak:
        at = rng.integers(0, n, (rows, 4))
        np.put_along_axis(z, at, np.take_along_axis(z, at, 1) + 6 * rng.random((rows, 4)), 1)
    y = z + rng.standard_normal((rows, n)) * agree
    draft = np.array([rng.choice(n, p=np.exp(r - r.max()) / np.exp(r - r.max()).sum()) for r in y])
    return z, y, draft, start, rng.random(rows), rng.random(len(counts))


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("with_y", [True, False])
@pytest.mark.parametrize("counts,n,gap,offset", [([0], 1, 0, 0), ([3], 2, 1, 1), ([2, 0, 5], 7, 0, 3), ([1, 4, 0, 3, 2], 255, 2, 0),
                                                 ([4, 4], 4096, 0, 0), ([3, 9], 4097, 3, 5), ([1, 2, 3, 0, 6], 50257, 0, 0),
                                                 ([4], 262144, 0, 0), ([1] * 70, 1000, 0, 0)])
def test_verify(gpu, counts, n, gap, offset, with_y, name):
    rng = np.random.default_rng(n + len(counts))
    say("verify", counts[:6], n, gap, offset, with_y, name)
    z, y, draft, start, u, v = sample(rng, counts, n)
    heat = rng.choice([0.0, 0.7, 1.0, 1.6], len(counts))
    check(z, y if with_y else None, draft, start, heat, u, v, name, gap=gap, offset=offset)


@pytest.mark.parametrize("with_y", [True, False])
def test_flat_rows(gpu, with_y):
    """Logits that are nearly alike over a whole vocabulary: borders 2^-18 apart, and draws at 0 and just below 1."""
    n, seqs = 262144, 16
    rng = np.random.default_rng(4)
    z, y, draft, start, u, v = sample(rng, [1] * seqs, n, peak=False, agree=1.0)
    z, y = z / 2, y / 2
    u[:] = 0.999999          # most drafts fall
    v[:4] = [0.0, np.nextafter(1.0, 0.0), 0.5, 1e-12]
    acc, tok, lp, clear = check(z, y if with_y else None, draft, start, np.ones(seqs), u, v, margin=1e-12)
    assert clear.sum() >= seqs - 4   # the three draws at an end of the axis are no further from a border than that
    _, rt, _, _ = verify(z.astype(np.float32).astype(np.float64), y.astype(np.float32).astype(np.float64) if with_y else None, draft, start,
                         np.ones(seqs), u, v)
    for s in (0, 1, 3):
        r = start[s] + acc[s]
        assert tok[r] == rt[r] or v[s] == v[1] and tok[r] > n - 10   # a draw of 0: the first id with any weight


def test_greedy(gpu):
    """Ties go to the lowest id; zeros of both signs are equal; the whole draft may stand."""
    n = 5000
    z = np.random.default_rng(1).standard_normal((12, n))
    z[0, [40, 4000]] = 9
    z[1, [7, 4999]] = 9
    z[2, 3] = 9
    z[3, 10] = 9
    z[4] = 0
    z[5] = -0.0
    z[5, 100:] = 0.0
    z[6] = 1
    z[7, n - 1] = 30
    draft = np.array([40, 7, 3, 0, 0, 0, 5, n - 1, n - 1, -1, n, 0])
    start = np.array([0, 4, 7, 9, 12])
    z[9], z[10] = z[0], z[0]
    acc, tok, lp, *_ = run(z, z * 0 + np.nan, draft, start, [0, 0, 0, 0], np.zeros(12), np.zeros(4))
    ra, rt, rl, _ = verify(z, None, draft, start, np.zeros(4), np.zeros(12), np.zeros(4))
    assert acc.tolist() == [3, 2, 1, 0] == ra.tolist()
    assert np.array_equal(tok, rt) and tok[:4].tolist() == [40, 7, 3, 10] and tok[6] == 0 and tok[9:].tolist() == [40, -1, -1]
    assert (np.abs(lp - rl) < 1e-5).all()


def test_masked_logits(gpu):
    """-inf and the type's lowest value; drafts of probability 0; nothing left of p when the draft is taken out."""
    n = 9000
    rng = np.random.default_rng(8)
    for name in ("f32", "bf16", "f16"):
        low = float(torch.finfo(TYPES[name][1]).min)
        z, y, draft, start, u, v = sample(rng, [2, 2, 1, 1, 3, 1], n)
        z[0, rng.random(n) < 0.9] = -np.inf
        z[1, :] = low
        z[1, 50] = 1.0
        z[3, draft[3]] = -np.inf              # probability 0: never stands
        y[4, draft[4]] = -np.inf              # not drawn from y at all: stands
        z[6, :] = -np.inf
        z[6, 77] = 3.0                        # one token: p = 1
        draft[6] = 77
        z[8, :] = -np.inf
        z[8, 5] = z[8, 8000] = 0.0
        draft[8], u[8] = 5, 0.75              # falls; 8000 is left
        z[13, :] = low
        y[13, :] = low
        for yy in (y, None):
            say("masked", name, yy is not None)
            check(z, yy, draft, start, [1, 0.8, 1, 1, 0.5, 1.0], u, v, name)


@pytest.mark.parametrize("with_y", [True, False])
def test_rows_without_a_distribution(gpu, with_y):
    n = 3000
    rng = np.random.default_rng(9)
    z, y, draft, start, u, v = sample(rng, [2] * 8, n)
    u[:] = 0.0                                # every draft that can stands
    z[0, 5] = np.nan
    z[4, 5] = np.inf
    z[8] = -np.inf
    y[9, 7] = np.nan
    y[13] = -np.inf
    y[17, 0] = np.nan                         # the last row of its sequence: not read
    z[18], z[19, 3] = np.nan, np.inf          # two in one sequence: the first ends it
    z[22, 0] = np.nan
    draft[21], u[21] = -1, 0.5                # falls before the bad row: not reached
    heat = [1, 1, 0, 1, 1, 1, 0, 1]
    acc, tok, lp, clear = check(z, y if with_y else None, draft, start, heat, u, v)
    assert clear.all()
    assert acc[0] == 0 and tok[:3].tolist() == [-1, -1, -1] and np.isnan(lp[0]) and (lp[1:3] == 0).all()
    assert acc[1] == 1 and tok[4] == -1 and tok[2 * 3 + 2] == -1 and tok[21] >= 0


def test_drafts_outside_the_vocabulary_and_empty_sequences(gpu):
    n = 600
    rng = np.random.default_rng(10)
    z, y, draft, start, u, v = sample(rng, [2, 2, 2], n)
    u[:] = 0
    draft[0], draft[4] = n, -7
    start = np.array([0, 3, 3, 6, 9, 9])
    for yy in (y, None):
        acc, tok, lp, *_ = run(z, yy, draft, start, [1, 1, 0.5, 1, 1], u, np.array([0.3, 0.3, 0.6, 0.9, 0.1]))
        ra, rt, rl, m = verify(z, yy, draft, start, [1, 1, 0.5, 1, 1], u, np.array([0.3, 0.3, 0.6, 0.9, 0.1]))
        assert (m > 1e-9).all() and np.array_equal(acc, ra) and np.array_equal(tok, rt)
        assert acc[1] == 0 and acc[4] == 0 and acc[0] == 0


def test_rows_behind_the_last_sequence(gpu):
    z, y, draft, start, u, v = sample(np.random.default_rng(11), [1, 1, 2], 400)
    acc, tok, lp, *_ = run(z, y, draft, start[:3], [1, 1], u, v[:2])
    assert (tok[4:] == 99).all() and (lp[4:] == 99).all()
    full = run(z, y, draft, start[:3], [1, 1], u, v[:2], logprobs=False)
    assert np.array_equal(full[1], tok) and (full[2] == 99).all()
    late = run(z, y, draft, start[1:], [1, 1], u, v[1:])     # rows before the first sequence
    assert (late[1][:2] == 99).all() and (late[1][2:] != 99).all()


def test_distribution_of_the_tokens(gpu):
    """Over 40000 sequences with one draft each, the first token is distributed as p: chi squared of 7 bins of freedom, below
    its 1 - 10^-9 quantile (57)."""
    n, seqs = 8, 40000
    rng = np.random.default_rng(12)
    z = np.tile(rng.standard_normal(n) * 1.5, (2 * seqs, 1))
    y = np.tile(rng.standard_normal(n) * 1.5, (2 * seqs, 1))
    q = np.exp(y[0]) / np.exp(y[0]).sum()
    p = np.exp(z[0]) / np.exp(z[0]).sum()
    draft = rng.choice(n, size=2 * seqs, p=q)
    start = np.arange(0, 2 * seqs + 1, 2)
    for yy, d in ((y, draft), (None, np.full(2 * seqs, 3))):
        acc, tok, *_ = run(z, yy, d, start, np.ones(seqs), rng.random(2 * seqs), rng.random(seqs))
        seen = np.bincount(tok[0::2], minlength=n)
        assert ((seen - seqs * p) ** 2 / (seqs * p)).sum() < 57
        bonus = tok[1::2][acc == 1]
        assert ((np.bincount(bonus, minlength=n) - len(bonus) * p) ** 2 / (len(bonus) * p)).sum() < 57


def test_verify_in_a_graph(gpu):
    n, counts = 30000, [3, 0, 5]
    rng = np.random.default_rng(13)
    z, y, draft, start, u, v = sample(rng, counts, n)
    rows, seqs = len(z), len(counts)
    zt, yt = (torch.zeros(rows, n, device="cuda:0") for _ in range(2))
    dt, st, ht = i32(draft), i32(start), torch.tensor([1.0, 0.0, 0.8], device="cuda:0")
    ut, vt = torch.zeros(rows, dtype=torch.float64, device="cuda:0"), torch.zeros(seqs, dtype=torch.float64, device="cuda:0")
    acc, tok = torch.zeros(seqs, dtype=torch.int32, device="cuda:0"), torch.zeros(rows, dtype=torch.int32, device="cuda:0")
    lp = torch.zeros(rows, device="cuda:0")
    ws = torch.full((capi.verify_drafts_workspace_size(rows, seqs, n),), 255, dtype=torch.uint8, device="cuda:0")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        capi.verify_drafts(zt.data_ptr(), yt.data_ptr(), capi.GG_TYPE_F32, rows, n, n, n, dt.data_ptr(), st.data_ptr(), seqs, ht.data_ptr(),
                           ut.data_ptr(), vt.data_ptr(), acc.data_ptr(), tok.data_ptr(), lp.data_ptr(), ws.data_ptr(),
                           torch.cuda.current_stream().cuda_stream)
    for rep in range(4):
        z, y, draft, start, u, v = sample(rng, counts, n)
        for t, a in ((zt, z), (yt, y), (dt, draft), (ut, u), (vt, v)):
            t.copy_(torch.from_numpy(np.asarray(a)))
        g.replay()
        torch.cuda.synchronize()
        ra, rt, rl, m = verify(zt.double().cpu().numpy(), yt.double().cpu().numpy(), draft, start, np.array([1.0, 0.0, np.float32(0.8)]), u, v)
        assert (m > 1e-9).all()
        assert np.array_equal(acc.cpu().numpy(), ra) and np.array_equal(tok.cpu().numpy(), rt)
        eager = run(zt.double().cpu().numpy(), yt.double().cpu().numpy(), draft, start, [1.0, 0.0, 0.8], u, v)
        assert np.array_equal(eager[2], lp.double().cpu().numpy())


def test_many_small_rows(gpu):
    """More parts than one grid's threads allow: 2^24 rows of two logits, half a million sequences."""
    rows, seqs = (1 << 24) + 32, (1 << 19) + 1
    each = 32
    z = torch.zeros(rows, 2, device="cuda:0")
    z[:, 1] = (torch.arange(rows, device="cuda:0") % 3 == 0) * 2.0 - 1.0     # id 1 is best in every third row
    start = (torch.arange(seqs + 1, device="cuda:0") * each).int()
    draft = torch.ones(rows, dtype=torch.int32, device="cuda:0")
    heat = torch.zeros(seqs, device="cuda:0")
    u, v = torch.zeros(rows, dtype=torch.float64, device="cuda:0"), torch.zeros(seqs, dtype=torch.float64, device="cuda:0")
    acc, tok = torch.full((seqs,), 9, dtype=torch.int32, device="cuda:0"), torch.full((rows,), 9, dtype=torch.int32, device="cuda:0")
    ws = torch.empty(capi.verify_drafts_workspace_size(rows, seqs, 2), dtype=torch.uint8, device="cuda:0")
    say("verify", rows, seqs)
    capi.verify_drafts(z.data_ptr(), None, capi.GG_TYPE_F32, rows, 2, 2, 2, draft.data_ptr(), start.data_ptr(), seqs, heat.data_ptr(),
                       u.data_ptr(), v.data_ptr(), acc.data_ptr(), tok.data_ptr(), None, ws.data_ptr(), stream())
    torch.cuda.synchronize()
    first = torch.arange(seqs, device="cuda:0") * each
    stands = first % 3 == 0
    assert torch.equal(acc, stands.int())
    body = tok.view(seqs, each)
    assert torch.equal(body[:, 0], stands.int())
    assert torch.equal(body[:, 1], torch.where(stands, 0, -1).int())
    assert (body[:, 2:] == -1).all()
