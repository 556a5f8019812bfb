"""Log probabilities, entropy and best alternatives of rows of logits against
64-bit plain forms; the chain hidden rows -> 4-bit LM head -> scores."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from mx_ref import TYPES, score_rel, scores

pytestmark = pytest.mark.gpu


def run(z, name, ids=None, top=0, ld=None, offset=0):
    """z: numpy [rows, n] -> the values kept in the type, and the outputs."""
    rows, n = z.shape
    ld = ld or n
    t = TYPES[name][1]
    buf = torch.full((offset + rows * ld,), 300.0, dtype=t, device="cuda:0")   # what lies between the rows would win
    view = buf[offset:].view(rows, ld)[:, :n]
    view[:] = torch.from_numpy(z).to("cuda:0").to(t)
    out = {"lse": torch.full((rows,), 9.0, device="cuda:0"), "entropy": torch.full((rows,), 9.0, device="cuda:0")}
    ni = 0 if ids is None else ids.shape[1]
    idt = None if ids is None else torch.from_numpy(np.ascontiguousarray(ids, np.int32)).to("cuda:0")
    out["lp"] = torch.full((rows, max(ni, 1)), 9.0, device="cuda:0")
    out["top_ids"] = torch.full((rows, max(top, 1)), 77, dtype=torch.int32, device="cuda:0")
    out["top_lp"] = torch.full((rows, max(top, 1)), 9.0, device="cuda:0")
    ws = torch.full((max(capi.score_workspace_size(rows, n, top), 16),), 255, dtype=torch.uint8, device="cuda:0")
    capi.score_logits(buf.data_ptr() + offset * buf.element_size(), TYPES[name][0], rows, n, ld,
                      None if idt is None else idt.data_ptr(), ni, out["lp"].data_ptr(), out["lse"].data_ptr(),
                      out["entropy"].data_ptr(), top, out["top_ids"].data_ptr(), out["top_lp"].data_ptr(), ws.data_ptr(), stream())
    torch.cuda.synchronize()
    return view.double().cpu().numpy(), {k: v.cpu().numpy().astype(np.float64) for k, v in out.items()}


def check(z, got, ids, top):
    n = z.shape[1]
    lse, ent, lp, order = scores(z, top)
    rel = score_rel(n)
    m = np.abs(z.max(1))
    assert (np.abs(got["lse"] - lse) <= rel + 2.0 ** -23 * (np.abs(lse) + m)).all()
    # ln S and W / S each carry the sums' error, W / S relative to itself
    assert (np.abs(got["entropy"] - ent) <= rel * (2 + 2 * np.log(n)) + 2.0 ** -22 * np.log(n)).all()

    def tol(ref):
        return rel + 2.0 ** -22 * (1 + np.log(n)) + 2.0 ** -23 * np.abs(ref)
    if ids is not None:
        ref = np.take_along_axis(lp, ids, 1)
        ok = np.isneginf(ref) & np.isneginf(got["lp"])
        with np.errstate(invalid="ignore"):
            assert (ok | (np.abs(got["lp"] - ref) <= tol(ref))).all()
    if top:
        vals = np.take_along_axis(z, order, 1)
        have = ~np.isneginf(vals)
        assert np.array_equal(got["top_ids"][:, :order.shape[1]], np.where(have, order, -1))
        assert (got["top_ids"][:, order.shape[1]:] == -1).all() and np.isneginf(got["top_lp"][:, order.shape[1]:]).all()
        ref = np.take_along_axis(lp, order, 1)
        with np.errstate(invalid="ignore"):
            assert np.where(have, np.abs(got["top_lp"][:, :order.shape[1]] - ref) <= tol(ref),
                            np.isneginf(got["top_lp"][:, :order.shape[1]])).all()


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("rows,n,top,ld,offset", [(1, 1, 1, 1, 0), (2, 2, 5, 3, 1), (3, 7, 7, 7, 0), (5, 255, 20, 257, 3),
                                                  (1, 8191, 20, 8191, 1), (2, 8192, 64, 8192, 0), (3, 8193, 1, 8200, 7),
                                                  (1, 262144, 20, 262144, 0), (7, 50257, 5, 50257, 0), (1100, 1000, 3, 1001, 2),
                                                  (2, 300001, 64, 300001, 1)])
def test_score(gpu, name, rows, n, top, ld, offset):
    rng = np.random.default_rng(rows * 13 + n)
    say("score", name, rows, n, top, ld, offset)
    z = rng.standard_normal((rows, n)) * 3
    ids = rng.integers(0, n, (rows, 3))
    kept, got = run(z, name, ids, top, ld, offset)
    check(kept, got, ids, top)


@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "few values", "last tile best", "zeros of both signs"])
@pytest.mark.parametrize("n,top", [(5000, 20), (40000, 64), (262144, 20)])
def test_ties_and_orders(gpu, kind, n, top):
    """Rows on which many elements pass the running threshold."""
    rng = np.random.default_rng(n)
    z = {"equal": np.full(n, 1.5), "ascending": np.arange(n) / 1024.0, "descending": -np.arange(n) / 1024.0,
         "few values": rng.integers(0, 3, n).astype(np.float64), "last tile best": np.where(np.arange(n) >= n - 4000, 5.0, 0.0),
         "zeros of both signs": np.where(rng.random(n) < 0.5, 0.0, -0.0)}[kind]
    say("ties", kind, n, top)
    z = np.stack([z, z[::-1]])
    ids = np.array([[0, n - 1], [n // 2, 1]])
    kept, got = run(z, "f32", ids, top)
    check(kept, got, ids, top)


@pytest.mark.parametrize("n", [9, 5000, 100000])
@pytest.mark.parametrize("name", list(TYPES))
def test_masks(gpu, n, name):
    """-inf, the type's lowest value, rows with one or no value left."""
    rng = np.random.default_rng(n)
    low = float(torch.finfo(TYPES[name][1]).min)
    z = rng.standard_normal((6, n))
    z[0, rng.random(n) < 0.9] = -np.inf
    z[0, 3] = 1.0
    z[1, :] = -np.inf
    z[1, n // 2] = -4.0                       # one value: probability 1
    z[2, rng.random(n) < 0.9] = low
    z[2, 5] = 2.0
    z[3, :] = low                             # all equal and finite: uniform
    z[4, : n - 1] = -np.inf
    z[4, n - 1] = low
    ids = np.stack([[3, n // 2]] * 6)
    keep = [0, 1, 2, 4, 5]
    say("masks", name, n)
    kept, got = run(z, name, ids, 8)
    check(kept[keep], {k: v[keep] for k, v in got.items()}, ids[keep], 8)
    assert np.allclose(got["entropy"][3], np.log(n), rtol=1e-5)
    assert np.allclose(got["lp"][3], -np.log(n), rtol=1e-5) and np.array_equal(got["top_ids"][3], np.arange(8))


@pytest.mark.parametrize("n", [10, 20000])
def test_empty_rows_nans_infinities_and_given_ids(gpu, n):
    z = np.random.default_rng(1).standard_normal((5, n))
    z[0] = -np.inf
    z[1, 4] = np.nan
    z[2, 6] = np.inf
    z[3] = np.nan
    ids = np.array([[0, -1, 2, 3]] * 4 + [[-1, -2, n, 0]])
    kept, got = run(z, "f32", ids, 3)
    assert np.isneginf(got["lse"][0]) and got["entropy"][0] == 0
    assert np.isneginf(got["lp"][0, [0, 2, 3]]).all() and got["lp"][0, 1] == 0
    assert (got["top_ids"][0] == -1).all() and np.isneginf(got["top_lp"][0]).all()
    for r in (1, 2, 3):
        assert np.isnan(got["lse"][r]) and np.isnan(got["entropy"][r])
        assert np.isnan(got["lp"][r, [0, 2, 3]]).all() and got["lp"][r, 1] == 0
    assert 4 not in got["top_ids"][1] and got["top_ids"][2, 0] == 6 and (got["top_ids"][3] == -1).all()
    assert got["lp"][4, 0] == 0 and np.isnan(got["lp"][4, [1, 2]]).all()
    assert abs(got["lp"][4, 3] - scores(kept[4:], 0)[2][0, 0]) < 1e-5


def test_outputs_may_be_left_out(gpu):
    z = torch.randn(3, 40000, device=gpu)
    lse = torch.zeros(3, device=gpu)
    ws = torch.empty(max(capi.score_workspace_size(3, 40000, 4), 16), dtype=torch.uint8, device=gpu)
    capi.score_logits(z.data_ptr(), capi.GG_TYPE_F32, 3, 40000, 40000, None, 0, None, lse.data_ptr(), None, 0, None, None,
                      ws.data_ptr(), stream())
    assert torch.allclose(lse, torch.logsumexp(z.double(), 1).float(), rtol=1e-6)
    ids = torch.zeros(3, 4, dtype=torch.int32, device=gpu)
    capi.score_logits(z.data_ptr(), capi.GG_TYPE_F32, 3, 40000, 40000, None, 0, None, None, None, 4, ids.data_ptr(), None,
                      ws.data_ptr(), stream())
    assert torch.equal(ids.long(), torch.topk(z, 4, dim=1).indices)


def test_score_in_a_graph(gpu):
    n, top = 70000, 10
    z = torch.zeros(2, n, device=gpu)
    ids = torch.tensor([[5], [69999]], dtype=torch.int32, device=gpu)
    lp, ti = torch.zeros(2, 1, device=gpu), torch.zeros(2, top, dtype=torch.int32, device=gpu)
    ws = torch.full((capi.score_workspace_size(2, n, top),), 255, dtype=torch.uint8, device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        capi.score_logits(z.data_ptr(), capi.GG_TYPE_F32, 2, n, n, ids.data_ptr(), 1, lp.data_ptr(), None, None, top,
                          ti.data_ptr(), None, ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for rep in range(4):
        z.copy_(torch.randn(2, n))
        g.replay()
        torch.cuda.synchronize()
        kept, got = run(z.double().cpu().numpy(), "f32", ids.cpu().numpy(), top)
        check(kept, got, ids.cpu().numpy().astype(np.int64), top)
        assert np.array_equal(got["lp"], lp.cpu().numpy()) and np.array_equal(got["top_ids"], ti.cpu().numpy())


@pytest.mark.parametrize("m", [1, 29])
def test_lm_head_in_four_bits_selected_and_scored(gpu, m):
    """Hidden rows -> 4-bit LM head -> the selection and the log probabilities of the next ids."""
    from mx_ref import product_bound, quantised
    V, H = 16384, 640
    rng = np.random.default_rng(m)
    w = (rng.standard_normal((V, H)) * 0.05).astype(np.float32)
    h = rng.standard_normal((m, H)).astype(np.float32)
    wd, hd = torch.from_numpy(w).to(gpu), torch.from_numpy(h).to(gpu)
    wp = torch.empty(capi.mxfp4_packed_size(V, H), dtype=torch.uint8, device=gpu)
    logits = torch.empty(m, V, device=gpu)
    ws = torch.empty(max(capi.mxfp4_linear_workspace_size(capi.GG_TYPE_F32, m, V, H), 16), dtype=torch.uint8, device=gpu)
    s = stream()
    capi.mxfp4_quantize(wd.data_ptr(), capi.GG_TYPE_F32, V, H, H, wp.data_ptr(), s)
    capi.mxfp4_linear(wp.data_ptr(), hd.data_ptr(), capi.GG_TYPE_F32, H, logits.data_ptr(), capi.GG_TYPE_F32, V, m, V, H,
                      ws.data_ptr(), s)
    sel = torch.empty(capi.select_workspace_size(V), dtype=torch.uint8, device=gpu)
    chosen = [capi.select_logits(logits[i].data_ptr(), V, None, 0.0, 0.9, 1.0, 0.0, sel.data_ptr(), None, s) for i in range(m)]
    ids = np.array(chosen)[:, None]
    kept, got = run(logits.double().cpu().numpy(), "f32", ids, 5)
    assert np.array_equal(got["top_ids"][:, 0], np.array(chosen))
    assert np.array_equal(got["top_lp"][:, 0], got["lp"][:, 0])
    # against 64 bits all the way: a log probability moves by at most twice what the logits do
    wq = quantised(w)
    z = h.astype(np.float64) @ wq.T
    move = product_bound(h.astype(np.float64), wq, z, "f32", "f32").max()
    lse, ent, lp, order = scores(z, 5)
    assert (np.abs(got["lp"] - np.take_along_axis(lp, ids, 1)) <= 2 * move + 1e-5).all()


def test_many_rows(gpu):
    """More rows than one grid's threads allow: 2^24 and a few, of two logits."""
    rows = (1 << 24) + 5
    say("score", rows)
    z = (torch.arange(2 * rows, device="cuda:0") % 7).to(torch.float32).view(rows, 2)
    ids = (torch.arange(rows, device="cuda:0", dtype=torch.int32) % 2)
    lp, lse, ent, top_lp = (torch.full((rows,), 9.0, device="cuda:0") for _ in range(4))
    top = torch.full((rows,), 9, dtype=torch.int32, device="cuda:0")
    assert capi.score_workspace_size(rows, 2, 1) == 0
    capi.score_logits(z.data_ptr(), capi.GG_TYPE_F32, rows, 2, 2, ids.data_ptr(), 1, lp.data_ptr(), lse.data_ptr(),
                      ent.data_ptr(), 1, top.data_ptr(), top_lp.data_ptr(), None, stream())
    torch.cuda.synchronize()
    all_lp = torch.log_softmax(z.double(), 1)
    tol = score_rel(2) + 2.0 ** -20
    assert ((lse - torch.logsumexp(z.double(), 1)).abs() <= tol + 2.0 ** -20).all()
    assert ((lp - all_lp.gather(1, ids.long()[:, None])[:, 0]).abs() <= tol).all()
    assert ((ent + (all_lp.exp() * all_lp).sum(1)).abs() <= 4 * tol).all()
    assert torch.equal(top.long(), z.argmax(1)) and ((top_lp - all_lp.amax(1)).abs() <= tol).all()


@pytest.mark.parametrize("path,vocab", [("fused", 16384), ("fused", 2048), ("graph", 2048)])
def test_score_of_the_token_loop(gpu, path, vocab):
    """gg_score against the logits that gg_read returns, after a select, steps and collected steps, on each decode path."""
    from dataclasses import replace

    from gemma_amd import synth
    shape = replace(synth.TINY, vocab=vocab).gemma3_mode(window=7)
    e = capi.Engine(shape.gg_config())
    e.set_decode_path(path)
    e.upload_model(synth.make_model(shape, seed=3))
    e.finalize()
    with pytest.raises(capi.GGError) as err:
        e.score([1])
    assert err.value.code == capi.GG_ERR_INVALID
    prompt = synth.prompt_ids(9, seed=11, vocab=shape.vocab)
    e.prefill(prompt, 0)

    def check_now(tok, greedy):
        got = e.score([tok, 0, -1], top_n=5)
        z = e.read(capi.READ_LOGITS).astype(np.float64)[None]
        lse, ent, lp, order = scores(z, 5)
        tol = score_rel(vocab) + 2.0 ** -22 * (1 + np.log(vocab)) + 2.0 ** -23 * np.abs(lp).max()
        assert abs(got["lse"] - lse[0]) <= tol + 2.0 ** -23 * abs(lse[0]) and abs(got["entropy"] - ent[0]) <= tol * 2
        assert np.array_equal(got["top_ids"], order[0])
        assert (np.abs(got["top_logprobs"] - lp[0, order[0]]) <= tol).all()
        assert abs(got["logprobs"][0] - lp[0, tok]) <= tol and abs(got["logprobs"][1] - lp[0, 0]) <= tol
        assert got["logprobs"][2] == 0
        if greedy:
            assert got["top_ids"][0] == tok

    say("score in the loop", path, vocab)
    tok = e.select()
    check_now(tok, True)
    pos = len(prompt)
    for i in range(3):
        tok = e.step(tok, pos + i, *((0.0, 0.9, 1.0, 0.0) if i < 2 else (0.7, 0.9, 1.2, 0.4)))
        check_now(tok, i < 2)
    e.step_submit(tok, pos + 3)
    with pytest.raises(capi.GGError):
        e.score([1])
    check_now(e.step_collect(), True)
    for bad in (dict(ids=[1] * 257), dict(top_n=65), dict(top_n=-1)):
        with pytest.raises(capi.GGError) as err:
            e.score(**bad)
        assert err.value.code == capi.GG_ERR_INVALID
    check_now(e.step(tok, pos + 4), True)
    e.close()
