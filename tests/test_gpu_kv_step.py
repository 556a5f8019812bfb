"""The K/V page, attention and verification calls together, as a server's steps
use them: QKV product in 4-bit weights -> rows into pages -> attention -> output
product -> logits -> verification of drafts -> the next step's lengths."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from kv_ref import Pool, TYPES, attention, e4m3_row, i32, norm_rope, seqs_of, verify
from mx_ref import quantised

pytestmark = pytest.mark.gpu
H, V, HEADS, KV, D, EPS, THETA = 256, 4096, 4, 2, 64, 1e-6, 1e4
F32 = capi.GG_TYPE_F32


class Weights:
    def __init__(self, rng):
        self.f64, self.packed = {}, {}
        for name, n, k in (("qkv", (HEADS + 2 * KV) * D, H), ("o", H, HEADS * D), ("head", V, H)):
            w = (rng.standard_normal((n, k)) * k ** -0.5 * (3 if name == "head" else 1)).astype(np.float32)
            t = torch.from_numpy(w).cuda()
            p = torch.empty(capi.mxfp4_packed_size(n, k), dtype=torch.uint8, device="cuda:0")
            capi.mxfp4_quantize(t.data_ptr(), F32, n, k, k, p.data_ptr(), stream())
            self.packed[name] = (p, n, k)
            self.f64[name] = quantised(w)
        self.embed = rng.standard_normal((V, H)).astype(np.float32)
        self.q_norm, self.k_norm = (rng.random(D) + 0.5).astype(np.float32), (rng.random(D) + 0.5).astype(np.float32)

    def linear(self, name, x):
        p, n, k = self.packed[name]
        m = x.shape[0]
        y = torch.empty(m, n, device="cuda:0")
        ws = torch.empty(max(capi.mxfp4_linear_workspace_size(F32, m, n, k), 16), dtype=torch.uint8, device="cuda:0")
        capi.mxfp4_linear(p.data_ptr(), x.data_ptr(), F32, k, y.data_ptr(), F32, n, m, n, k, ws.data_ptr(), stream())
        return y


def forward(w, pool, seqs, tokens, window, sinks):
    """Logits of every new row; the rows are stored on the way."""
    x = torch.from_numpy(w.embed[tokens]).cuda()
    qkv = w.linear("qkv", x)
    n, width = qkv.shape
    q = torch.empty(n, HEADS * D, device="cuda:0")
    qn, kn = torch.from_numpy(w.q_norm).cuda(), torch.from_numpy(w.k_norm).cuda()
    base = qkv.data_ptr()
    pages = pool.pages()
    capi.kv_store(pages, seqs, F32, base, width, base + 4 * HEADS * D, width, base + 4 * (HEADS + KV) * D, width, HEADS, qn.data_ptr(),
                  kn.data_ptr(), EPS, THETA, q.data_ptr(), F32, HEADS * D, stream())
    out = torch.empty_like(q)
    ws = torch.empty(max(capi.kv_attention_workspace_size(pages, seqs, HEADS, window, sinks), 16), dtype=torch.uint8, device="cuda:0")
    capi.kv_attention(pages, seqs, q.data_ptr(), F32, HEADS * D, HEADS, D ** -0.5, window, sinks, out.data_ptr(), HEADS * D, None,
                      ws.data_ptr(), stream())
    return w.linear("head", x + w.linear("o", out))


def plain(w, tokens, first, cache, window, sinks):
    """Logits of rows first.. of one sequence, 64 bits throughout but for what the pages keep."""
    x = w.embed[tokens].astype(np.float64)
    qkv = (x @ w.f64["qkv"].T).reshape(len(tokens), -1, D)
    pos = np.arange(len(tokens))
    q = norm_rope(qkv[:, :HEADS], w.q_norm.astype(np.float64), pos, EPS, THETA)
    k = norm_rope(qkv[:, HEADS:HEADS + KV], w.k_norm.astype(np.float64), pos, EPS, THETA)
    v = qkv[:, HEADS + KV:]
    if cache == "e4m3":
        k, v = e4m3_row(k), e4m3_row(v)
    else:
        k, v = (torch.from_numpy(t).to(TYPES[cache][1]).double().numpy() for t in (k, v))
    out = np.stack([attention(q[first:, h], k[:, h // 2], v[:, h // 2], pos[first:], D ** -0.5, window, sinks, "bf16", "f32")[0]
                    for h in range(HEADS)], 1)
    x = x[first:] + out.reshape(len(x) - first, -1) @ w.f64["o"].T
    return x @ w.f64["head"].T


@pytest.mark.parametrize("cache,window,sinks", [("bf16", 0, 0), ("e4m3", 40, 4)])
def test_speculative_steps(gpu, cache, window, sinks):
    rng = np.random.default_rng(3)
    w = Weights(rng)
    prompts = [rng.integers(0, V, n) for n in (150, 1, 37)]
    room = [n + 40 for n in (150, 1, 37)]
    pool = Pool(room, 16, KV, D, cache, extra_columns=2)
    # the prompts but for their last tokens
    rows = [len(p) - 1 for p in prompts]
    seqs, keep = seqs_of(pool, rows, rows, max_len=200)
    z = forward(w, pool, seqs, np.concatenate([p[:-1] for p in prompts]), window, sinks)
    torch.cuda.synchronize()
    at = 0
    for p in prompts:
        if len(p) > 1:
            ref = plain(w, p[:-1], 0, cache, window, sinks)
            # a value of K or V that lands on the other side of a border (f32 products) moves a logit by up to 2^-4 of one
            # weight's share of 150: far under 1% of the largest logit; everything else is f32 sums of 256
            assert np.abs(z[at:at + len(p) - 1].double().cpu().numpy() - ref).max() < 0.01 * np.abs(ref).max()
            at += len(p) - 1
    texts = [list(p) for p in prompts]
    heat = torch.tensor([0.0, 1.0, 0.7], device="cuda:0")
    for step in range(4):
        drafts = [list(rng.integers(0, V, rng.integers(0, 5))) for _ in texts]
        if step == 1:   # a draft that stands: what the greedy sequence says next
            drafts[0] = [int(np.argmax(plain(w, np.array(texts[0]), len(texts[0]) - 1, cache, window, sinks)[0]))]
        rows = [1 + len(d) for d in drafts]
        lengths = [len(t) + len(d) for t, d in zip(texts, drafts)]
        seqs, keep = seqs_of(pool, rows, lengths, max_len=200)
        new = np.concatenate([[t[-1]] + d for t, d in zip(texts, drafts)]).astype(np.int64)
        z = forward(w, pool, seqs, new, window, sinks)
        n, start = len(new), np.concatenate([[0], np.cumsum(rows)])
        ids = np.concatenate([d + [0] for d in drafts])
        u, v = rng.random(n), rng.random(3)
        dt, st, ut, vt = i32(ids), i32(start), torch.from_numpy(u).cuda(), torch.from_numpy(v).cuda()
        acc, tok = torch.empty(3, dtype=torch.int32, device="cuda:0"), torch.empty(n, dtype=torch.int32, device="cuda:0")
        lp = torch.empty(n, device="cuda:0")
        ws = torch.empty(capi.verify_drafts_workspace_size(n, 3, V), dtype=torch.uint8, device="cuda:0")
        capi.verify_drafts(z.data_ptr(), None, F32, n, V, V, V, dt.data_ptr(), st.data_ptr(), 3, heat.data_ptr(), ut.data_ptr(), vt.data_ptr(),
                           acc.data_ptr(), tok.data_ptr(), lp.data_ptr(), ws.data_ptr(), stream())
        torch.cuda.synchronize()
        zk = z.double().cpu().numpy()
        ref = np.concatenate([plain(w, np.array(t + d), len(t) - 1, cache, window, sinks) for t, d in zip(texts, drafts)])
        say("step", step, rows, lengths, acc.tolist(), "logits off by", np.abs(zk - ref).max() / np.abs(ref).max())
        assert np.abs(zk - ref).max() < 0.01 * np.abs(ref).max()
        ra, rt, rl, m = verify(zk, None, ids, start, np.array([0.0, 1.0, np.float32(0.7)]), u, v)
        assert (m > 1e-9).all() and np.array_equal(acc.cpu().numpy(), ra) and np.array_equal(tok.cpu().numpy(), rt)
        if step == 1:
            assert int(acc[0]) == 1
        # what does not stand is written over by the next step's rows
        for s in range(3):
            texts[s] += [int(t) for t in tok[start[s]:start[s] + int(acc[s]) + 1]]
