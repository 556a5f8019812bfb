"""Timed cases of the 4-bit matrix operators and of scoring.

MXFP4 (4-bit elements e2m1, one power-of-two scale for 32 of them): rows
quantised, and products with weights held in it. Log probabilities of given
tokens over rows of logits, with entropy and the best alternatives. Both in a
plain form of elementary torch operations and, with `own` true, through the
library's kernel-level entry points (gemma_amd.capi).

Sizes are those of the Gemma-3 1B shape where a case says so (hidden 1152, QKV
1536, intermediate 6912, vocabulary 262144), otherwise generic.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
VOCAB = 262144
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the FFN activations of a ragged conversation turn through 4 bits and back: what 4-bit inputs would cost in accuracy
        {"name": "quantize_turn", "kind": "round_trip", "rows": 187, "k": 6912, "type": "f32"},
        # the tied LM head of the 1B shape, from a bf16 checkpoint: the largest tensor of a model at load
        {"name": "quantize_lm_head", "kind": "round_trip", "rows": VOCAB, "k": 1152, "type": "bf16"},
        # one token's QKV projection: the smallest product, where latency counts
        {"name": "linear_qkv_token", "kind": "linear", "m": 1, "n": 1536, "k": 1152, "x": "f32", "y": "f32"},
        # one token's down projection: few rows, long sums
        {"name": "linear_down_token", "kind": "linear", "m": 1, "n": 1152, "k": 6912, "x": "f32", "y": "f32"},
        # one token's LM head: a stream of weights from memory
        {"name": "linear_lm_head_token", "kind": "linear", "m": 1, "n": VOCAB, "k": 1152, "x": "f32", "y": "f32"},
        # gate and up for a few sequences that decode together
        {"name": "linear_gate_up_batch7", "kind": "linear", "m": 7, "n": 13824, "k": 1152, "x": "f32", "y": "f32"},
        # gate and up of a 2048-id prompt
        {"name": "linear_gate_up_prompt", "kind": "linear", "m": 2048, "n": 13824, "k": 1152, "x": "f32", "y": "f32"},
        # a layer of a larger model on a long prompt, bf16 activations: bound by the matrix rate
        {"name": "linear_bf16_large", "kind": "linear", "m": 4000, "n": 8192, "k": 8192, "x": "bf16", "y": "bf16"},
        # a ragged turn with its activations quantised too
        {"name": "linear_both_turn", "kind": "linear_both", "m": 187, "n": 13824, "k": 1152, "x": "bf16", "y": "bf16"},
        # the larger layer with both operands in 4 bits
        {"name": "linear_both_large", "kind": "linear_both", "m": 4096, "n": 8192, "k": 8192, "x": "bf16", "y": "bf16"},
        # the chosen token's log probability and twenty alternatives, once a decode step
        {"name": "score_token", "kind": "score", "rows": 1, "n": VOCAB, "type": "f32", "ids": 1, "top": 20},
        # the log probabilities of a prompt's own tokens
        {"name": "score_prompt", "kind": "score", "rows": 1021, "n": VOCAB, "type": "bf16", "ids": 1, "top": 5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["round_trip", "linear", "linear", "linear_both", "score"])
    if kind == "round_trip":
        k = _log_int(rng, 32, 16384)
        return {"kind": kind, "rows": _log_int(rng, 1, max(1, min(VOCAB, VOCAB * 1152 // k))), "k": k,
                "type": rng.choice(list(DTYPES))}
    if kind == "score":
        n = _log_int(rng, 1000, VOCAB)
        return {"kind": kind, "rows": _log_int(rng, 1, min(2048, 1000 * VOCAB // n)), "n": n, "type": rng.choice(list(DTYPES)),
                "ids": rng.randint(1, 4), "top": rng.randint(0, 20)}
    m = _log_int(rng, 1, 4096) if rng.random() < 0.6 or kind == "linear_both" else rng.randint(1, 16)
    k = _log_int(rng, 64, 8192)
    n = _log_int(rng, 64, max(64, min(VOCAB, 1152 * VOCAB // k, (1 << 37) // (m * k), (1 << 28) // m)))
    x = rng.choice(list(DTYPES))
    return {"kind": kind, "m": m, "n": n, "k": k, "x": x, "y": rng.choice(["f32", x])}


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _activations(gen, m, k):
    """N(0, 1) with a few channels twenty times as large, as hidden states have them."""
    ch = torch.where(torch.rand(k, generator=gen, device=DEV) < 0.01, 20.0, 1.0)
    return torch.randn(m, k, generator=gen, device=DEV) * ch


def _weights(gen, n, k):
    """N(0, 0.02), f32."""
    return torch.randn(n, k, generator=gen, device=DEV) * 0.02


def _logits(gen, case):
    """Logits of a model that is fairly sure: N(0, 2), the best of them raised."""
    z = torch.randn(case["rows"], case["n"], generator=gen, device=DEV) * 2
    best = torch.randint(0, case["n"], (case["rows"], 8), generator=gen, device=DEV)
    up = torch.rand(case["rows"], 8, generator=gen, device=DEV) * 8
    return z.scatter_add_(1, best, up).to(DTYPES[case["type"]])


def _given(gen, case):
    return torch.randint(0, case["n"], (case["rows"], case["ids"]), generator=gen, device=DEV, dtype=torch.int32)


def _inputs(case, seed):
    """The tensors of a case: rows, (activations, f32 weights) or (logits, ids)."""
    gen = _generator(seed)
    if case["kind"] == "round_trip":
        return _activations(gen, case["rows"], case["k"]).to(DTYPES[case["type"]])
    if case["kind"] == "score":
        return _logits(gen, case), _given(gen, case)
    x = _activations(gen, case["m"], case["k"]).to(DTYPES[case["x"]])
    return x, _weights(gen, case["n"], case["k"])


# ---- the library's calls -----------------------------------------------------

def _capi():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webgpu-gemma_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from gemma_amd import capi
    return capi


def _bytes(n):
    return torch.empty(max(int(n), 1), dtype=torch.uint8, device=DEV)


def _ggml(capi, name):
    return {"f32": capi.GG_TYPE_F32, "bf16": capi.GG_TYPE_BF16, "f16": capi.GG_TYPE_F16}[name]


def prepare(case, seed):
    kind = case["kind"]
    state = {"case": case}
    if own:
        capi = _capi()
        state.update(capi=capi, stream=torch.cuda.current_stream().cuda_stream)
    if kind == "round_trip":
        x = state["x"] = _inputs(case, seed)
        if own:
            state.update(packed=_bytes(capi.mxfp4_packed_size(*x.shape)), out=torch.empty(x.shape, device=DEV))
        return state
    if kind == "score":
        state["logits"], state["ids"] = _inputs(case, seed)
        if own:
            r, t = case["rows"], case["top"]
            state.update(ws=_bytes(capi.score_workspace_size(r, case["n"], t)), lp=torch.empty(r, case["ids"], device=DEV),
                         lse=torch.empty(r, device=DEV), entropy=torch.empty(r, device=DEV),
                         top_ids=torch.empty(r, t, dtype=torch.int32, device=DEV), top_lp=torch.empty(r, t, device=DEV))
        return state
    x, w = _inputs(case, seed)
    state["x"] = x
    if not own:
        state["w"] = _plain_quantize(w)   # what is kept of the weights: nibbles and scale bytes
        return state
    m, n, k = case["m"], case["n"], case["k"]
    wp = _bytes(capi.mxfp4_packed_size(n, k))
    capi.mxfp4_quantize(w.data_ptr(), capi.GG_TYPE_F32, n, k, k, wp.data_ptr(), state["stream"])
    xt = capi.GG_TYPE_MXFP4 if kind == "linear_both" else _ggml(capi, case["x"])
    state.update(w=wp, xt=xt, yt=_ggml(capi, case["y"]), y=torch.empty(m, n, dtype=DTYPES[case["y"]], device=DEV),
                 ws=_bytes(capi.mxfp4_linear_workspace_size(xt, m, n, k)))
    if kind == "linear_both":
        state["xp"] = _bytes(capi.mxfp4_packed_size(m, k))
    return state


def run(state):
    case = state["case"]
    if not own:
        return _plain(state)
    capi, stream, kind = state["capi"], state["stream"], case["kind"]
    if kind == "round_trip":
        x, rows, k = state["x"], case["rows"], case["k"]
        capi.mxfp4_quantize(x.data_ptr(), _ggml(capi, case["type"]), rows, k, k, state["packed"].data_ptr(), stream)
        capi.mxfp4_dequant(state["packed"].data_ptr(), state["out"].data_ptr(), rows, k, k, stream)
        return state["out"]
    if kind == "score":
        capi.score_logits(state["logits"].data_ptr(), _ggml(capi, case["type"]), case["rows"], case["n"], case["n"],
                          state["ids"].data_ptr(), case["ids"], state["lp"].data_ptr(), state["lse"].data_ptr(),
                          state["entropy"].data_ptr(), case["top"], state["top_ids"].data_ptr(), state["top_lp"].data_ptr(),
                          state["ws"].data_ptr(), stream)
        return {k: state[k] for k in ("lp", "lse", "entropy", "top_ids", "top_lp")[:5 if case["top"] else 3]}
    m, n, k = case["m"], case["n"], case["k"]
    x = state["x"]
    if kind == "linear_both":
        capi.mxfp4_quantize(x.data_ptr(), _ggml(capi, case["x"]), m, k, k, state["xp"].data_ptr(), stream)
        x = state["xp"]
    capi.mxfp4_linear(state["w"].data_ptr(), x.data_ptr(), state["xt"], k, state["y"].data_ptr(), state["yt"], n, m, n, k,
                      state["ws"].data_ptr(), stream)
    return state["y"]


# ---- the plain form: 32 bits, elementary operations ----------------------------

def _plain_quantize(x):
    """(nibbles uint8 [rows, ceil(k / 32), 16], scale bytes uint8 [rows, ceil(k / 32)]) of rows of x."""
    rows, k = x.shape
    nb = -(-k // 32)
    x = torch.nn.functional.pad(x.float(), (0, nb * 32 - k)).view(rows, nb, 32)
    e = (torch.frexp(x.abs().amax(2))[1] - 3).clamp_(-127, 127)          # floor(log2(max)) - 2
    a = torch.ldexp(x.abs(), -e[:, :, None])
    code = (a > 0.25).to(torch.uint8)
    for limit, tie_up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= limit) if tie_up else (a > limit)
    code += (x < 0).to(torch.uint8) * 8
    return code[:, :, 0::2] | (code[:, :, 1::2] << 4), (e + 127).to(torch.uint8)


def _plain_dequant(nibbles, scale, k):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    table = torch.cat([table, -table])
    v = torch.stack([table[(nibbles & 15).int()], table[(nibbles >> 4).int()]], 3).view(*scale.shape, 32)
    v = torch.ldexp(v, (scale.int() - 127)[:, :, None])
    return v.view(scale.shape[0], -1)[:, :k]


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "round_trip":
        return _plain_dequant(*_plain_quantize(state["x"]), case["k"])
    if kind == "score":
        return _plain_score(state["logits"].float(), state["ids"].long(), case["top"])
    x = state["x"].float()
    if kind == "linear_both":
        x = _plain_dequant(*_plain_quantize(x), case["k"])
    return (x @ _plain_dequant(*state["w"], case["k"]).T).to(DTYPES[case["y"]])


def _plain_score(z, ids, top):
    m = z.amax(1, keepdim=True)
    d = z - m
    p = torch.exp(d)
    s = p.sum(1, keepdim=True)
    log_s = torch.log(s)
    out = {"lp": d.gather(1, ids) - log_s, "lse": (m + log_s)[:, 0], "entropy": (log_s - (p * d).sum(1, keepdim=True) / s)[:, 0]}
    del p
    if top == 0:
        return out
    # values as ordered integers over the reversed index: among equal values the lowest id comes first
    key = z.view(torch.int32).long()
    key = torch.where(key < 0, -(key & 0x7FFFFFFF), key)
    key = (key << 32) + (z.shape[1] - torch.arange(z.shape[1], device=DEV))
    best = z.shape[1] - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)
    out["top_ids"], out["top_lp"] = best.int(), d.gather(1, best) - log_s
    return out


# ---- work ----------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "round_trip":
        n = case["rows"] * case["k"]
        return {"bytes": n * (SIZES[case["type"]] + 4), "flops": 2 * n}
    if kind == "score":
        n = case["rows"] * case["n"]
        return {"bytes": n * SIZES[case["type"]] + case["rows"] * (8 * case["ids"] + 8 + 8 * case["top"]), "flops": 5 * n}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": n * -(-k // 32) * 17 + m * k * SIZES[case["x"]] + m * n * SIZES[case["y"]], "flops": 2 * m * n * k}


# ---- the definition in 64 bits ---------------------------------------------------

def _exact_mx(x):
    """The values that MXFP4 keeps of the rows of x, f64: rounding to a step of a half, one or two of the block's unit."""
    rows, k = x.shape
    x = torch.cat([x.double(), x.new_zeros(rows, -k % 32, dtype=torch.float64)], 1).view(rows, -1, 32)
    top = x.abs().amax(2, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2).clamp_(2.0 ** -127, 2.0 ** 127)
    y = x / unit
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp_(-6, 6)
    return (y * unit).view(rows, -1)[:, :k]


def exact(case, seed):
    kind = case["kind"]
    if kind == "round_trip":
        return _exact_mx(_inputs(case, seed))
    if kind == "score":
        z, ids = _inputs(case, seed)
        parts = [_exact_score(z[i:i + 64].double(), ids[i:i + 64].long(), case["top"]) for i in range(0, case["rows"], 64)]
        return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    x, w = _inputs(case, seed)
    x = _exact_mx(x) if kind == "linear_both" else x.double()
    return torch.cat([x @ _exact_mx(w[i:i + 32768]).T for i in range(0, case["n"], 32768)], 1)


def _exact_score(z, ids, top):
    lse = torch.logsumexp(z, 1, keepdim=True)
    lp = z - lse
    out = {"lp": lp.gather(1, ids), "lse": lse[:, 0], "entropy": -(torch.exp(lp) * lp).sum(1)}
    if top:
        order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
        out.update(top_ids=order.int(), top_lp=lp.gather(1, order))
    return out
