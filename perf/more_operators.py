"""Timed cases of serving with K/V pages: rows stored in them, attention over
them, and verification of drafted tokens.

Keys and values live in pages of a few positions that a table gives to each
sequence, in 16 bits or in 8 (e4m3 with a power-of-two scale for each row). New
rows are normed, rotated and stored; a chunk of new rows of every sequence, one
or many, attends to all that its sequence has, or to a sliding window and a few
first positions; drafted tokens are accepted or replaced by given random
numbers. All in a plain form of elementary torch operations and, with `own`
true, through the library's kernel-level entry points (gemma_amd.capi).

Sizes are those of the Gemma-3 1B shape where a case says so (4 query heads on
one K/V head of 256, window 512, vocabulary 262144), otherwise generic.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
VOCAB = 262144
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
EPS, THETA = 1e-6, 1e6


def listed():
    return [
        # one token's QKV rows of the 1B shape: the smallest call, where latency counts
        {"name": "store_token", "kind": "store", "seqs": 1, "rows": 1, "max_len": 2049, "heads": 4, "kv_heads": 1, "dim": 256,
         "page": 64, "cache": "bf16", "x": "f32"},
        # five ragged prompts of a larger model into an 8-bit cache, as a server admits them together
        {"name": "store_prompts_e4m3", "kind": "store", "seqs": 5, "rows": 1021, "max_len": 1500, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "cache": "e4m3", "x": "bf16"},
        # one token of the 1B shape on a global layer
        {"name": "attention_token", "kind": "attention", "seqs": 1, "rows": 1, "max_len": 2049, "heads": 4, "kv_heads": 1, "dim": 256,
         "page": 64, "cache": "bf16", "x": "f32", "window": 0, "sinks": 0},
        # one token of the 1B shape on a local layer, late in a long conversation, with four first positions kept
        {"name": "attention_token_window", "kind": "attention", "seqs": 1, "rows": 1, "max_len": 32760, "heads": 4, "kv_heads": 1,
         "dim": 256, "page": 64, "cache": "bf16", "x": "f32", "window": 512, "sinks": 4},
        # a server's decode step: sequences of all lengths
        {"name": "attention_batch", "kind": "attention", "seqs": 61, "rows": 1, "max_len": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "cache": "bf16", "x": "bf16", "window": 0, "sinks": 0},
        # few very long sequences in 8 bits: a stream from memory
        {"name": "attention_long_e4m3", "kind": "attention", "seqs": 3, "rows": 1, "max_len": 131072, "heads": 16, "kv_heads": 4, "dim": 256,
         "page": 64, "cache": "e4m3", "x": "bf16", "window": 0, "sinks": 0},
        # drafted tokens of several sequences, verified in one pass
        {"name": "attention_drafts", "kind": "attention", "seqs": 16, "rows": 6, "max_len": 4096, "heads": 16, "kv_heads": 8, "dim": 128,
         "page": 32, "cache": "f16", "x": "f16", "window": 0, "sinks": 0},
        # a chunk of a long prompt behind what is cached: bound by the matrix rate
        {"name": "attention_chunk", "kind": "attention", "seqs": 1, "rows": 2048, "max_len": 32768, "heads": 4, "kv_heads": 1, "dim": 256,
         "page": 64, "cache": "bf16", "x": "bf16", "window": 0, "sinks": 0},
        # ragged turns of four conversations on a local layer, f32 rows as the token loop has them
        {"name": "attention_turns_window", "kind": "attention", "seqs": 4, "rows": 800, "max_len": 5000, "heads": 4, "kv_heads": 1, "dim": 256,
         "page": 64, "cache": "bf16", "x": "f32", "window": 512, "sinks": 4},
        # whole ragged prompts of a larger model, nothing cached before them
        {"name": "attention_prompts", "kind": "attention", "seqs": 5, "rows": 1500, "max_len": 1500, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "cache": "bf16", "x": "bf16", "window": 0, "sinks": 0},
        # four tokens drafted from the prompt's own n-grams, one sequence
        {"name": "verify_one", "kind": "verify", "seqs": 1, "drafts": 4, "vocab": VOCAB, "z": "f32", "draft": False},
        # a server's step with a draft model, sequences with none to six drafts, some of them greedy
        {"name": "verify_batch", "kind": "verify", "seqs": 48, "drafts": 6, "vocab": VOCAB, "z": "bf16", "draft": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "attention", "attention", "attention", "verify"])
    if kind == "verify":
        vocab, drafts = _log_int(rng, 1000, VOCAB), rng.randint(1, 8)
        return {"kind": kind, "seqs": _log_int(rng, 1, max(1, min(64, 48 * 7 * VOCAB // (vocab * (drafts + 1))))), "drafts": drafts,
                "vocab": vocab, "z": rng.choice(["f32", "bf16", "f16"]), "draft": rng.random() < 0.5}
    kv, dim = rng.choice([1, 1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 128, 192, 256, 256])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    cache = rng.choice(["bf16", "bf16", "f16", "e4m3"])
    c = {"kind": kind, "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([1, 16, 16, 24, 32, 64, 64, 100, 256, 1000]),
         "cache": cache, "x": "f16" if cache == "f16" and kind == "attention" else rng.choice(["f32", "bf16", "f16"])}
    few = rng.random() < 0.5
    rows = rng.randint(1, 8) if few else _log_int(rng, 9, 2048)
    seqs = _log_int(rng, 1, 64 if few else max(1, min(16, 6000 // rows)))
    most = 1 << 27   # what the plain form expands: K or V, and scores
    max_len = _log_int(rng, max(rows, 16), max(rows, 16, min(131072, most // (seqs * kv * dim), most // (seqs * heads * rows))))
    c.update(seqs=seqs, rows=min(rows, max_len), max_len=max_len)
    if kind == "attention":
        window = 0 if rng.random() < 0.5 else _log_int(rng, 1, 4096)
        c.update(window=window, sinks=rng.choice([0, 1, 4, 70]) if window else 0)
    return c


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(case):
    """(rows, length behind them) of each sequence, ragged: the first has the largest of both."""
    rng = random.Random(7919 * case["max_len"] + case["seqs"])
    rows, length = [], []
    for s in range(case["seqs"]):
        length.append(case["max_len"] if s == 0 else max(case["rows"], int(case["max_len"] * rng.uniform(0.15, 1.0))))
        rows.append(case["rows"] if s == 0 else rng.randint((case["rows"] + 1) // 2, case["rows"]))
        if case["kind"] == "attention" and case["rows"] == case["max_len"]:   # whole prompts: nothing cached before
            rows[s] = length[s] = case["rows"] if s == 0 else rng.randint((case["rows"] + 4) // 5, case["rows"])
    return rows, length


def _pages(case, gen, length):
    """Page tables of a pool in which the sequences' pages lie in any order, with some pages that no sequence has."""
    need = [-(-n // case["page"]) for n in length]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, n_pages


def _inputs(case, seed):
    gen = _generator(seed)
    if case["kind"] == "verify":
        return _verify_inputs(case, seed, gen)
    rows, length = _lengths(case)
    d, kv, heads = case["dim"], case["kv_heads"], case["heads"]
    table, n_pages = _pages(case, gen, length)
    start = [sum(rows[:s]) for s in range(len(rows) + 1)]
    shape = (n_pages, case["page"], kv, d)
    t = {"rows": rows, "length": length, "start": torch.tensor(start, dtype=torch.int32, device=DEV),
         "len": torch.tensor(length, dtype=torch.int32, device=DEV), "table": table}
    for name in ("k", "v"):
        if case["cache"] == "e4m3":   # values of any row's size: a power of two for each
            t[name] = (torch.randn(shape, generator=gen, device=DEV) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
            t[name + "_scale"] = torch.exp2(torch.randint(-8, -5, shape[:3], generator=gen, device=DEV).float())
        else:
            t[name] = torch.randn(shape, generator=gen, device=DEV).to(DTYPES[case["cache"]])
    x = DTYPES[case["x"]]
    if case["kind"] == "attention":
        t["q"] = (torch.randn(start[-1], heads * d, generator=gen, device=DEV) * 2).to(x)
    else:
        # rows of a QKV product: some channels much larger than others
        big = torch.where(torch.rand((heads + 2 * kv) * d, generator=gen, device=DEV) < 0.02, 10.0, 1.0)
        t["x"] = (torch.randn(start[-1], (heads + 2 * kv) * d, generator=gen, device=DEV) * big).to(x)
        t["q_norm"], t["k_norm"] = (torch.rand(d, generator=gen, device=DEV) + 0.5 for _ in range(2))
    return t


def _drafts(case):
    """Drafted tokens of each sequence: the first has the most."""
    rng = random.Random(case["vocab"])
    return [case["drafts"]] + [rng.randint(0, case["drafts"]) for _ in range(case["seqs"] - 1)]


def _verify_inputs(case, seed, gen):
    rng = random.Random(int(seed) * 104729 + 1)
    n, seqs = case["vocab"], case["seqs"]
    drafts = _drafts(case)
    start = [sum(drafts[:s]) + s for s in range(seqs + 1)]
    rows = start[-1]
    z = torch.randn(rows, n, generator=gen, device=DEV) * 2
    best = torch.randint(0, n, (rows, 8), generator=gen, device=DEV)
    z.scatter_add_(1, best, 2 + torch.rand(rows, 8, generator=gen, device=DEV) * 10)
    t = {"start": torch.tensor(start, dtype=torch.int32, device=DEV),
         "temperature": torch.tensor([0.0 if rng.random() < 0.25 and s else rng.choice([0.7, 1.0, 1.3]) for s in range(seqs)], device=DEV),
         "u": torch.rand(rows, generator=gen, device=DEV, dtype=torch.float64),
         "v": torch.rand(seqs, generator=gen, device=DEV, dtype=torch.float64)}
    # drafts that the target mostly agrees with
    guess = z + torch.randn(rows, n, generator=gen, device=DEV) * 0.5
    t["ids"] = guess.argmax(1).int()
    t["z"] = z.to(DTYPES[case["z"]])
    if case["draft"]:
        t["y"] = guess.to(DTYPES[case["z"]])
    return t


# ---- the library's calls -----------------------------------------------------

def _capi():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webgpu-gemma_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from gemma_amd import capi
    return capi


def _bytes(n):
    return torch.empty(max(int(n), 1), dtype=torch.uint8, device=DEV)


def _type(capi, name):
    return {"f32": capi.GG_TYPE_F32, "bf16": capi.GG_TYPE_BF16, "f16": capi.GG_TYPE_F16, "e4m3": capi.GG_TYPE_E4M3}[name]


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if not own:
        return state
    capi = _capi()
    state.update(capi=capi, stream=torch.cuda.current_stream().cuda_stream)
    if case["kind"] == "verify":
        seqs = case["seqs"]
        rows = state["z"].shape[0]
        state.update(accepted=torch.empty(seqs, dtype=torch.int32, device=DEV), tokens=torch.empty(rows, dtype=torch.int32, device=DEV),
                     logprobs=torch.empty(rows, device=DEV),
                     ws=_bytes(capi.verify_drafts_workspace_size(rows, seqs, case["vocab"])))
        return state
    n, d, kv, heads = sum(state["rows"]), case["dim"], case["kv_heads"], case["heads"]
    scales = [state[name].data_ptr() if name in state else None for name in ("k_scale", "v_scale")]
    state["pages"] = capi.kv_pages(state["k"].data_ptr(), state["v"].data_ptr(), _type(capi, case["cache"]), state["k"].shape[0],
                                   case["page"], kv, d, k_scale=scales[0], v_scale=scales[1])
    state["seqs"] = capi.kv_seqs(state["start"].data_ptr(), state["len"].data_ptr(), state["table"].data_ptr(), case["seqs"], n,
                                 max(state["rows"]), max(state["length"]), state["table"].shape[1])
    if case["kind"] == "attention":
        state.update(out=torch.empty(n, heads * d, dtype=DTYPES[case["x"]], device=DEV), lse=torch.empty(n, heads, device=DEV),
                     ws=_bytes(capi.kv_attention_workspace_size(state["pages"], state["seqs"], heads, case["window"], case["sinks"])))
    else:
        state["q_out"] = torch.empty(n, heads * d, dtype=DTYPES[case["x"]], device=DEV)
        if case["cache"] == "e4m3":
            state["k_out"], state["v_out"] = (torch.empty(n, kv * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    return state


def run(state):
    case = state["case"]
    if not own:
        return {"store": _plain_store, "attention": _plain_attention, "verify": _plain_verify}[case["kind"]](state)
    capi, stream = state["capi"], state["stream"]
    if case["kind"] == "verify":
        capi.verify_drafts(state["z"].data_ptr(), state["y"].data_ptr() if case["draft"] else None, _type(capi, case["z"]),
                           state["z"].shape[0], case["vocab"], case["vocab"], case["vocab"], state["ids"].data_ptr(), state["start"].data_ptr(),
                           case["seqs"], state["temperature"].data_ptr(), state["u"].data_ptr(), state["v"].data_ptr(),
                           state["accepted"].data_ptr(), state["tokens"].data_ptr(), state["logprobs"].data_ptr(),
                           state["ws"].data_ptr(), stream)
        return {name: state[name] for name in ("accepted", "tokens", "logprobs")}
    d, kv, heads = case["dim"], case["kv_heads"], case["heads"]
    if case["kind"] == "attention":
        capi.kv_attention(state["pages"], state["seqs"], state["q"].data_ptr(), _type(capi, case["x"]), heads * d, heads, d ** -0.5,
                          case["window"], case["sinks"], state["out"].data_ptr(), heads * d, state["lse"].data_ptr(), state["ws"].data_ptr(), stream)
        return {"out": state["out"], "lse": state["lse"]}
    x, size, ld = state["x"], SIZES[case["x"]], (heads + 2 * kv) * d
    capi.kv_store(state["pages"], state["seqs"], _type(capi, case["x"]), x.data_ptr(), ld, x.data_ptr() + heads * d * size, ld,
                  x.data_ptr() + (heads + kv) * d * size, ld, heads, state["q_norm"].data_ptr(), state["k_norm"].data_ptr(), EPS, THETA,
                  state["q_out"].data_ptr(), _type(capi, case["x"]), heads * d, stream)
    if case["cache"] != "e4m3":
        return {"q": state["q_out"], "k": state["k"], "v": state["v"]}
    capi.kv_load(state["pages"], state["seqs"], state["k_out"].data_ptr(), kv * d, state["v_out"].data_ptr(), kv * d, capi.GG_TYPE_BF16, stream)
    return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}


# ---- the plain form: elementary operations, 32 bits or 64 -----------------------

def _row_places(state):
    """Of each row: its sequence, its position, and where that lies in the pool."""
    case, start, length = state["case"], state["start"].long(), state["len"].long()
    row = torch.arange(sum(state["rows"]), device=DEV)
    seq = torch.searchsorted(start[1:], row, right=True)
    pos = length[seq] - (start[seq + 1] - row)
    return seq, pos, state["table"][seq, pos // case["page"]].long() * case["page"] + pos % case["page"]


def _plain_store(state):
    # in 64 bits: angles of far positions, and values next to a border of the 8-bit format
    case = state["case"]
    d, kv, heads = case["dim"], case["kv_heads"], case["heads"]
    _, pos, place = _row_places(state)
    n = pos.numel()
    x = state["x"].double().view(n, heads + 2 * kv, d)
    qk = x[:, :heads + kv]
    w = torch.cat([state["q_norm"].double().expand(heads, d), state["k_norm"].double().expand(kv, d)])
    qk = qk / torch.sqrt((qk * qk).mean(2, keepdim=True) + EPS) * w
    angle = pos.double()[:, None] * torch.pow(torch.tensor(THETA, dtype=torch.float64, device=DEV),
                                              -torch.arange(d // 2, device=DEV, dtype=torch.float64) * 2 / d)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = qk[:, :, :d // 2], qk[:, :, d // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    q = qk[:, :heads].reshape(n, -1).to(DTYPES[case["x"]])
    if case["cache"] != "e4m3":
        state["k"].view(-1, kv, d)[place] = qk[:, heads:].to(DTYPES[case["cache"]])
        state["v"].view(-1, kv, d)[place] = x[:, heads + kv:].to(DTYPES[case["cache"]])
        return {"q": q, "k": state["k"], "v": state["v"]}
    for name, r in (("k", qk[:, heads:]), ("v", x[:, heads + kv:])):
        m, e = torch.frexp(r.abs().amax(2))
        e = (e - 9 + (m > 0.875).int()).clamp_(min=-126)      # the least with max <= 448 2^e
        t = torch.ldexp(r, -e[:, :, None].double())
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_(min=2.0 ** -6))) - 3)
        state[name].view(-1, kv, d)[place] = (torch.round(t / step) * step).to(torch.float8_e4m3fn)
        state[name + "_scale"].view(-1, kv)[place] = torch.exp2(e.double()).float()
    k, v = (state[name].view(-1, kv, d)[place].float() * state[name + "_scale"].view(-1, kv)[place][:, :, None] for name in ("k", "v"))
    return {"q": q, "k": k.view(n, -1).bfloat16(), "v": v.view(n, -1).bfloat16()}


def _plain_attention(state):
    case = state["case"]
    d, kv, heads, page = case["dim"], case["kv_heads"], case["heads"], case["page"]
    g, rows, most = heads // kv, max(state["rows"]), max(state["length"])
    seqs = case["seqs"]
    key = torch.arange(most, device=DEV)
    place = state["table"][:, key // page].long().clamp_(min=0) * page + key % page          # [seqs, most]
    seen = key < state["len"].long()[:, None]
    k, v = (state[name].view(-1, kv, d)[place].float() for name in ("k", "v"))                 # [seqs, most, kv, d]
    if case["cache"] == "e4m3":
        k, v = (t * state[name].view(-1, kv)[place][..., None] for t, name in ((k, "k_scale"), (v, "v_scale")))
    v = torch.where(seen[:, :, None, None], v, 0.0)
    start, length = state["start"].long(), state["len"].long()
    n_rows = start[1:] - start[:-1]
    i = torch.arange(rows, device=DEV)
    live = i < n_rows[:, None]                                                              # [seqs, rows]
    at = torch.where(live, start[:-1, None] + i, 0)
    q = state["q"].float()[at].view(seqs, rows, kv, g, d).permute(0, 2, 1, 3, 4).reshape(seqs, kv, rows * g, d)
    s = (q.contiguous() @ k.permute(0, 2, 3, 1).contiguous()) * d ** -0.5                   # [seqs, kv, rows g, most]
    pos = (length - n_rows)[:, None] + i
    ok = (key <= pos[:, :, None]) & seen[:, None]
    if case["window"]:
        ok &= (key > pos[:, :, None] - case["window"]) | (key < case["sinks"])
    s.view(seqs, kv, rows, g, most).masked_fill_(~ok[:, None, :, None, :], -math.inf)
    m = s.amax(3, keepdim=True)
    m = torch.where(torch.isfinite(m), m, 0.0)
    s = s.sub_(m).exp_()
    total = s.sum(3, keepdim=True)
    o = (s @ v.permute(0, 2, 1, 3).contiguous()) / torch.where(total > 0, total, 1.0)
    o = o.view(seqs, kv, rows, g, d).permute(0, 2, 1, 3, 4).reshape(seqs, rows, heads * d)[live]
    lse = (m + total.log()).view(seqs, kv, rows, g).permute(0, 2, 1, 3).reshape(seqs, rows, heads)[live]
    return {"out": o.to(DTYPES[case["x"]]), "lse": lse}


def _plain_verify(state):
    # in 64 bits: the draw picks among borders that lie closer than 32 bits tell apart
    case = state["case"]
    start, t = state["start"].long(), state["temperature"].double()
    rows, n, seqs = state["z"].shape[0], case["vocab"], case["seqs"]
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(start[1:], row, right=True)
    greedy = t == 0
    heat = torch.where(greedy, 1.0, t)[seq][:, None]

    def softmax(x):
        x = x.double() / heat
        x = (x - x.amax(1, keepdim=True)).exp_()
        return x / x.sum(1, keepdim=True)
    p = softmax(state["z"])
    ids = state["ids"].long()
    best = torch.where(state["z"] == state["z"].amax(1, keepdim=True), torch.arange(n, device=DEV), n).amin(1)
    at_id = p.gather(1, ids[:, None])[:, 0]
    if case["draft"]:
        q = softmax(state["y"])
        keep = state["u"] * q.gather(1, ids[:, None])[:, 0] < at_id
    else:
        keep = state["u"] < at_id
    keep = torch.where(greedy[seq], ids == best, keep)
    last = row == start[seq + 1] - 1
    # the first row of each sequence that does not keep its draft; its last row has none
    stop = torch.where(keep & ~last, rows, row)
    stop = torch.full((seqs,), rows, device=DEV).scatter_reduce_(0, seq, stop, "amin")
    w = p[stop]
    rejected = ~last[stop]
    if case["draft"]:
        w = torch.where(rejected[:, None], (w - q[stop]).clamp_(min=0), w)
    else:
        w = torch.where(rejected[:, None] & (torch.arange(n, device=DEV) == ids[stop][:, None]), 0.0, w)
    sums = torch.cumsum(w, 1)
    pick = (sums <= (state["v"] * sums[:, -1])[:, None]).sum(1).clamp_(max=n - 1)
    pick = torch.where(greedy, best[stop], pick)
    tokens = torch.where(row < stop[seq], ids, torch.where(row == stop[seq], pick[seq], -1))
    logprobs = torch.where(tokens >= 0, p.gather(1, tokens.clamp(min=0)[:, None])[:, 0].log(), 0.0)
    return {"accepted": (stop - start[:-1]).int(), "tokens": tokens.int(), "logprobs": logprobs.float()}


# ---- work ----------------------------------------------------------------------

def _seen(case, rows, length):
    """(keys that some row sees, pairs of row and key that are seen) of one sequence."""
    keys = pairs = 0
    w, sinks = case["window"] or length + 1, case["sinks"]
    first = length - rows
    lo = max(0, first - w + 1)
    keys = length - lo + min(sinks, lo)
    for pos in range(first, length):
        a = max(0, pos - w + 1)
        pairs += pos + 1 - a + min(sinks, a)
    return keys, pairs


def work(case):
    if case["kind"] == "verify":
        rows = case["seqs"] + sum(_drafts(case))
        z = rows * case["vocab"] * SIZES[case["z"]]
        # the drafts' rows too, where there is a draft model
        both = z + (z - case["seqs"] * case["vocab"] * SIZES[case["z"]] if case["draft"] else 0)
        return {"bytes": both + rows * 24, "flops": 4 * both / SIZES[case["z"]]}
    rows, length = _lengths(case)
    d, kv, heads, n = case["dim"], case["kv_heads"], case["heads"], sum(rows)
    element = 2 * kv * d * SIZES[case["cache"]] + (8 * kv if case["cache"] == "e4m3" else 0)
    if case["kind"] == "store":
        own_reads = n * 2 * kv * d * 2 if case["cache"] == "e4m3" else 0     # the values handed back
        return {"bytes": n * ((2 * heads + 2 * kv) * d * SIZES[case["x"]] + element * (2 if case["cache"] == "e4m3" else 1)) + own_reads,
                "flops": 10 * n * (heads + 2 * kv) * d}
    seen = [_seen(case, r, length[s]) for s, r in enumerate(rows)]
    return {"bytes": sum(s[0] for s in seen) * element + 2 * n * heads * d * SIZES[case["x"]] + 4 * n * heads,
            "flops": 4 * heads * d * sum(s[1] for s in seen)}


# ---- the definition in 64 bits ---------------------------------------------------

def exact(case, seed):
    t = _inputs(case, seed)
    return {"store": _exact_store, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]](case, t)


def _exact_8_bits(r):
    """What a row keeps in e4m3 with a power-of-two scale: the nearest of the format's values, by a table of them."""
    grid = torch.tensor(sorted({m / 8 * 2.0 ** -6 for m in range(8)} | {(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)} - {480.0}),
                        dtype=torch.float64, device=DEV)
    top = r.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448)).clamp_(min=-126)
    e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e).clamp_(min=-126)
    e = torch.where(top > 0, e, -126.0)
    a = (r / torch.exp2(e)).abs()
    hi = torch.searchsorted(grid, a.contiguous()).clamp_(max=grid.numel() - 1)
    lo = (hi - 1).clamp_(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    take = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return grid[take] * torch.sign(r) * torch.exp2(e)


def _exact_store(case, t):
    d, kv, heads, page = case["dim"], case["kv_heads"], case["heads"], case["page"]
    out = {"q": [], "k": [], "v": []}
    pools = {name: t[name].double() for name in ("k", "v")} if case["cache"] != "e4m3" else None
    freq = torch.exp(-math.log(THETA) * torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    at = 0
    for s, n in enumerate(t["rows"]):
        x = t["x"][at:at + n].double().view(n, -1, d)
        at += n
        pos = torch.arange(t["length"][s] - n, t["length"][s], device=DEV)
        turn = torch.polar(torch.ones(n, d // 2, dtype=torch.float64, device=DEV), pos.double()[:, None] * freq)[:, None]

        def norm_turn(y, weight):
            y = y * weight.double() * torch.rsqrt(y.square().mean(2, keepdim=True) + EPS)
            y = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
            return torch.cat([y.real, y.imag], 2)
        q, k, v = norm_turn(x[:, :heads], t["q_norm"]), norm_turn(x[:, heads:heads + kv], t["k_norm"]), x[:, heads + kv:]
        out["q"].append(q.reshape(n, -1))
        for name, r in (("k", k), ("v", v)):
            if pools:
                pools[name][t["table"][s].long()[pos // page], pos % page] = r
            else:
                out[name].append(_exact_8_bits(r).reshape(n, -1))
    return {name: pools[name] if pools and name != "q" else torch.cat(out[name]) for name in out}


def _exact_attention(case, t):
    d, kv, heads, page = case["dim"], case["kv_heads"], case["heads"], case["page"]
    outs, lses, at = [], [], 0
    for s, n in enumerate(t["rows"]):
        length = t["length"][s]
        pages = t["table"][s, :-(-length // page)].long()
        k, v = (t[name][pages].reshape(-1, kv, d)[:length].double() for name in ("k", "v"))
        if case["cache"] == "e4m3":
            k, v = (y * t[name][pages].reshape(-1, kv)[:length, :, None].double() for y, name in ((k, "k_scale"), (v, "v_scale")))
        q = t["q"][at:at + n].double().view(n, heads, d)
        at += n
        pos = torch.arange(length - n, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)[None]
        hidden = j > pos
        if case["window"]:
            hidden |= (j <= pos - case["window"]) & (j >= case["sinks"])
        o, l = [], []
        for h in range(heads):
            z = (q[:, h] @ k[:, h * kv // heads].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            l.append(torch.logsumexp(z, 1))
            o.append(torch.exp(z - l[-1][:, None]) @ v[:, h * kv // heads])
        outs.append(torch.stack(o, 1).reshape(n, -1))
        lses.append(torch.stack(l, 1))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_verify(case, t):
    accepted, tokens, logprobs = [], [], []
    start, heats = t["start"].tolist(), t["temperature"].tolist()
    for s in range(case["seqs"]):
        greedy = heats[s] == 0
        heat = t["temperature"][s].double() if not greedy else 1.0
        r, done = start[s], False
        while not done:
            lp = torch.log_softmax(t["z"][r].double() / heat, 0)
            last, d = r == start[s + 1] - 1, int(t["ids"][r])
            lq = torch.log_softmax(t["y"][r].double() / heat, 0) if case["draft"] else None
            if greedy:
                token = int(torch.nonzero(t["z"][r] == t["z"][r].max())[0])
                done = last or token != d
            elif not last and t["u"][r] * (torch.exp(lq[d]) if case["draft"] else 1.0) < torch.exp(lp[d]):
                token = d
            else:
                done = True
                w = torch.exp(lp)
                if not last and case["draft"]:
                    w = torch.relu(w - torch.exp(lq))
                elif not last:
                    w[d] = 0
                c = w.cumsum(0)
                token = min(int(torch.searchsorted(c, t["v"][s] * c[-1], right=True)), case["vocab"] - 1)
            tokens.append(token)
            logprobs.append(lp[token])
            r += 1
        accepted.append(r - 1 - start[s])
        rest = start[s + 1] - r
        tokens += [-1] * rest
        logprobs += [torch.zeros((), dtype=torch.float64, device=DEV)] * rest
    return {"accepted": torch.tensor(accepted, dtype=torch.int32, device=DEV), "tokens": torch.tensor(tokens, dtype=torch.int32, device=DEV),
            "logprobs": torch.stack(logprobs)}
