"""K/V pages, attention over them and verification of drafts in 64 bits (numpy),
a pool of pages with anything in between, and the errors that the library's
formats allow."""
import numpy as np
import torch

from gemma_amd import capi

TYPES = {"f32": (capi.GG_TYPE_F32, torch.float32), "f16": (capi.GG_TYPE_F16, torch.float16),
         "bf16": (capi.GG_TYPE_BF16, torch.bfloat16), "e4m3": (capi.GG_TYPE_E4M3, torch.float8_e4m3fn)}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}   # half a step of the smallest values


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda:0")


def typed(values, name):
    """float64 numpy -> a device tensor of the type, and the values it keeps."""
    t = torch.from_numpy(np.ascontiguousarray(values, np.float64)).to("cuda:0").to(TYPES[name][1])
    return t, t.double().cpu().numpy()


class Pool:
    """Pages for sequences of the given lengths, in shuffled order, with pages that belong to nobody. Everything that
    is not written holds NaN (bits all ones in 8 bits). `layout`: "phd" [page][place][head], "hpd" [page][head][place],
    "both" K and V rows side by side, "pad" with gaps."""

    def __init__(self, lengths, page, n_kv, dim, cache, seed=0, layout="phd", spare=3, extra_columns=0):
        rng = np.random.default_rng(seed)
        self.page, self.n_kv, self.dim, self.cache, self.layout = page, n_kv, dim, cache, layout
        need = [-(-n // page) for n in lengths]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lengths), max(max(need), 1) + extra_columns), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        d = dim
        if layout == "phd":
            self.strides = (page * n_kv * d, n_kv * d, d)
        elif layout == "hpd":
            self.strides = (page * n_kv * d, d, page * d)
        elif layout == "both":
            self.strides = (page * n_kv * 2 * d, n_kv * 2 * d, 2 * d)
        else:
            self.strides = (page * (n_kv * (d + 16) + 32) + 48, n_kv * (d + 16) + 32, d + 16)
        ps, os, hs = self.strides
        size = (self.n_pages - 1) * ps + (page - 1) * os + (n_kv - 1) * hs + d
        self.size = size + (d if layout == "both" else 0)
        code = {"bf16": torch.bfloat16, "f16": torch.float16}.get(cache)
        if cache == "e4m3":
            self.buf = [torch.full((self.size,), 255, dtype=torch.uint8, device="cuda:0") for _ in range(1 if layout == "both" else 2)]
        else:
            self.buf = [torch.full((self.size,), float("nan"), dtype=code, device="cuda:0") for _ in range(1 if layout == "both" else 2)]
        es = self.buf[0].element_size()
        self.k_ptr = self.buf[0].data_ptr()
        self.v_ptr = self.buf[0].data_ptr() + d * es if layout == "both" else self.buf[1].data_ptr()
        self.scales = [torch.full((self.n_pages, page, n_kv), float("nan"), device="cuda:0") for _ in range(2)] if cache == "e4m3" else None
        self.table_dev = i32(self.table)

    def pages(self, **change):
        sc = [t.data_ptr() for t in self.scales] if self.scales else [None, None]
        p = capi.kv_pages(self.k_ptr, self.v_ptr, TYPES[self.cache][0], self.n_pages, self.page, self.n_kv, self.dim, *self.strides,
                          k_scale=sc[0], v_scale=sc[1])
        for name, value in change.items():
            setattr(p, name, value)
        return p

    def views(self):
        """K and V as [page, place, head, dim] of the stored type."""
        ps, os, hs = self.strides
        out = []
        for i in range(2):
            b = self.buf[0] if self.layout == "both" else self.buf[i]
            out.append(torch.as_strided(b, (self.n_pages, self.page, self.n_kv, self.dim), (ps, os, hs, 1),
                                        self.dim if self.layout == "both" and i else 0))
        return out

    def put(self, seq, k, v, scale_exponents=None):
        """Rows k, v [len, n_kv, dim] (float64) of a sequence from position 0 on -> the values kept."""
        n = len(k)
        pos = np.arange(n)
        pg, pl = torch.from_numpy(self.table[seq, pos // self.page].astype(np.int64)).cuda(), torch.from_numpy(pos % self.page).cuda()
        kept = []
        for i, (view, x) in enumerate(zip(self.views(), (k, v))):
            x = torch.from_numpy(np.ascontiguousarray(x, np.float64)).cuda()
            if self.cache == "e4m3":
                e = torch.from_numpy(np.exp2(scale_exponents[i])).cuda()          # [n, n_kv]
                code = (x / e[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                view[pg, pl] = code.view(torch.uint8)
                self.scales[i][pg, pl] = e.float()
                kept.append((code.double() * e[:, :, None]).cpu().numpy())
            else:
                t = x.to(view.dtype)
                view[pg, pl] = t
                kept.append(t.double().cpu().numpy())
        return kept


def seqs_of(pool, rows, lengths, n_rows=None, max_len=None, max_rows=None, first=0):
    """(structure, what it points to) for sequences with `rows` new rows each; their rows begin at row `first`."""
    start = i32(np.concatenate([[0], np.cumsum(rows)]) + first)
    length = i32(lengths)
    s = capi.kv_seqs(start.data_ptr(), length.data_ptr(), pool.table_dev.data_ptr(), len(rows), n_rows or sum(rows) + first,
                     max_rows or max(max(rows), 1), max_len or max(max(lengths), 1), pool.table.shape[1])
    return s, (start, length)


def sees(pos, key, window, sinks):
    """[rows, keys]"""
    pos, key = np.asarray(pos)[:, None], np.asarray(key)[None]
    ok = key <= pos
    if window:
        ok &= (key > pos - window) | (key < sinks)
    return ok


WEIGHT_BITS = {("bf16", "f32"): 2.0 ** -24, ("bf16", "bf16"): 2.0 ** -8, ("bf16", "f16"): 2.0 ** -16,
               ("e4m3", "f32"): 2.0 ** -24, ("e4m3", "bf16"): 2.0 ** -8, ("e4m3", "f16"): 2.0 ** -16, ("f16", "f16"): 2.0 ** -11}


def attention(q, k, v, pos, scale, window, sinks, cache, x):
    """One head: q [rows, d], k and v [keys, d] -> out, lse and their bounds.

    A score is a sum of d products in f32 (24 steps at most, each off by 2^-24 of the sum of magnitudes, or twice that
    where an instruction cuts), times the scale; the difference to the reference and 2^x add 2^-22 of the score and
    2^-22. Weights keep WEIGHT_BITS; a row's sums take a step for 32 or more keys of a wave, and 32 more where waves and chunks
    are joined. All of it counts for the numerator and for the sum that it is divided by."""
    ok = sees(pos, np.arange(len(k)), window, sinks)
    kk, vv = np.where(np.isfinite(k), k, 0), np.where(np.isfinite(v), v, 0)
    s = np.where(ok, scale * (q @ kk.T), -np.inf)
    m = s.max(1, initial=-np.inf, keepdims=True)
    m = np.where(np.isfinite(m), m, 0)
    w = np.exp(s - m)
    total = w.sum(1, keepdims=True)
    some = total[:, 0] > 0
    p = w / np.where(total > 0, total, 1)
    out = p @ vv
    with np.errstate(divide="ignore"):
        lse = m[:, 0] + np.log(total[:, 0])
    size = np.where(ok, abs(scale) * (np.abs(q) @ np.abs(kk).T), 0).max(1, initial=0)
    d_score = size * 48 * 2.0 ** -24 + np.where(ok, np.abs(np.where(ok, s, 0)), 0).max(1, initial=0) * 2.0 ** -21 + 2.0 ** -21
    sums = (len(k) / 32 + 32) * 2.0 ** -24
    bound = (p @ np.abs(vv)) * (2 * d_score + 2 * WEIGHT_BITS[cache, x] + 2 * sums)[:, None] + np.abs(out) * HALF_STEP[x] + LEAST[x]
    lse_bound = d_score + sums + 2.0 ** -22 * (1 + np.abs(np.where(some, lse, 0)) + np.abs(m[:, 0]))
    return out, lse, bound, lse_bound


def e4m3_row(r):
    """Rows [.., d] -> the values kept with the least power-of-two scale that holds them (float64)."""
    grid = np.array(sorted({i / 8 * 2.0 ** -6 for i in range(8)} | {(1 + i / 8) * 2.0 ** e for e in range(-6, 9) for i in range(8)} - {480.0}))
    top = np.abs(r).max(-1, keepdims=True)
    e = np.full(top.shape, -126.0)
    for step in range(-126, 121):
        e = np.where(top > 448 * 2.0 ** (step - 1), np.maximum(step, -126), e) if step > -126 else e
    a = np.abs(r) / np.exp2(e)
    hi = np.searchsorted(grid, a).clip(0, len(grid) - 1)
    lo = (hi - 1).clip(0)
    take = np.where((grid[hi] - a < a - grid[lo]) | ((grid[hi] - a == a - grid[lo]) & (hi % 2 == 0)), hi, lo)
    return grid[take] * np.sign(r) * np.exp2(e)


def norm_rope(x, weight, pos, eps, theta):
    """x [rows, heads, d] (float64) -> normed (weight None: not) and rotated (theta 0: not)."""
    d = x.shape[-1]
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    if theta:
        ang = np.asarray(pos, np.float64)[:, None] * theta ** (-2.0 * np.arange(d // 2) / d)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = x[..., :d // 2], x[..., d // 2:]
        x = np.concatenate([a * c - b * s, b * c + a * s], -1)
    return x


def verify(z, y, draft, start, heat, u, v):
    """-> accepted, tokens, logprobs, margins: how far (relative) each decision of a sequence was from the other one."""
    rows, n = z.shape
    acc, tokens, lps, margins = [], np.full(rows, -1), np.zeros(rows), []
    for s in range(len(start) - 1):
        margin, count = np.inf, 0
        for r in range(start[s], start[s + 1]):
            last = r == start[s + 1] - 1
            g = not heat[s] > 0
            T = 1.0 if g else float(heat[s])
            bad = not (z[r] < np.inf).all() or z[r].max() == -np.inf
            if y is not None and not last and not g:
                bad |= not (y[r] < np.inf).all() or y[r].max() == -np.inf
            if bad:
                tokens[r], lps[r] = -1, np.nan
                break
            w = np.exp((z[r] - z[r].max()) / T)
            p = w / w.sum()
            d = int(draft[r]) if not last else -1
            real = 0 <= d < n
            if g:
                best = int(np.argmax(z[r]))
                tokens[r] = best
                stands = d == best
            else:
                q = None
                if y is not None and not last:
                    q = np.exp((y[r] - y[r].max()) / T)
                    q = q / q.sum()
                qd = 1.0 if q is None else (q[d] if real else 0.0)
                stands = real and not last and u[r] * qd < p[d]
                if real and not last:
                    margin = min(margin, abs(u[r] * qd - p[d]) / max(p[d], 1e-300))
                if not stands:
                    res = p.copy()
                    if not last and q is not None:
                        res = np.maximum(p - q, 0)
                    elif not last and real:
                        res[d] = 0
                    if not res.sum() > 0:
                        res = p
                    c = np.cumsum(res)
                    t = v[s] * c[-1]
                    tokens[r] = min(int(np.searchsorted(c, t, side="right")), n - 1)
                    margin = min(margin, np.abs(c - t).min() / c[-1])
                else:
                    tokens[r] = d
            with np.errstate(divide="ignore"):
                lps[r] = np.log(p[tokens[r]])
            if not stands:
                break
            count += 1
        acc.append(count)
        margins.append(margin)
    return np.array(acc), tokens, lps, np.array(margins)
