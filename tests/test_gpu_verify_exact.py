"""Verification of drafted tokens where decisions are close: next to the border
of acceptance, draws from a draft model's row next to the target's, and the
ends of the range of temperatures."""
import numpy as np
import pytest
import torch

from gpu_util import say
from kv_ref import verify
from test_gpu_verify import run

pytestmark = pytest.mark.gpu


def soft(z, heat):
    """softmax(z / heat), f64, without an infinity times zero."""
    with np.errstate(over="ignore"):
        w = np.where(np.isneginf(z), 0.0, np.exp((np.where(np.isneginf(z), 0.0, z) - z.max()) / heat))
    return w / w.sum()


@pytest.mark.parametrize("with_y", [True, False])
@pytest.mark.parametrize("n,seqs", [(1000, 40), (50257, 24), (262144, 8), (262144, 40)])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_drafts_next_to_the_border(gpu, name, n, seqs, with_y):
    """u q(d) is p(d) but for one part in 10^10: f64 sums of some 10^5 weights are off by 10^-13 of it at most, f32 ones by 10^-7."""
    say("border", name, n, seqs, with_y)
    rng = np.random.default_rng(n + seqs)
    z = rng.standard_normal((2 * seqs, n)) * 3
    y = z + rng.standard_normal((2 * seqs, n))
    z, y = (torch.from_numpy(t).to(dict(f32=torch.float32, bf16=torch.bfloat16)[name]).double().numpy() for t in (z, y))
    heat = rng.choice([0.5, 1.0, 1.7], seqs).astype(np.float32)
    draft, u = np.zeros(2 * seqs, int), np.zeros(2 * seqs)
    stands = np.arange(seqs) % 2 == 0
    for s in range(seqs):
        p, q = soft(z[2 * s], float(heat[s])), soft(y[2 * s], float(heat[s]))
        d = int(np.argmax(np.where(p < q, p, 0))) if with_y else int(rng.choice(n, p=p))
        draft[2 * s] = d
        u[2 * s] = p[d] / (q[d] if with_y else 1.0) * (1 - 1e-10 if stands[s] else 1 + 1e-10)
    start = np.arange(0, 2 * seqs + 1, 2)
    v = rng.random(seqs)
    acc, tok, lp, _, _ = run(z, y if with_y else None, draft, start, heat, u, v, name)
    assert np.array_equal(acc, stands.astype(int))
    ra, rt, rl, margin = verify(z, y if with_y else None, draft, start, heat, u, v)
    assert (margin > 1e-11).all() and np.array_equal(tok, rt)


@pytest.mark.parametrize("n", [4096, 50000, 262144])
def test_a_draft_model_next_to_the_target(gpu, n):
    """The target is the draft model's row but for two tokens: d's probability is gone and a rises by a part of it. All others then
    have p above q by the rest, some 10^-9 of their own: less than f32 sums tell, and half of what the draw is from."""
    seqs = 64
    rng = np.random.default_rng(n)
    y = (rng.standard_normal((2 * seqs, n))).astype(np.float32)
    z = y.copy()
    d, a = n // 3, n // 2
    for s in range(seqs):
        r = 2 * s
        w = np.exp(y[r].astype(np.float64) - y[r].max())
        small = 2.0 ** -28 * w.sum()
        y[r, d] = np.float32(np.log(2 * small) + y[r].max())
        z[r] = y[r]
        z[r, d] = -np.inf
        z[r, a] = np.float32(np.log(np.exp(np.float64(y[r, a]) - y[r].max()) + small) + y[r].max())
    draft = np.full(2 * seqs, d)
    start = np.arange(0, 2 * seqs + 1, 2)
    u, v, heat = np.full(2 * seqs, 0.5), (np.arange(seqs) + 0.5) / seqs, np.ones(seqs, np.float32)
    z64, y64 = z.astype(np.float64), y.astype(np.float64)
    p, q = soft(z64[0], 1.0), soft(y64[0], 1.0)
    rest = np.maximum(p - q, 0)
    assert 0.2 < rest[a] / rest.sum() < 0.8 and (rest > 0).sum() > n // 2     # that is what the inputs are
    acc, tok, lp, _, _ = run(z64, y64, draft, start, heat, u, v)
    ra, rt, rl, margin = verify(z64, y64, draft, start, heat, u, v)
    assert (acc == 0).all()
    # p - q is 2^-28 of either, in f64 off by 2^-50 of them: borders within 10^-6 of the whole may fall either way
    clear = margin > 1e-6
    say("next to the target", n, int(clear.sum()))
    for s in range(seqs):
        res = np.maximum(soft(z64[2 * s], 1.0) - soft(y64[2 * s], 1.0), 0)
        c = np.cumsum(res)
        lo, hi = (int(np.searchsorted(c, (v[s] + e) * c[-1], side="right")) for e in (-1e-6, 1e-6))
        assert lo <= tok[2 * s] <= hi and res[tok[2 * s]] > 0, (s, tok[2 * s], rt[2 * s], lo, hi)
        assert tok[2 * s + 1] == -1


@pytest.mark.parametrize("heat", [1.0, 0.7])
@pytest.mark.parametrize("n", [7, 37, 500, 5000, 70000])
def test_a_draft_model_that_differs_by_roundings(gpu, n, heat):
    """y is z but for the last bits of some logits, and the draft has no probability under either: p - q is some 2^-24 of them, about what
    f32 sums are off by, and which tokens have any of it is decided by that."""
    say("roundings", n, heat)
    seqs = 64
    rng = np.random.default_rng(n)
    z = (rng.standard_normal((2 * seqs, n)) * 2).astype(np.float32)
    if n > 7:
        z[:, rng.random(n) < 0.3] = -np.inf
    z[:, 0] = -np.inf
    z[:, n - 1] = 0.5
    y = z.copy()
    change = rng.random(y.shape) < 0.4
    y[change] = np.nextafter(y[change], np.where(rng.random(change.sum()) < 0.5, np.float32(10), np.float32(-10)))
    y[:, 0] = -np.inf
    y[:, n - 1] = np.nextafter(np.float32(0.5), np.float32(1))
    start = np.arange(0, 2 * seqs + 1, 2)
    T = float(np.float32(heat))
    v = rng.random(seqs)
    z64, y64 = z.astype(np.float64), y.astype(np.float64)
    acc, tok, lp, _, _ = run(z64, y64, np.zeros(2 * seqs, int), start, np.full(seqs, T), np.full(2 * seqs, 0.5), v)
    assert (acc == 0).all()
    for s in range(seqs):
        r, t = 2 * s, tok[2 * s]
        assert np.isfinite(z[r, t]) and np.isfinite(lp[r])
        res = np.maximum(soft(z64[r], T) - soft(y64[r], T), 0)
        c = np.cumsum(res)
        # f64 leaves 2^-50 of p and q: 2^-22 of what is left, in all of its tokens at once
        lo, hi = (int(np.searchsorted(c, (v[s] + e) * c[-1], side="right")) for e in (-2e-6, 2e-6))
        assert lo <= t <= min(hi, n - 1) and res[t] > 0, (s, t, lo, hi, res[t] / c[-1])


@pytest.mark.parametrize("with_y", [True, False])
@pytest.mark.parametrize("n", [50, 20000])
@pytest.mark.parametrize("heat,scale", [(np.inf, 1.0), (3e38, 1e38), (1e30, 1e29), (2.0 ** 64, 1e19), (2.0 ** -126, 2.0 ** -126), (1e-30, 1e-30),
                                        (1e-40, 1.0), (1e-45, 1.0)])
def test_ends_of_the_range_of_temperatures(gpu, heat, scale, n, with_y):
    """Any temperature above 0 gives the formula's probabilities (one below 2^-126 those of 2^-126), masked logits among them 0."""
    say("temperature", heat, scale, n, with_y)
    seqs = 20
    rng = np.random.default_rng(n)
    heat32 = np.float32(heat)
    assert heat32 > 0
    z = rng.uniform(-3, 3, (2 * seqs, n)) * scale
    y = z + rng.uniform(-1, 0, (2 * seqs, n)) * scale * 0.3
    z, y = np.clip(z, -3.4e38, 3.4e38).astype(np.float32), np.clip(y, -3.4e38, 3.4e38).astype(np.float32)
    z[:, rng.random(n) < 0.3] = -np.inf
    z[:, 0], y[:, 1] = -np.inf, -np.inf
    z[:, 2] = scale
    start = np.arange(0, 2 * seqs + 1, 2)
    z64, y64 = z.astype(np.float64), y.astype(np.float64)
    T = max(float(heat32), 2.0 ** -126)
    T = 1e300 if np.isinf(T) else T               # flat to the last bit
    draft = np.array([int(rng.choice(n, p=soft((y64 if with_y else z64)[r], T))) for r in range(2 * seqs)])
    u, v = rng.random(2 * seqs), rng.random(seqs)
    u[:seqs] *= 1e-3                              # some stand without y too
    acc, tok, lp, _, _ = run(z64, y64 if with_y else None, draft, start, np.full(seqs, heat32), u, v)
    with np.errstate(over="ignore", invalid="ignore"):
        ra, rt, rl, margin = verify(z64, y64 if with_y else None, draft, start, np.full(seqs, T), u, v)
    clear = margin > 1e-9
    rows = np.repeat(clear, 2)
    assert clear.sum() >= seqs - 2
    assert np.array_equal(acc[clear], ra[clear]) and np.array_equal(tok[rows], rt[rows])
    assert (np.abs(lp[rows] - rl[rows]) <= 40 * 2.0 ** -22 + 2.0 ** -22 * np.abs(rl[rows])).all()
    assert not np.isnan(lp).any()
