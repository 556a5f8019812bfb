"""Verification of drafted tokens where decisions are close: next to the border
of acceptance, and at the ends of the range of temperatures."""
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
