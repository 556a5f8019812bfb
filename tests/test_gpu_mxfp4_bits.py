"""Products of MXFP4 weights use every bit of x: rows whose large elements meet
zero weights, and weights that pick out single elements."""
import numpy as np
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from mx_ref import HALF_STEP, LEAST, TYPES, quantised

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def product(w, x, x_name, y_name):
    """x w^T through the library: the kept x, the kept w and y, in 64 bits."""
    (n, k), m = w.shape, x.shape[0]
    s = stream()
    wd = torch.from_numpy(np.ascontiguousarray(w, np.float32)).to(DEV)
    wp = torch.empty(capi.mxfp4_packed_size(n, k), dtype=torch.uint8, device=DEV)
    capi.mxfp4_quantize(wd.data_ptr(), capi.GG_TYPE_F32, n, k, k, wp.data_ptr(), s)
    xd = torch.from_numpy(x).to(TYPES[x_name][1]).to(DEV)
    y = torch.full((m, n), 55.0, dtype=TYPES[y_name][1], device=DEV)
    xt = TYPES[x_name][0]
    ws = torch.full((max(capi.mxfp4_linear_workspace_size(xt, m, n, k), 16),), 255, dtype=torch.uint8, device=DEV)
    capi.mxfp4_linear(wp.data_ptr(), xd.data_ptr(), xt, k, y.data_ptr(), TYPES[y_name][0], n, m, n, k, ws.data_ptr(), s)
    torch.cuda.synchronize()
    return xd.double().cpu().numpy(), quantised(wd.double().cpu().numpy()), y.double().cpu().numpy()


def sums_bound(x, w, y, y_name):
    """f32 sums of at most three terms an element of x, in any order: an add errs by at most 2^-23 of what it adds up,
    here taken as the sum of all magnitudes each time; then one rounding to the result's type."""
    bound = (3 * x.shape[1] + 8) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    return bound + HALF_STEP[y_name] * (np.abs(y) + bound) + LEAST[y_name]


@pytest.mark.parametrize("y_name", list(TYPES))
@pytest.mark.parametrize("x_name,up", [("f32", 10), ("f32", 13), ("f32", 30), ("f32", 90), ("bf16", 10), ("bf16", 13),
                                       ("bf16", 30), ("bf16", 90), ("f16", 10), ("f16", 13)])
@pytest.mark.parametrize("m,n,k", [(1, 48, 96), (3, 130, 64), (9, 100, 200), (70, 300, 96), (200, 1000, 130)])
def test_large_elements_at_zero_weights(gpu, m, n, k, x_name, up, y_name):
    """Channels 2^up times as large as the others whose weights are zero: they add nothing, their neighbours all they have."""
    say("zero weights", m, n, k, x_name, up, y_name)
    rng = np.random.default_rng(m + 7 * n + 31 * k + up)
    x = rng.uniform(-2, 2, (m, k))
    w = rng.standard_normal((n, k)) * 0.05
    big = np.arange(5, k, 32)
    x[:, big] *= 2.0 ** up
    w[:, big] = 0
    x, w, y = product(w, x, x_name, y_name)
    want = x @ w.T
    assert (np.abs(y - want) <= sums_bound(x, w, want, y_name)).all()


@pytest.mark.parametrize("y_name", list(TYPES))
@pytest.mark.parametrize("x_name", list(TYPES))
@pytest.mark.parametrize("m,k", [(1, 64), (4, 100), (5, 130), (40, 128), (90, 257)])
def test_weights_that_pick_single_elements(gpu, m, k, x_name, y_name):
    """W the unit matrix: y is x, rounded to y's type and nothing else, whatever lies beside it in the row."""
    say("unit matrix", m, k, x_name, y_name)
    rng = np.random.default_rng(m * k)
    least, most = {"f32": (-100, 120), "bf16": (-100, 120), "f16": (-14, 14)}[x_name]
    x = rng.uniform(1, 2, (m, k)) * np.exp2(rng.integers(least, most, (m, k)).astype(np.float64)) * rng.choice([-1, 1], (m, k))
    x[:, ::7] = 0
    x, w, y = product(np.eye(k), x, x_name, y_name)
    assert np.array_equal(w, np.eye(k))
    with np.errstate(over="ignore"):
        want = torch.from_numpy(x).to(torch.float32).to(TYPES[y_name][1]).double().numpy()
    assert np.array_equal(y, want)


@pytest.mark.parametrize("x_name", list(TYPES))
@pytest.mark.parametrize("m", [2, 40])
def test_ends_of_the_types(gpu, m, x_name):
    """The largest values, the smallest normal ones and denormals, alone and beside each other."""
    t = torch.finfo(TYPES[x_name][1])
    least = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[x_name]
    vals = np.array([t.max, -t.max, t.max * (1 - t.eps), t.tiny, -t.tiny, t.tiny * (2 - t.eps), least, -5 * least, 101 * least,
                     t.tiny - least, 0.0, 1.0, 1 + t.eps, 2.0 ** -20])
    k = 70
    x = vals[np.random.default_rng(m).integers(0, len(vals), (m, k))]
    x, w, y = product(np.eye(k), x, x_name, "f32")
    say("ends", m, x_name)
    # below 2^-110 an f32 has bits under 2^-133, which are cut off
    loss = np.where((np.abs(x) < 2.0 ** -110) & (x_name == "f32"), 2.0 ** -133, 0.0)
    assert (np.abs(y - x) <= loss).all()


@pytest.mark.parametrize("byte", [0, 1, 2, 3, 100, 251, 252])
@pytest.mark.parametrize("x_name,x_exp", [("f32", 0), ("bf16", 0), ("f16", 0), ("f32", 100), ("bf16", -126)])
@pytest.mark.parametrize("m", [1, 33])
def test_every_weight_scale(gpu, m, x_name, x_exp, byte):
    """Weights from the smallest block to the largest: each element alone, times a power of two."""
    say("scales", m, x_name, x_exp, byte)
    k = 32
    w = np.zeros((15, k))
    grid = np.array([0.5, 1, 1.5, 2, 3, 4, 6])
    unit = 2.0 ** (byte - 127)
    w[:7, 3], w[7:14, 9] = grid, -grid
    w *= unit
    w[:, 20] = 4 * unit                      # the block's largest: its scale is `unit`
    x = np.zeros((m, k))
    x[:, 3] = 2.0 ** x_exp
    x[:, 9] = 2.0 ** x_exp
    x, w, y = product(w, x, x_name, "f32")
    with np.errstate(over="ignore"):
        want = (x @ w.T).astype(np.float32).astype(np.float64)
    assert np.array_equal(y, want)


@pytest.mark.parametrize("x_name", list(TYPES))
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("m", [3, 50])
def test_infinities_and_nans_of_each_type(gpu, m, bad, x_name):
    """A row of x with one is NaN throughout, also where the weight there is zero; the others keep their values."""
    say("inf and nan", m, bad, x_name)
    n, k = 70, 100
    rng = np.random.default_rng(m)
    x, w = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    x[1, 41] = bad
    w[::2, 41] = 0
    x, w, y = product(w, x, x_name, "f32")
    assert np.isnan(y[1]).all()
    rest = np.arange(m) != 1
    want = x[rest] @ w.T
    assert (np.abs(y[rest] - want) <= sums_bound(x[rest], w, want, "f32")).all()
