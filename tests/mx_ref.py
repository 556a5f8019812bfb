"""MXFP4 quantisation, products and log probabilities in 64 bits (numpy), and
the error that the library's formats allow."""
import numpy as np
import torch

from gemma_amd import capi

TYPES = {"f32": (capi.GG_TYPE_F32, torch.float32), "f16": (capi.GG_TYPE_F16, torch.float16),
         "bf16": (capi.GG_TYPE_BF16, torch.bfloat16)}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}   # half a step of the smallest values
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantised(x):
    """The values that MXFP4 keeps of the rows of x (float64 [rows, k])."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    nb = -(-k // 32)
    b = np.zeros((rows, nb * 32))
    b[:, :k] = x
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(2)
    top = np.where(np.isfinite(b), np.abs(b), 0).max(2)
    e = np.where(top > 0, np.frexp(top)[1] - 3, -127).clip(-127, 127)
    a = np.abs(b) / np.exp2(e.astype(np.float64))[:, :, None]
    hi = np.searchsorted(GRID, np.where(np.isfinite(a), a, 0), side="left").clip(1, 7)
    up, down = GRID[hi], GRID[hi - 1]
    take_up = (a - down > up - a) | ((a - down == up - a) & (hi % 2 == 0))   # a tie goes to the even code
    q = np.where(take_up, up, down) * np.sign(np.where(np.isfinite(b), b, 0)) * np.exp2(e.astype(np.float64))[:, :, None]
    q[bad] = np.nan
    return q.reshape(rows, -1)[:, :k]


def parts(x_type, y_type):
    """5-bit parts that the product takes of x (None: x is packed)."""
    if y_type == "bf16":
        return 3
    if y_type == "f16":
        return 3 if x_type == "bf16" else 4
    return 5


def product_bound(x, w, y, x_type, y_type):
    """Largest error of each element of x w^T computed as y (float64):
    - of a block of x the parts keep 2^-(5 parts - 1) of the power of two at or below its maximum;
    - each 64-deep matrix instruction adds its products to the sum with an error of at most 2^-20 of its largest
      term for the products and 2^-23 of the sum for the running total;
    - one rounding to the result's type."""
    n, (m, k) = 1 if x_type is None else parts(x_type, y_type), x.shape
    mags = np.abs(x) @ np.abs(w).T
    bound = (2.0 ** -20 + (-(-k // 64) * n + 8) * 2.0 ** -23) * mags
    if x_type is not None:
        nb = -(-k // 32)
        b = np.zeros((m, nb * 32))
        b[:, :k] = np.abs(x)
        top = np.repeat(b.reshape(m, nb, 32).max(2), 32, axis=1)[:, :k]
        bound += 2.0 ** (1 - 5 * n) * (np.maximum(top, 2.0 ** -106) @ np.abs(w).T)
    return bound + HALF_STEP[y_type] * (np.abs(y) + bound) + LEAST[y_type]


def scores(z, top):
    """lse, entropy, log probabilities and the best ids of rows of z (float64; finite or -inf, a value in each row)."""
    m = z.max(1, keepdims=True)
    p = np.exp(z - m)
    s = p.sum(1, keepdims=True)
    d = np.where(p > 0, z - m, 0)
    lp = z - m - np.log(s)
    order = np.argsort(-z, axis=1, kind="stable")[:, :top]
    return (m + np.log(s))[:, 0], (np.log(s) - (p * d).sum(1, keepdims=True) / s)[:, 0], lp, order


def score_rel(n):
    """Relative error of the sums: 32 adds in a tile, one a tile, 10 joining threads and chunks, each 2^-24; the
    exponential's argument and value another 2^-21."""
    return (32 + (n + 8191) // 8192 + 10) * 2.0 ** -24 + 2.0 ** -21
