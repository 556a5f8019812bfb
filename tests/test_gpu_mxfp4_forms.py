"""Every form of the MXFP4 product: tiles with and without slices of k for each
kind of x, column tiles and wave splits of the few-row kernel. Whole-number
operands whose sums f32 holds exactly, so that each result has one right value."""
import os
import subprocess

import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream
from mx_ref import TYPES

DEV = "cuda:0"
PARTS = {"mxfp4": 0, "bf16": 1, "f16": 2, "f32": 3}
# (x, rows, features, k): (tile, k in slices)
TILES = {
    ("mxfp4", 2277, 4487, 303): ("256x256", False), ("mxfp4", 1519, 1405, 9037): ("256x256", True),
    ("mxfp4", 1153, 771, 301): ("128x64", False), ("mxfp4", 683, 417, 5693): ("128x64", True),
    ("mxfp4", 23, 101, 311): ("128x32", False), ("mxfp4", 23, 103, 2867): ("128x32", True),
    ("bf16", 7009, 1583, 1601): ("256x256", False), ("bf16", 1805, 2209, 5179): ("256x256", True),
    ("bf16", 2723, 1041, 309): ("256x64", False), ("bf16", 1243, 797, 3759): ("256x64", True),
    ("bf16", 23, 103, 301): ("128x32", False), ("bf16", 23, 107, 1253): ("128x32", True),
    ("f16", 3839, 3115, 789): ("256x256", False), ("f16", 1953, 2151, 2809): ("256x256", True),
    ("f16", 2277, 1287, 313): ("256x64", False), ("f16", 1051, 911, 2061): ("256x64", True),
    ("f16", 25, 103, 303): ("128x32", False), ("f16", 23, 105, 581): ("128x32", True),
    ("f32", 3333, 3611, 519): ("256x256", False), ("f32", 1465, 2863, 2071): ("256x256", True),
    ("f32", 2487, 1155, 301): ("256x64", False), ("f32", 1671, 517, 1391): ("256x64", True),
    ("f32", 23, 103, 303): ("128x32", False), ("f32", 23, 101, 455): ("128x32", True),
}
# (x, rows, features, k): (column tiles, waves that share k)
FEW = {
    ("f32", 1, 33, 1153): (1, 8), ("f32", 5, 8100, 700): (1, 4), ("f32", 7, 14001, 515): (2, 2), ("f32", 10, 40003, 300): (2, 1),
    ("f32", 11, 101, 1700): (3, 8), ("f32", 16, 70001, 200): (3, 1), ("f32", 17, 515, 640): (4, 4), ("f32", 21, 16500, 130): (4, 1),
    ("f32", 21, 97, 900): (4, 8), ("f16", 1, 40, 9000): (1, 8), ("f16", 8, 50001, 129): (1, 1), ("f16", 9, 203, 513): (2, 4),
    ("f16", 16, 20005, 257): (2, 1), ("f16", 22, 66, 1500): (3, 8), ("f16", 22, 13001, 400): (3, 2), ("bf16", 1, 270001, 65): (1, 1),
    ("bf16", 2, 1001, 3001): (1, 8), ("bf16", 3, 7001, 515): (1, 4),
    ("bf16", 16, 9001, 777): (1, 2), ("bf16", 17, 129, 1030): (2, 8), ("bf16", 22, 60011, 333): (2, 1),
}
PLAN = r"""
#include <cstdio>
#include <cstdlib>
#include "gg_internal.h"
int main(int argc, char** argv) {
  const char* names[gg::MT_COUNT] = {"256x256", "256x64", "128x64", "128x32"};
  for (int i = 1; i + 3 < argc; i += 4) {
    const int parts = atoi(argv[i]);
    const long long m = atoll(argv[i + 1]), n = atoll(argv[i + 2]), k = atoll(argv[i + 3]);
    if (parts && gg::mx_gemv_fits(m, parts, k)) {
      printf("few %lld %d\n", (m * parts + 15) / 16, gg::mx_gemv_waves(n, k));
    } else {
      const gg::Mx4Plan p = gg::mx4_plan(parts == 0, parts ? parts : 1, m, n, k);
      printf("%s %d\n", names[p.tile], p.slices > 1);
    }
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The rules that pick a form, compiled for the host."""
    d = tmp_path_factory.mktemp("plan")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webgpu-gemma_amd", "csrc")
    (d / "plan.cpp").write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-D__host__=", "-D__device__=", "-I", csrc, str(d / "plan.cpp"), "-o", str(d / "plan")],
                   check=True)

    def forms(cases):
        args = [str(v) for x, m, n, k in cases for v in (PARTS[x], m, n, k)]
        return [line.split() for line in subprocess.run([str(d / "plan"), *args], check=True, capture_output=True,
                                                        text=True).stdout.splitlines()]
    return forms


def test_cases_reach_the_forms_they_are_listed_for(plan):
    assert plan(TILES) == [[t, str(int(s))] for t, s in TILES.values()]
    assert plan(FEW) == [["few", str(c), str(w)] for c, w in FEW.values()]


def test_cases_reach_every_form(plan):
    """What the rules pick over a grid of sizes is among the cases, for each kind of x."""
    sizes = [(m, n, k) for m in (1, 2, 4, 7, 11, 16, 19, 21, 22, 23, 40, 100, 300, 700, 1500, 4000, 9000)
             for n in (1, 40, 150, 500, 1500, 4000, 9000, 14000, 40000, 262144) for k in (1, 64, 130, 300, 700, 1500, 4000, 9000, 30000)]
    for x in PARTS:
        listed = {tuple(f) for f in plan([c for c in [*TILES, *FEW] if c[0] == x])}
        got = {tuple(f) for f in plan([(x, *s) for s in sizes])}
        tiles = {f for f in got if f[0] != "few"}
        assert tiles <= listed, (x, tiles - listed)
        columns, waves = {f[1] for f in got if f[0] == "few"}, {f[2] for f in got if f[0] == "few"}
        few = [f for f in listed if f[0] == "few"]
        assert columns <= {f[1] for f in few} and waves <= {f[2] for f in few}, (x, columns, waves)


def fourbit(gen, rows, k):
    """Values of the format, whole numbers up to 24: the elements times two, each 32 of them times 1 or 2."""
    grid = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=DEV)
    v = grid[torch.randint(0, 8, (rows, k), generator=gen, device=DEV)]
    v = v * (1 - 2 * torch.randint(0, 2, (rows, k), generator=gen, device=DEV))
    up = torch.randint(0, 2, (rows, -(-k // 32)), generator=gen, device=DEV) + 1
    return v * up.repeat_interleave(32, 1)[:, :k]


def operands(x_name, m, n, k):
    """x and w, in 64 bits. Of x, six values a row fill the type's bits, the others are -3 to 3: any sum is below 2^24."""
    gen = torch.Generator(device=DEV).manual_seed(m + 3 * n + 7 * k)
    w = fourbit(gen, n, k)
    if x_name == "mxfp4":
        return fourbit(gen, m, k) / 8, w            # up to 3, steps of 1/8: 16000 x 24 x 24 < 2^24
    x = torch.randint(-3, 4, (m, k), generator=gen, device=DEV).double()
    big = {"bf16": 2.0 ** 7 + 1, "f16": 2.0 ** 10 + 1, "f32": 2.0 ** 16 + 2.0 ** 8 + 1}[x_name]
    at = torch.randint(0, k, (m, 6), generator=gen, device=DEV)
    sign = 1 - 2 * torch.randint(0, 2, (m, 6), generator=gen, device=DEV).double()
    return x.scatter_(1, at, sign * big), w


def check(x_name, m, n, k, y_name, pad):
    say("form", x_name, m, n, k, y_name, pad)
    s = stream()
    x, w = operands(x_name, m, n, k)
    if y_name == "f16":
        x = x / 1024                                # results that f16 holds; exact, like every power of two
    wd = w.float()
    wp = torch.full((capi.mxfp4_packed_size(n, k),), 255, dtype=torch.uint8, device=DEV)
    capi.mxfp4_quantize(wd.data_ptr(), capi.GG_TYPE_F32, n, k, k, wp.data_ptr(), s)
    if x_name == "mxfp4":
        xd = torch.full((capi.mxfp4_packed_size(m, k),), 255, dtype=torch.uint8, device=DEV)
        xf = x.float()
        capi.mxfp4_quantize(xf.data_ptr(), capi.GG_TYPE_F32, m, k, k, xd.data_ptr(), s)
        xt = capi.GG_TYPE_MXFP4
    else:
        xt, t = TYPES[x_name]
        xd = x.to(t)
        assert torch.equal(xd.double(), x)
    ldy = -(-n // 8) * 8 + 8 if pad else n
    y = torch.full((m, ldy), 55.0, dtype=TYPES[y_name][1], device=DEV)
    ws = torch.full((max(capi.mxfp4_linear_workspace_size(xt, m, n, k), 16),), 255, dtype=torch.uint8, device=DEV)
    capi.mxfp4_linear(wp.data_ptr(), xd.data_ptr(), xt, k, y.data_ptr(), TYPES[y_name][0], ldy, m, n, k, ws.data_ptr(), s)
    want = (x @ w.T).float().to(TYPES[y_name][1])
    torch.cuda.synchronize()
    assert torch.equal(y[:, :n], want)
    assert (y[:, n:] == 55).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(TILES), ids=lambda c: "-".join(map(str, c)))
def test_tiles(gpu, case):
    check(*case, "f32", False)                                            # rows at odd addresses
    check(*case, "bf16" if case[0] == "mxfp4" else case[0], True)         # whole 16 bytes


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(FEW), ids=lambda c: "-".join(map(str, c)))
def test_few_rows(gpu, case):
    check(*case, "f32", False)
    check(*case, "f16" if case[0] == "f32" else case[0], True)
