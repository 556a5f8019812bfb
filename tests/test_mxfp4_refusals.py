"""What the MXFP4 and scoring entry points refuse, and their sizes: checked on
the host before anything is queued, so no GPU is needed."""
import pytest

from gemma_amd import capi

P = 1 << 20   # stands for a device address; never read
BAD = capi.GG_ERR_INVALID
F32, F16, BF16, MX = capi.GG_TYPE_F32, capi.GG_TYPE_F16, capi.GG_TYPE_BF16, capi.GG_TYPE_MXFP4


def call(name, args, **change):
    args = dict(args, **change)
    return getattr(capi.lib(), name)(*args.values())


def test_packed_sizes():
    size = capi.mxfp4_packed_size
    assert size(32, 64) == 1024 + 256
    assert size(1, 1) == 1024 + 256                       # one tile, one group of scale dwords
    assert size(33, 257) == 2 * 5 * 1024 + 2 * 2 * 256
    assert size(262144, 1152) == 8192 * (18 * 1024 + 5 * 256)
    for rows, k in [(0, 32), (-1, 32), (32, 0), (32, -5), ((1 << 30) + 1, 32), (32, (1 << 20) + 1)]:
        assert size(rows, k) == 0


def test_workspace_sizes():
    ws = capi.mxfp4_linear_workspace_size
    assert ws(F32, 1, 1152, 6912) == 0 and ws(F32, 3, 1536, 1152) == 0     # few rows: none
    parts = 64 * (18 + 7) * 5 * 48 + 2 * 5 * 256                           # at least the parts of x
    assert ws(F32, 64, 1536, 1152) >= parts - 7 * 5 * 1536
    assert ws(MX, 4096, 8192, 8192) == 0                                    # enough blocks: no slices of k
    assert ws(MX, 16, 64, 1 << 20) > 0
    assert ws(capi.GG_TYPE_Q8_0, 64, 1536, 1152) == 0 and ws(F32, 0, 1, 1) == 0
    assert ws(F32, 1 << 30, 1 << 30, 1 << 20) > 1 << 50                     # no overflow
    assert capi.score_workspace_size(1 << 20, 1000, 5) == 0     # one block a row
    assert capi.score_workspace_size(1, 262144, 20) > 0
    assert capi.score_workspace_size(0, 1000, 5) == 0 and capi.score_workspace_size(1, 0, 5) == 0
    assert capi.score_workspace_size(1, 1000, 65) == 0 and capi.score_workspace_size(1, 1000, -1) == 0


QUANT = dict(src=P, type=F32, rows=4, k=64, ld=64, packed=P, stream=None)


@pytest.mark.parametrize("change", [dict(src=None), dict(packed=None), dict(type=capi.GG_TYPE_Q8_0), dict(type=MX),
                                    dict(rows=0), dict(k=0), dict(rows=-3), dict(ld=63), dict(k=(1 << 20) + 1, ld=1 << 21),
                                    dict(src=P + 2), dict(type=F16, src=P + 1), dict(packed=P + 8)])
def test_quantize_refuses(change):
    assert call("gg_mxfp4_quantize", QUANT, **change) == BAD


DEQUANT = dict(packed=P, out=P, rows=4, k=64, ld=64, stream=None)


@pytest.mark.parametrize("change", [dict(packed=None), dict(out=None), dict(rows=0), dict(k=-1), dict(ld=60),
                                    dict(packed=P + 4), dict(out=P + 2)])
def test_dequant_refuses(change):
    assert call("gg_mxfp4_dequant", DEQUANT, **change) == BAD


LINEAR = dict(w=P, x=P, x_type=F32, ldx=64, y=P, y_type=F32, ldy=32, m=40, rows=32, k=64, workspace=P, stream=None)


@pytest.mark.parametrize("change", [dict(w=None), dict(x=None), dict(y=None), dict(x_type=capi.GG_TYPE_Q8_0), dict(y_type=MX),
                                    dict(y_type=7), dict(ldx=63), dict(ldy=31), dict(m=0), dict(rows=0), dict(k=0),
                                    dict(m=-1), dict(w=P + 8), dict(x=P + 2), dict(x_type=MX, x=P + 8), dict(y=P + 1),
                                    dict(y_type=BF16, y=P + 1), dict(workspace=None), dict(workspace=P + 4)])
def test_linear_refuses(change):
    assert call("gg_mxfp4_linear", LINEAR, **change) == BAD


SCORE = dict(logits=P, type=F32, rows=2, n=300000, ld=300000, ids=P, n_ids=1, lp=P, lse=P, entropy=P, top=5, top_ids=P,
             top_lp=P, workspace=P, stream=None)


@pytest.mark.parametrize("change", [dict(logits=None), dict(type=MX), dict(rows=0), dict(n=0), dict(n=-4), dict(ld=299999),
                                    dict(n_ids=-1), dict(ids=None), dict(lp=None), dict(top=-1), dict(top=65),
                                    dict(logits=P + 2), dict(type=BF16, logits=P + 1), dict(workspace=None),
                                    dict(workspace=P + 8), dict(n=(1 << 30) + 1, ld=1 << 31)])
def test_score_refuses(change):
    assert call("gg_score_logits", SCORE, **change) == BAD


def test_binding_raises():
    with pytest.raises(capi.GGError) as e:
        capi.mxfp4_quantize(P, F32, 0, 64, 64, P)
    assert e.value.code == BAD
