"""What the K/V page and verification entry points refuse, and their sizes:
checked on the host before anything is queued, so no GPU is needed."""
import ctypes

import pytest

from gemma_amd import capi

P = 1 << 20   # stands for a device address; never read
BAD = capi.GG_ERR_INVALID
F32, F16, BF16, MX, E4M3 = capi.GG_TYPE_F32, capi.GG_TYPE_F16, capi.GG_TYPE_BF16, capi.GG_TYPE_MXFP4, capi.GG_TYPE_E4M3
PAGES = dict(k=P, v=P, k_scale=None, v_scale=None, page_stride=4096, pos_stride=256, head_stride=128, type=BF16, n_pages=8, page_size=16,
             n_kv_heads=2, head_dim=128)
SEQS = dict(row_start=P, len=P, table=P, n_seqs=3, n_rows=10, max_rows=6, max_len=100, table_ld=7)
STORE = dict(type=F32, q=P, ldq=1024, k=P, ldk=1024, v=P, ldv=1024, n_q_heads=4, q_norm=P, k_norm=P, eps=1e-6, theta=1e4, q_out=P,
             q_out_type=F32, ldqo=512, stream=None)
LOAD = dict(k_out=P, ldk=256, v_out=P, ldv=256, type=F32, stream=None)
ATTN = dict(q=P, type=BF16, ldq=512, n_q_heads=4, scale=0.1, window=0, sinks=0, out=P, ldo=512, lse=P, workspace=P, stream=None)
VERIFY = dict(z=P, y=P, type=F32, rows=10, n=1000, ldz=1000, ldy=1000, draft=P, row_start=P, n_seqs=3, temperature=P, accept_u=P, draw_u=P,
              accepted=P, tokens=P, logprobs=P, workspace=P, stream=None)


def call(name, own, change):
    parts = [dict(PAGES), dict(SEQS), dict(own)]
    for key, value in change.items():
        part = next((d for d in (parts[2], parts[0], parts[1]) if key in d and not key.startswith("pages_")), None)
        if key.startswith("pages_"):
            parts[0][key[6:]] = value
        else:
            part[key] = value
    pages, seqs = capi.GGKvPages(*(parts[0][f[0]] for f in capi.GGKvPages._fields_)), capi.GGKvSeqs(*parts[1].values())
    return getattr(capi.lib(), name)(ctypes.byref(pages), ctypes.byref(seqs), *parts[2].values())


POOL = [dict(pages_k=None), dict(pages_v=None), dict(pages_k=P + 8), dict(pages_v=P + 2), dict(pages_type=F32), dict(pages_type=MX),
        dict(pages_type=capi.GG_TYPE_Q8_0), dict(page_stride=4100), dict(pos_stride=257), dict(head_stride=132), dict(page_stride=-4096),
        dict(head_stride=0), dict(pos_stride=64), dict(page_stride=8), dict(n_pages=0), dict(n_pages=-1), dict(page_size=0),
        dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(head_dim=0), dict(head_dim=8), dict(head_dim=120), dict(head_dim=272),
        dict(pages_type=E4M3), dict(pages_type=E4M3, k_scale=P), dict(pages_type=E4M3, k_scale=P, v_scale=P + 2),
        dict(row_start=None), dict(len=None), dict(table=None), dict(row_start=P + 2), dict(table=P + 1), dict(n_seqs=0),
        dict(n_seqs=(1 << 22) + 1), dict(n_rows=0), dict(n_rows=-5), dict(max_rows=0), dict(max_len=0), dict(max_len=(1 << 30) + 1), dict(table_ld=0)]


@pytest.mark.parametrize("name,own", [("gg_kv_store", STORE), ("gg_kv_load", LOAD), ("gg_kv_attention", ATTN)])
@pytest.mark.parametrize("change", POOL)
def test_pool_and_sequences(name, own, change):
    assert call(name, own, change) == BAD


@pytest.mark.parametrize("change", [dict(type=MX), dict(type=E4M3), dict(q=None), dict(n_q_heads=0), dict(n_q_heads=-1), dict(ldq=511), dict(k=None),
                                    dict(v=None), dict(ldk=255), dict(ldv=0), dict(q_out=None), dict(q_out_type=E4M3), dict(ldqo=500),
                                    dict(q=P + 2), dict(k=P + 1), dict(v=P + 2), dict(q_out=P + 2), dict(q_norm=P + 2), dict(k_norm=P + 1),
                                    dict(eps=-1.0), dict(eps=float("nan")), dict(theta=-1.0), dict(theta=float("inf")),
                                    dict(type=BF16, k=P + 1), dict(n_q_heads=(1 << 16) + 1, ldq=1 << 40, ldqo=1 << 40)])
def test_store_refuses(change):
    assert call("gg_kv_store", STORE, change) == BAD


@pytest.mark.parametrize("change", [dict(type=MX), dict(k_out=None, v_out=None), dict(ldk=255), dict(ldv=-1), dict(k_out=P + 2), dict(v_out=P + 1)])
def test_load_refuses(change):
    assert call("gg_kv_load", LOAD, change) == BAD


@pytest.mark.parametrize("change", [dict(q=None), dict(out=None), dict(type=MX), dict(type=E4M3), dict(n_q_heads=0), dict(n_q_heads=3), dict(ldq=511),
                                    dict(ldo=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(window=-1), dict(sinks=-1),
                                    dict(q=P + 1), dict(out=P + 1), dict(lse=P + 2), dict(pages_type=F16), dict(pages_type=F16, type=F32),
                                    dict(workspace=None, max_len=4096), dict(workspace=P + 8, max_len=4096),
                                    dict(n_rows=1 << 28, n_q_heads=8, ldq=1024, ldo=1024)])
def test_attention_refuses(change):
    assert call("gg_kv_attention", ATTN, change) == BAD


@pytest.mark.parametrize("change", [dict(z=None), dict(type=MX), dict(rows=0), dict(rows=(1 << 30) + 1), dict(n=0), dict(ldz=999), dict(ldy=999),
                                    dict(draft=None), dict(row_start=None), dict(n_seqs=0), dict(n_seqs=(1 << 22) + 1), dict(temperature=None),
                                    dict(accept_u=None), dict(draw_u=None), dict(accepted=None), dict(tokens=None), dict(workspace=None),
                                    dict(workspace=P + 8), dict(z=P + 2), dict(y=P + 1), dict(type=BF16, y=P + 1), dict(draft=P + 1),
                                    dict(accept_u=P + 4), dict(draw_u=P + 4), dict(logprobs=P + 2), dict(tokens=P + 2)])
def test_verify_refuses(change):
    assert capi.lib().gg_verify_drafts(*dict(VERIFY, **change).values()) == BAD


def structures(pages=None, seqs=None):
    p, s = dict(PAGES, **(pages or {})), dict(SEQS, **(seqs or {}))
    return capi.GGKvPages(*(p[f[0]] for f in capi.GGKvPages._fields_)), capi.GGKvSeqs(*s.values())


def test_null_structures():
    p, s = structures()
    L = capi.lib()
    assert L.gg_kv_load(None, ctypes.byref(s), *LOAD.values()) == BAD
    assert L.gg_kv_load(ctypes.byref(p), None, *LOAD.values()) == BAD
    assert L.gg_kv_attention(None, None, *ATTN.values()) == BAD
    assert L.gg_kv_attention_workspace_size(None, ctypes.byref(s), 4, 0, 0) == 0


def test_workspace_sizes():
    ws = capi.kv_attention_workspace_size
    assert ws(*structures(), 4) == 0                                       # one chunk
    assert ws(*structures(), 3) == 0 and ws(*structures(), 0) == 0 and ws(*structures(pages=dict(type=F32)), 4) == 0
    long = structures(seqs=dict(max_len=1 << 17))
    assert ws(*long, 4) % (10 * 4 * (128 + 4) * 4) == 0 and ws(*long, 4) > 0
    assert ws(*long, 4, 64, 4) == 0                                        # a window of one chunk
    assert ws(*structures(seqs=dict(max_len=1 << 30, table_ld=1 << 30)), 512) > 0
    assert ws(*structures(seqs=dict(max_len=1 << 30, n_rows=1 << 20, table_ld=1 << 30)), 512) == 0   # blocks enough without chunks
    v = capi.verify_drafts_workspace_size
    assert v(10, 3, 1000) > 0 and v(0, 3, 1000) == 0 and v(10, 0, 1000) == 0 and v(10, 3, 0) == 0
    assert v(1 << 30, 1 << 22, 1 << 30) > 1 << 50


def test_binding_raises():
    p, s = structures(pages=dict(head_dim=8))
    with pytest.raises(capi.GGError) as e:
        capi.kv_load(p, s, P, 256, P, 256, F32)
    assert e.value.code == BAD


def test_struct_layouts_match_header():
    assert ctypes.sizeof(capi.GGKvPages) == 4 * 8 + 3 * 8 + 5 * 4 + 4
    assert ctypes.sizeof(capi.GGKvSeqs) == 3 * 8 + 5 * 4 + 4
