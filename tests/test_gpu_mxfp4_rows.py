"""Products of more rows than one grid of the many-row kernel holds."""
import pytest
import torch

from gemma_amd import capi

from gpu_util import say, stream

pytestmark = pytest.mark.gpu


# packed x: 2^24 blocks of 384 threads; parts: 2^24 + 2 blocks of 256
@pytest.mark.parametrize("x_name,m", [("mxfp4", 1 << 30), ("bf16", (1 << 29) + 64)])
def test_product_of_many_rows(gpu, x_name, m):
    say("product", x_name, m)
    s, dev = stream(), "cuda:0"
    w = torch.tensor([[1.5]], device=dev)
    wp = torch.empty(capi.mxfp4_packed_size(1, 1), dtype=torch.uint8, device=dev)
    capi.mxfp4_quantize(w.data_ptr(), capi.GG_TYPE_F32, 1, 1, 1, wp.data_ptr(), s)
    values = torch.tensor([0, 1, 2, 3, -4, 6, -1.5, 0.5, 8, -12, 16], dtype=torch.bfloat16, device=dev)   # as MXFP4 holds them
    x = torch.empty(m, dtype=torch.bfloat16, device=dev)
    for lo in range(0, m, 1 << 26):
        x[lo:lo + (1 << 26)] = values[torch.arange(lo, min(m, lo + (1 << 26)), device=dev) % 11]
    y = torch.full((m,), 55.0, dtype=torch.bfloat16, device=dev)
    t, xs, ld = capi.GG_TYPE_BF16, x, 1
    if x_name == "mxfp4":
        xs = torch.empty(capi.mxfp4_packed_size(m, 1), dtype=torch.uint8, device=dev)
        capi.mxfp4_quantize(x.data_ptr(), t, m, 1, 1, xs.data_ptr(), s)
        t, ld = capi.GG_TYPE_MXFP4, 0
    need = capi.mxfp4_linear_workspace_size(t, m, 1, 1)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    try:
        capi.mxfp4_linear(wp.data_ptr(), xs.data_ptr(), t, ld, y.data_ptr(), capi.GG_TYPE_BF16, 1, m, 1, 1, ws.data_ptr(), s)
        torch.cuda.synchronize()
        for lo in range(0, m, 1 << 26):
            assert torch.equal(y[lo:lo + (1 << 26)], x[lo:lo + (1 << 26)] * 1.5)
    finally:
        del x, y, xs, ws
        torch.cuda.empty_cache()
