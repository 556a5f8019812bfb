"""gg_verify_drafts refuses tokens that lie over the drafts: a launch reads these after another has written tokens."""
import pytest

from gemma_amd import capi

P, Q, ROWS = 1 << 20, 1 << 24, 10   # stand for device addresses; never read


@pytest.mark.parametrize("off", [0, 4, 4 * (ROWS - 1), -4, -4 * (ROWS - 1)])
def test_tokens_over_drafts_are_refused(off):
    args = (P, P, capi.GG_TYPE_F32, ROWS, 1000, 1000, 1000, Q, P, 3, P, P, P, P, Q + off, P, P, None)
    assert capi.lib().gg_verify_drafts(*args) == capi.GG_ERR_INVALID
