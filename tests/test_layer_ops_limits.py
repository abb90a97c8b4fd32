"""The feed-forward block's largest calls: rows whose tiles are more than a launch has are refused before it, whatever kernel the rule chooses."""
import pytest

from test_token_ops_refusals import _refused


@pytest.mark.parametrize("H,I", [(8, 8), (8, 264), (264, 8)])
def test_more_tiles_than_a_launch_has(H, I):
    from ancora_cutile_amd import _lib
    lib, a, rows = _lib.load(), [(i + 1) << 42 for i in range(9)], (1 << 31) - 1
    _refused(lib, "anc_gated_ffn", (a[0], a[1], a[2], 0, 0, 0, rows, rows, H, I, a[3], a[4], a[5], 0), "too large")
    _refused(lib, "anc_ffn_down", (a[0], a[1], 0, 0, 0, rows, rows, I, H, 0, a[2], 1, 0), "too large")
    _refused(lib, "anc_gated_ffn_grad", (a[0], a[1], a[2], a[3], 0, 0, 0, rows, rows, H, I, a[4], a[5], 0, 0), "too large")
    _refused(lib, "anc_gated_ffn_dx", (a[0], a[1], a[2], a[3], 0, 0, 0, rows, rows, H, I, 0, a[4], 1, 0), "too large")
