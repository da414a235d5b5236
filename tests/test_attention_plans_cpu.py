"""What the attention calls ask for beside their tensors, from sizes alone (no GPU)."""
import ctypes

import pytest

from gpt_neox_amd import _lib


def backward_scratch(b, s, h, h_kv, d, window, sinks):
    need = ctypes.c_int64()
    assert _lib.lib().neox_window_attention_bwd_workspace(need, b, s, s, h, h_kv, d, window, sinks) == 0
    return need.value


@pytest.mark.parametrize("b,s,h,h_kv,d,window", [
    (1, 8192, 32, 32, 128, 4096), (8, 8192, 32, 32, 128, 4096), (1, 131072, 32, 8, 128, 4096), (4, 16384, 16, 16, 64, 1024), (2, 20000, 12, 4, 256, 2048)])
def test_scratch_of_a_few_sinks_is_a_part_of_the_keys(b, s, h, h_kv, d, window):
    # sums in pieces are kept for the key tiles that are cut into pieces, here the first, whatever the number of tiles; rows
    # behind the window add sums of the sinks alone, in at most 64 pieces
    rows, keys = 4 * b * h * s, 2 * b * s * h_kv * d
    assert backward_scratch(b, s, h, h_kv, d, window, 0) == rows
    for sinks in (1, 4, 16):
        sums = backward_scratch(b, s, h, h_kv, d, window, sinks) - rows
        assert 0 < sums <= 4 * b * h_kv * 2 * d * (128 + 64 * sinks)
        assert sums < 0.25 * keys
