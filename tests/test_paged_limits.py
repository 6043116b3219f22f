"""Extremes of the paged calls' arguments."""
import ctypes as C

import pytest

from ma_transformer_b200 import _native as nat
from test_paged_attention import _decode, _struct


@pytest.mark.parametrize("left", [2 ** 63 - 1, 2 ** 63 - 16, 2 ** 62])
@pytest.mark.parametrize("B, width", [(1, 40), (2, 1 << 16), (300, 512)])
def test_a_window_wider_than_any_sequence_plans_for_the_whole_cache(left, B, width):
    s, _ = _struct()
    size = lambda taps: nat.lib.mat_paged_decode_workspace_bytes(C.byref(s), B, 4, width, taps, 0)  # noqa: E731
    assert size(left) == size(-1) == size(width * 16)


@pytest.mark.parametrize("n_sel", [2 ** 27, 2 ** 59, 2 ** 60, 2 ** 63 - 1])
def test_a_list_of_more_pages_than_32_bits_of_tokens_is_refused(n_sel):
    s, base = _struct()
    assert nat.lib.mat_paged_decode_workspace_bytes(C.byref(s), 2, 4, 3, -1, n_sel) == 0
    assert _decode(s, base, pages=base, n_sel=n_sel) == 1 and b"list of pages" in nat.lib.mat_last_error()
