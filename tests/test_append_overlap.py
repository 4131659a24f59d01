"""norm_rope_append refuses a q_out whose tokens overlap: warps would write one place in any order.  No GPU needed."""
import ctypes as C

import pytest

from test_prompt_refusals import append_args, lib


@pytest.mark.parametrize("stride", [0, 8, 8 * 128 - 8, -8 * 128])
def test_overlapping_tokens(stride):
    L, _lib = lib()
    assert L.pkv_norm_rope_append(0, C.byref(append_args(_lib, q_out_stride=stride)), None, None) == -1
    assert "overlap" in L.pkv_last_error().decode()
