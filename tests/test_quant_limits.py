"""Sizes that the launches over the 8-bit cache have no room for are refused by name, in every form (no device is needed)."""
import ctypes

import pytest

from edgelm_b200.csrc import ops


@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("dtype,max_keys", [(0, 64), (1, 64), (1, 4096)])
def test_more_kv_heads_than_a_grid_has_rows(form, dtype, max_keys):
    lib = ops.lib()
    fn = lib.edgelm_attn_prefill_quantized
    fn.argtypes = [ctypes.c_char_p]
    nkv, hd = 70000, 16
    call = ops._QUANT_PREFILL(*[256] * 13, 0, nkv * hd, nkv * hd, dtype, 0, 1, 1, 1, 1, nkv, nkv, hd, 1, max_keys, 0, form, 0.1)
    assert fn(call) < 0 and "70000 key/value heads (takes up to 65,535)" in lib.edgelm_last_error().decode()
