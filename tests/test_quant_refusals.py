"""What the 8-bit cache's entry points refuse, before anything is launched (no device is needed)."""
import ctypes

import pytest
import torch

from edgelm_b200.csrc import ops


def cache(nkv=2, hd=64, dtype=torch.int8, pages=3):
    return (torch.zeros((pages, nkv, 64, hd), dtype=dtype), torch.zeros((pages, nkv, 64, hd), dtype=dtype), torch.zeros((pages, nkv, 64)), torch.zeros((pages, nkv, 64)))


def i32(n):
    return torch.zeros(n, dtype=torch.int32)


def call(which, c, nh=4, nkv=2, hd=64):
    table, cos = torch.zeros((1, 3), dtype=torch.int32), torch.zeros((8, hd // 2))
    q = torch.zeros((1, (nh + 2 * nkv) * hd))
    if which == "append":
        return ops.rope_quantize_append(q, i32(1), i32(1), i32(1), table, cos, cos, *c, nh, nkv, hd, i32(1))
    if which == "rows":
        return ops.quantized_rows(*c, i32(1), i32(1), i32(1), table, torch.zeros((1, nkv, hd)), torch.zeros((1, nkv, hd)), i32(1))
    if which == "decode":
        return ops.attn_decode_quantized(q, q, *c, table, i32(1), i32(1), 1, nh, nkv, hd, 0.1)
    if which == "decode_rope":
        return ops.attn_decode_rope_quantized(q, q, *c, table, i32(1), i32(1), cos, cos, 1, nh, nkv, hd, 0.1)
    return ops.attn_prefill_quantized(q, q, *c, table, i32(1), i32(1), i32(1), i32(1), i32(1), 1, nh, nkv, hd, 0.1)


ALL = ("append", "rows", "decode", "decode_rope", "prefill")


@pytest.mark.parametrize("which", ALL)
def test_refused(which):
    with pytest.raises(ops.KernelError, match="int8 or float8"):
        call(which, cache(dtype=torch.uint8))
    k, v, ks, vs = cache()
    with pytest.raises(ops.KernelError, match="alike"):
        call(which, (k, cache(dtype=torch.float8_e4m3fn)[1], ks, vs))
    with pytest.raises(ops.KernelError, match="codes must be"):
        call(which, (k[:, :1], v[:, :1], ks, vs))
    with pytest.raises(ops.KernelError, match="codes must be"):
        call(which, (k, v[:2], ks, vs))
    with pytest.raises(ops.KernelError, match="scales must be"):
        call(which, (k, v, ks.double(), vs))
    with pytest.raises(ops.KernelError, match="scales must be"):
        call(which, (k, v, ks, vs[:2]))
    with pytest.raises(ops.KernelError, match="contiguous"):
        call(which, (cache(pages=6)[0][::2], v, ks, vs))
    with pytest.raises(ops.KernelError, match="current device"):      # (tensors of the host)
        call(which, cache())


@pytest.mark.parametrize("which", ALL)
@pytest.mark.parametrize("hd", [8, 24, 272])
def test_head_sizes_that_are_not_taken(which, hd):
    with pytest.raises(ops.KernelError, match="head size"):
        call(which, cache(hd=hd), hd=hd)


@pytest.mark.parametrize("which", [w for w in ALL if w != "rows"])
def test_heads_that_do_not_divide(which):
    with pytest.raises(ops.KernelError, match="not a multiple"):
        call(which, cache(nkv=3), nh=4, nkv=3)


def test_the_library_refuses_too():
    lib = ops.lib()
    message = lambda: lib.edgelm_last_error().decode()      # noqa: E731

    def run(name, packed):
        fn = getattr(lib, name)
        fn.argtypes = [ctypes.c_char_p]
        return fn(packed)

    def go(dtype=0, fmt=0, n_seqs=1, nh=4, nkv=2, hd=64, splits=1, window=0, cos=0, sin=0, max_pos=0, k=256):
        return run("edgelm_attn_decode_quantized", ops._QUANT_DECODE(256, 256, k, 256, 256, 256, 256, 256, 256, cos, sin, 0, 0, 0, 512, 512, dtype, fmt, 1, 1, max_pos,
                                                                     n_seqs, nh, nkv, hd, splits, window, 0, 0.1))
    assert go(n_seqs=0) == 0
    for bad, word in (({"nh": 3}, "multiple"), ({"hd": 20}, "head size"), ({"fmt": 2}, "format"), ({"dtype": 5}, "dtype"), ({"splits": 12}, "splits"), ({"splits": 136}, "splits"), ({"splits": 16}, "scratch"),
                      ({"splits": 0}, "splits"), ({"window": -1}, "window"), ({"cos": 256}, "tables"), ({"n_seqs": 70000}, "sequences"), ({"k": 264}, "16-byte")):
        assert go(**bad) < 0 and word in message(), (bad, message())

    def go2(dtype=0, fmt=0, n_tiles=1, most=128, nh=4, nkv=2, hd=64, splits=1, window=0, q=256, ldq=512, form=0):
        return run("edgelm_attn_prefill_quantized", ops._QUANT_PREFILL(q, 256, 256, 256, 256, 256, 256, 256, 256, 256, 256, 256, 0, 0, ldq, 512, dtype, fmt, 1, 1, n_tiles,
                                                                       most, nh, nkv, hd, splits, 64, window, form, 0.1))
    assert go2(n_tiles=0) == 0
    for bad, word in (({"nh": 3}, "multiple"), ({"hd": 20}, "head size"), ({"fmt": 2}, "format"), ({"most": 129}, "tokens"), ({"splits": 9}, "splits"),
                      ({"window": -1}, "window"), ({"form": 3}, "form"), ({"form": 2}, "tcgen05"), ({"q": 264}, "16-byte"), ({"ldq": 510}, "multiple of 4"),
                      ({"n_tiles": 60000, "nh": 8}, "65,535")):
        assert go2(**bad) < 0 and word in message(), (bad, message())

    def go3(n=1, nh=4, hd=64, fmt=0, dtype=0, qkv=256):
        return run("edgelm_rope_quantize_append", ops._QUANT_APPEND(qkv, 0, 256, 256, 256, 256, 256, 256, 256, 256, 256, 256, 256, 0, dtype, fmt, 1, 1, 8, n, nh, 2, hd))
    assert go3(n=0) == 0
    for bad, word in (({"nh": 0}, "sizes"), ({"hd": 40}, "head size"), ({"fmt": 3}, "format"), ({"dtype": 2}, "dtype"), ({"qkv": 260}, "16-byte"), ({"n": 1 << 30}, "grid")):
        assert go3(**bad) < 0 and word in message(), (bad, message())

    def go4(n=1, nkv=2, hd=64, fmt=0, dtype=0, keys=256):
        return run("edgelm_quantized_rows", ops._QUANT_ROWS(256, 256, 256, 256, 256, 256, 256, 256, keys, 256, 256, 0, fmt, dtype, 1, 1, n, nkv, hd))
    assert go4(n=0) == 0
    for bad, word in (({"nkv": 0}, "sizes"), ({"hd": 40}, "head size"), ({"fmt": 3}, "format"), ({"dtype": 2}, "dtype"), ({"keys": 260}, "16-byte"), ({"n": 1 << 30}, "grid")):
        assert go4(**bad) < 0 and word in message(), (bad, message())


def test_numbers_that_no_field_holds():
    for field, value in ((18, 1 << 31), (18, 64.5), (0, -1)):
        args = [0] * 19
        args[field] = value
        with pytest.raises(ops.KernelError, match="quantized_rows"):
            ops._call_packed("edgelm_quantized_rows", 0, ops._QUANT_ROWS, *args)
