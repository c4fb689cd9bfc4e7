"""Page tables of the 8-bit cache's entry points as views: rows apart, columns of a wider table, one row for all."""
import pytest
import torch

from edgelm_b200.csrc import ops
from tests import quant_reference as ref
from tests.test_quant_cache_gpu import DEV, cache_args, i32, word
from tests.test_quant_prefill_gpu import tiles_of

pytestmark = pytest.mark.gpu
NH, NKV, HD, LENGTHS = 4, 2, 64, [130, 200, 64]


def every_entry(cache, table, pos, dtype):
    """Outputs of the five entry points for one token a sequence at `pos`, and their error words."""
    B, cache = len(pos), {k: v.clone() for k, v in cache.items()}
    cos, sin = ref.tables(512, HD, DEV)
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn((B, (NH + 2 * NKV) * HD), generator=g).to(dtype).to(DEV)
    slot, at, kept, err = i32(range(B)), i32(pos), cache_args(cache), word()
    keys, values = (torch.zeros((B, NKV, HD), dtype=dtype, device=DEV) for _ in range(2))
    ops.quantized_rows(*kept, at, slot, slot, table, keys, values, err)
    outs, words = [keys, values], [err]
    rows = qkv[:, :NH * HD].contiguous()
    for meta_ready in (False, True):
        out, err = torch.zeros_like(rows), word()
        ops.attn_decode_quantized(rows, out, *kept, table, slot, at, B, NH, NKV, HD, 0.125, err=err, n_splits=2, meta_ready=meta_ready)
        outs.append(out)
        words.append(err)
    tiles = [slot, slot, i32([1] * B), at]
    for form in (1, 2) if dtype == torch.bfloat16 else (1,):
        out, err = torch.zeros_like(rows), word()
        ops.attn_prefill_quantized(rows, out, *kept, table, slot, *tiles, B, NH, NKV, HD, 0.125, err=err, n_splits=1, form=form)
        outs.append(out)
        words.append(err)
    out, err = torch.zeros_like(rows), word()
    ops.attn_decode_rope_quantized(qkv, out, *kept, table, slot, at, cos, sin, B, NH, NKV, HD, 0.125, err=err, n_splits=2)
    words.append(err)
    err = word()
    turned = qkv.clone()
    ops.rope_quantize_append(turned, at, slot, slot, table, cos, sin, *kept, NH, NKV, HD, err)
    words.append(err)
    return outs + [out, turned, *cache.values()], [int(w) for w in words]


def same(a, b):
    return all(torch.equal(x.contiguous().view(torch.int8), y.contiguous().view(torch.int8)) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_of_tables(dtype):
    cache, table = ref.make_cache("int8", NKV, HD, LENGTHS, DEV, 3)
    pos = [n - 1 for n in LENGTHS]
    want, words = every_entry(cache, table, pos, dtype)
    assert not any(words)
    wide = torch.full((6, table.shape[1] + 5), 1, dtype=torch.int32, device=DEV)
    wide[::2, 2:2 + table.shape[1]] = table
    got, words = every_entry(cache, wide[::2, 2:2 + table.shape[1]], pos, dtype)
    assert not any(words) and same(got, want)
    # one row for all (a step of 0 from row to row)
    row, pos = table[1:2], [60, 130, 199]
    want, words = every_entry(cache, row.repeat(3, 1), pos, dtype)
    assert not any(words)
    got, words = every_entry(cache, row.expand(3, -1), pos, dtype)
    assert not any(words) and same(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_behind_a_views_width_are_not_looked_up(dtype):
    """A position whose page the table has no column for is reported, also where the view's storage goes on there."""
    cache, table = ref.make_cache("int8", NKV, HD, LENGTHS, DEV, 3)
    wide = torch.full((3, 8), 1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    _, words = every_entry(cache, wide[:, :table.shape[1]], [129, 64 * table.shape[1] + 3, 63], dtype)
    assert all(w == 4 for w in words), words
