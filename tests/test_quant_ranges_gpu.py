"""Attention over the 8-bit cache where its numbers are far from 1, against the plain statement (tests/quant_reference.py)."""
import math

import pytest
import torch

from edgelm_b200.csrc import ops
from tests import quant_reference as ref
from tests.test_quant_cache_gpu import DEV, DTYPES, cache_args, i32, word
from tests.test_quant_prefill_gpu import tiles_of

pytestmark = pytest.mark.gpu

# kernel, model type, query heads, kv heads, head size, blocks that share keys
KERNELS = [("decode", "bf16", 4, 2, 64, 1), ("decode", "f32", 8, 1, 64, 5), ("decode", "bf16", 6, 1, 128, 24), ("mma", "bf16", 4, 2, 64, 1), ("mma", "f32", 3, 1, 48, 3),
           ("tcgen05", "bf16", 4, 2, 64, 1), ("tcgen05", "bf16", 8, 1, 64, 3), ("tcgen05", "bf16", 4, 1, 128, 1)]


def attend(kernel, q, cache, table, total, nh, nkv, hd, scale, splits):
    """q [n, nh, hd], the last n tokens of one sequence of `total`: [n, nh, hd] by the kernel."""
    n, err, out = q.shape[0], word(), torch.empty((q.shape[0], nh * hd), dtype=q.dtype, device=DEV)
    rows = q.reshape(n, nh * hd)
    if kernel == "decode":      # each token as a sequence of its own over the same pages
        ops.attn_decode_quantized(rows, out, *cache_args(cache), table.expand(n, -1).contiguous(), i32(range(n)), i32(range(total - n, total)), n, nh, nkv, hd, scale,
                                  n_splits=splits, err=err)
    else:
        tiles, n_tiles = tiles_of([total], [n])
        ops.attn_prefill_quantized(rows, out, *cache_args(cache), table, i32([0]), *tiles, n_tiles, nh, nkv, hd, scale, err=err, n_splits=splits,
                                   form=2 if kernel == "tcgen05" else 1)
    assert int(err) == 0
    return out.view(n, nh, hd)


def check_one_key_takes_all(kernel, q, cache, table, total, nh, nkv, hd, scale, splits):
    """Scores so far apart that a row is the value row of its largest one.  Rows are looked at whose largest score leads by more than 2^-8 of
    sum |q_i k_i| scale, twice what the operands' roundings (2^-11 of a query, 2 x 2^-11 of a key, both ways) can move two scores, and by more than
    400.  Off by: the output's rounding, the weight's (2^-11 of one float16 term), on tcgen05 the value's two (its factor, its product with a
    code: 2^-11 each) and 2^-25 of the largest scale (a float16 number's smallest half step), and float32's own (2^-20)."""
    out, n = attend(kernel, q, cache, table, total, nh, nkv, hd, scale, splits).double(), q.shape[0]
    assert bool(out.isfinite().all())
    keys, values = ref.sequence_rows(cache, table[0], total)
    g = nh // nkv
    s = torch.einsum("nhd,lhd->hnl", q.double(), keys.repeat_interleave(g, 1)) * scale
    size = torch.einsum("nhd,lhd->hnl", q.double().abs(), keys.abs().repeat_interleave(g, 1)) * scale
    seen = torch.arange(total, device=DEV)[None] <= torch.arange(total - n, total, device=DEV)[:, None]
    s, size = s.masked_fill(~seen, -math.inf), size.masked_fill(~seen, 0.0)
    top = s.topk(2)
    lead = top.values[..., 0] - top.values[..., 1]
    clear = (lead > 2.0 ** -8 * size.amax(-1)) & (lead > 400)
    assert int(clear.sum()) * 2 >= clear.numel(), "the inputs' premise"
    want = values.repeat_interleave(g, 1)[top.indices[..., 0], torch.arange(nh, device=DEV)[:, None]].transpose(0, 1)      # [n, nh, hd]
    tol = torch.finfo(q.dtype).eps / 2 + (2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -22) + 2.0 ** -20
    floor = 0.0
    if kernel == "tcgen05":
        tol, floor = tol + 2 * 2.0 ** -11, 2.0 ** -25 * float(cache["vs"].max())
    off = (out - want).abs() - floor - tol * want.abs()
    assert bool((off <= 0).transpose(0, 1)[clear].all()), float(off.transpose(0, 1)[clear].max())


@pytest.mark.parametrize("power", [20, 25, 26, 27, 28, 29, 30, 31, 33, 40, 60, 90])
@pytest.mark.parametrize("kernel,dtype,nh,nkv,hd,splits", KERNELS)
def test_scores_far_from_zero(kernel, dtype, nh, nkv, hd, splits, power):
    """Scores of up to about 2^power, where 46 - M (the lift of the weights less the row's reference) is far from exact in float32."""
    total, n = 700, 150
    for fmt, per_key in (("int8", False), ("fp8", True)):
        cache, table = ref.make_cache(fmt, nkv, hd, [total], DEV, 3)
        g = torch.Generator().manual_seed(power)
        # the pages' keys (or the keys one by one: groups whose scales differ by more than 2^8) of several sizes, the largest anywhere
        shape = cache["ks"].shape if per_key else cache["ks"].shape[:1] + (1, 1)
        cache["ks"].mul_(2.0 ** (power - torch.randint(0, 13 if per_key else 6, shape, generator=g)).to(DEV))
        q = torch.randn((n, nh, hd), generator=g).to(DTYPES[dtype]).to(DEV)
        check_one_key_takes_all(kernel, q, cache, table, total, nh, nkv, hd, 1 / math.sqrt(hd), splits)


@pytest.mark.parametrize("power", [-90, -40, 60, 101, 104, 110, 118])
@pytest.mark.parametrize("kernel,dtype,nh,nkv,hd,splits", KERNELS)
def test_queries_of_any_size(kernel, dtype, nh, nkv, hd, splits, power):
    """Queries 2^power times as large under a scale 2^-power times as large are the same scores: the same bits.  (tcgen05: also where
    scales go into the scores a key at a time.)"""
    total, n = 300, 70
    for fmt, per_key in (("int8", False), ("fp8", True)):
        cache, table = ref.make_cache(fmt, nkv, hd, [total], DEV, 3)
        g = torch.Generator().manual_seed(5)
        if per_key:
            cache["ks"].mul_(2.0 ** -torch.randint(0, 13, cache["ks"].shape, generator=g).to(DEV))
        q, scale = torch.randn((n, nh, hd), generator=g).to(DTYPES[dtype]).to(DEV), 1 / math.sqrt(hd)
        args = (cache, table, total, nh, nkv, hd)
        assert torch.equal(attend(kernel, q, *args, scale, splits), attend(kernel, q * 2.0 ** power, *args, scale * 2.0 ** -power, splits))


@pytest.mark.parametrize("power", [100, 101, 104, 110])
@pytest.mark.parametrize("kernel,dtype,nh,nkv,hd,splits", KERNELS)
def test_queries_as_large_as_float32_holds(kernel, dtype, nh, nkv, hd, splits, power):
    """.. and under the usual scale they are numbers too: every row the value of one key."""
    total, n = 300, 70
    cache, table = ref.make_cache("int8", nkv, hd, [total], DEV, 3)
    q = torch.randn((n, nh, hd), generator=torch.Generator().manual_seed(5)).to(DTYPES[dtype]).to(DEV) * 2.0 ** power
    check_one_key_takes_all(kernel, q, cache, table, total, nh, nkv, hd, 1 / math.sqrt(hd), splits)


@pytest.mark.parametrize("kernel,dtype,nh,nkv,hd,splits", KERNELS)
def test_large_keys_under_small_queries(kernel, dtype, nh, nkv, hd, splits):
    """Keys of up to 2^118 under queries of about 2^-98, each key with a scale of its own: that scale times the codes' product is beyond
    float32 before the query's factor joins them, the score is not."""
    total, n = 300, 70
    cache, table = ref.make_cache("fp8", nkv, hd, [total], DEV, 3)
    g = torch.Generator().manual_seed(5)
    cache["ks"].mul_(2.0 ** (115 - torch.randint(0, 13, cache["ks"].shape, generator=g)).to(DEV))
    q = torch.randn((n, nh, hd), generator=g).to(DTYPES[dtype]).to(DEV) * 2.0 ** -98
    check_one_key_takes_all(kernel, q, cache, table, total, nh, nkv, hd, 1 / math.sqrt(hd), splits)


@pytest.mark.parametrize("kernel,dtype,nh,nkv,hd,splits", KERNELS)
def test_rows_far_from_zero_stay_to_themselves(kernel, dtype, nh, nkv, hd, splits):
    """Rows whose scores are far from zero (a query 2^14 or 2^60 times as large) beside usual ones: the usual ones' bits do not change."""
    total, n = 300, 70
    cache, table = ref.make_cache("int8", nkv, hd, [total], DEV, 3)
    q = torch.randn((n, nh, hd), generator=torch.Generator().manual_seed(5)).to(DTYPES[dtype]).to(DEV)
    large, hit = q.clone(), torch.zeros((n, nh), dtype=torch.bool, device=DEV)
    for i, (t, h) in enumerate([(0, 0), (3, nh - 1), (9, 1), (40, 0), (69, nh - 1)]):
        large[t, h] *= 2.0 ** (14 if i % 2 else 60)
        hit[t, h] = True
    args = (cache, table, total, nh, nkv, hd, 1 / math.sqrt(hd), splits)
    a, b = attend(kernel, q, *args), attend(kernel, large, *args)
    assert torch.equal(a[~hit], b[~hit]) and bool((a[hit] != b[hit]).any()) and bool(b.isfinite().all())
