"""Prompt attention over the 8-bit cache against its plain statement (tests/quant_reference.py)."""
import math

import pytest
import torch

from edgelm_b200.csrc import ops
from tests import quant_reference as ref
from tests.test_quant_cache_gpu import DEV, DTYPES, cache_args, check, i32, off_bound, same, word

pytestmark = pytest.mark.gpu


def tiles_of(totals, news, size=128):
    rows, t0 = [], 0
    for b, (n, m) in enumerate(zip(totals, news)):
        rows += [(b, t0 + a, min(size, m - a), n - m + a) for a in range(0, m, size)]
        t0 += m
    return [i32(r[i] for r in rows) for i in range(4)], len(rows)


def prompt_case(fmt, dtype, nh, nkv, hd, totals, news, window=0, splits=None, seed=1, spoil=True, change=None, size=128, max_keys=0, pad=0, form=0):
    dtype = DTYPES[dtype]
    cache, table = ref.make_cache(fmt, nkv, hd, totals, DEV, seed, k_size=1.5)
    if spoil:     # what lies behind a sequence's end is not its own: no number at all
        for b, n in enumerate(totals):
            if n % 64:
                p = int(table[b, n // 64])
                cache["ks"][p, :, n % 64:] = float("nan")
                cache["vs"][p, :, n % 64:] = float("inf")
                if fmt == "fp8":
                    cache["v"].view(torch.int8)[p, :, n % 64:] = 0x7f
                    cache["k"].view(torch.int8)[p, :, n % 64:] = 0x7f
    if change:
        change(cache, table)
    before = {k: v.clone() for k, v in cache.items()}
    T = sum(news)
    q = torch.randn((T, (nh + 2 * nkv) * hd + pad), generator=torch.Generator().manual_seed(seed + 1)).to(dtype).to(DEV)
    out = torch.full((T, nh * hd + 16), 3.0, dtype=dtype, device=DEV)
    err, scale = word(), 1 / math.sqrt(hd)
    tiles, n_tiles = tiles_of(totals, news, size)
    ops.attn_prefill_quantized(q, out[:, :nh * hd], *cache_args(cache), table, i32(range(len(totals))), *tiles, n_tiles, nh, nkv, hd, scale, err=err, window=window,
                               max_keys=max_keys, n_splits=splits, form=form)
    assert int(err) == 0 and bool((out[:, nh * hd:] == 3.0).all())
    for k in before:
        assert same(before[k], cache[k])
    t0 = 0
    for b, (n, m) in enumerate(zip(totals, news)):
        keys, values = ref.sequence_rows(cache, table[b], n)
        qq = q[t0:t0 + m, :nh * hd].double().view(m, nh, hd)
        exact = ref.attend(qq, n - m, keys, values, scale, window)
        check(out[t0:t0 + m, :nh * hd].view(m, nh, hd), exact, off_bound(qq, n - m, keys, values, scale, window, exact, dtype, True))
        t0 += m
    return out[:, :nh * hd].view(T, nh, hd)


TOTALS, NEWS = [1, 17, 64, 65, 200, 400, 300], [1, 17, 64, 2, 200, 129, 1]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (4, 4, 64), (4, 1, 128), (3, 3, 32), (6, 2, 96), (2, 1, 16), (5, 1, 48), (3, 1, 80), (2, 2, 256), (12, 1, 64),
                                       (24, 2, 112), (7, 1, 192), (2, 1, 208), (2, 2, 144)])
def test_prompt_heads_and_lengths(fmt, dtype, nh, nkv, hd):
    prompt_case(fmt, dtype, nh, nkv, hd, TOTALS, NEWS, form=1)
    prompt_case(fmt, dtype, nh, nkv, hd, TOTALS, NEWS)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (4, 4, 64), (12, 1, 64), (4, 1, 128), (3, 3, 128), (32, 2, 128), (6, 2, 16), (5, 5, 32), (9, 3, 48), (3, 1, 80), (8, 2, 96), (7, 1, 112)])
def test_prompt_on_tcgen05(fmt, nh, nkv, hd):
    prompt_case(fmt, "bf16", nh, nkv, hd, [1], [1], form=2)
    prompt_case(fmt, "bf16", nh, nkv, hd, [17, 64], [17, 64], form=2)
    prompt_case(fmt, "bf16", nh, nkv, hd, TOTALS, NEWS, form=2)
    prompt_case(fmt, "bf16", nh, nkv, hd, [128, 1300, 129], [128, 700, 65], form=2)
    prompt_case(fmt, "bf16", nh, nkv, hd, TOTALS, NEWS, form=2, size=50, pad=40)
    for window in (1, 64, 65, 130, 300, 5000):
        prompt_case(fmt, "bf16", nh, nkv, hd, TOTALS + [900], NEWS + [500], window=window, form=2)


@pytest.mark.parametrize("splits", [1, 2, 3, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (4, 1, 128), (3, 1, 256), (3, 1, 48), (4, 2, 96)])
def test_prompt_splits(splits, dtype, nh, nkv, hd):
    prompt_case("int8", dtype, nh, nkv, hd, TOTALS + [2500], NEWS + [70], splits=splits, form=1)
    if dtype == "bf16" and hd <= 128:
        for window in (0, 300):
            prompt_case("int8", dtype, nh, nkv, hd, TOTALS + [2500], NEWS + [70], splits=splits, form=2, window=window)
            prompt_case("fp8", dtype, nh, nkv, hd, [2500, 40], [3, 40], splits=splits, form=2, window=window)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 130, 5000])
def test_prompt_window(window):
    prompt_case("int8", "bf16", 9, 3, 64, TOTALS, NEWS, window=window)
    prompt_case("fp8", "f32", 4, 1, 128, TOTALS, NEWS, window=window, splits=4)
    prompt_case("fp8", "bf16", 2, 2, 160, TOTALS, NEWS, window=window)


def test_prompt_long_and_smaller_tiles():
    prompt_case("fp8", "bf16", 4, 2, 64, [1500], [1500])
    prompt_case("int8", "bf16", 4, 4, 64, [64 * 40 + 3], [300], splits=1)     # more tiles of keys than a lane of the copying warp holds pages of
    for size in (1, 5, 64, 100):
        prompt_case("int8", "bf16", 6, 2, 64, [130, 70], [130, 33], size=size, max_keys=130)


def test_prompt_rows_lie_where_the_strides_say():
    prompt_case("int8", "bf16", 9, 3, 64, TOTALS, NEWS, pad=24)
    prompt_case("fp8", "f32", 9, 3, 48, TOTALS, NEWS, pad=4)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_scales_of_all_sizes(fmt, dtype):
    def change(cache, table):
        cache["vs"].mul_((10.0 ** (torch.rand(cache["vs"].shape, generator=torch.Generator().manual_seed(9)) * 40 - 20)).to(DEV))
        cache["v"].view(torch.int8)[:, :, ::7] = 0
        cache["vs"][:, :, ::7] = 2.0 ** -60 / ref.TOP[fmt]
    for form in (1, 2) if dtype == "bf16" else (1,):
        prompt_case(fmt, dtype, 9, 3, 64, [200, 70], [200, 7], change=change, spoil=False, form=form)


@pytest.mark.parametrize("splits", [1, 4])
def test_prompt_a_row_that_is_no_number_reaches_who_sees_it(splits):
    def change(cache, table):
        cache["vs"][int(table[0, 1]), 0, 5] = float("nan")       # value of position 69, kv head 0
        cache["v"].view(torch.int8)[int(table[0, 1]), 0, 5] = 0
        cache["ks"][int(table[0, 0]), 1, 3] = float("nan")       # key of position 3, kv head 1
        cache["k"].view(torch.int8)[int(table[0, 0]), 1, 3] = 0
    for window, form, hd in ((0, 1, 64), (50, 1, 64), (0, 2, 64), (50, 2, 64), (0, 2, 128)):
        out = prompt_case("fp8", "bf16", 4, 2, hd, [200], [200], change=change, spoil=False, splits=splits, window=window, form=form)
        nan = torch.isnan(out).all(-1).cpu()
        p = torch.arange(200)
        first = (p >= 69) & ((p < 69 + window) if window else p >= 0)
        second = (p >= 3) & ((p < 3 + window) if window else p >= 0)
        assert torch.equal(nan, torch.stack([first, first, second, second], 1))


def test_prompt_in_a_graph():
    cache, table = ref.make_cache("int8", 3, 64, [200, 64], DEV, 3)
    tiles, n = tiles_of([200, 64], [150, 64])
    q, err = torch.randn((214, 9 * 64), device=DEV).bfloat16(), word()
    out, captured = torch.empty_like(q), torch.zeros_like(q)
    run = lambda o: ops.attn_prefill_quantized(q, o, *cache_args(cache), table, i32s, *tiles, n, 9, 3, 64, 0.125, err=err)   # noqa: E731
    i32s = i32([0, 1])
    run(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(captured)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, captured) and int(err) == 0
    ops.attn_prefill_quantized(q, out, *cache_args(cache), table, i32s, *tiles, 0, 9, 3, 64, 0.125)


def test_prompt_pages_that_are_not_there_are_reported():
    for page in (-1, 99):
        cache, table = ref.make_cache("int8", 1, 64, [128], DEV, 3)
        table[0, 0] = page
        tiles, n = tiles_of([128], [20])
        err = word()
        q = torch.randn((20, 128), device=DEV)
        ops.attn_prefill_quantized(q, torch.empty_like(q), *cache_args(cache), table, i32([0]), *tiles, n, 2, 1, 64, 0.125, err=err)
        assert int(err) == 4
        err.zero_()
        q = q.bfloat16()
        ops.attn_prefill_quantized(q, torch.empty_like(q), *cache_args(cache), table, i32([0]), *tiles, n, 2, 1, 64, 0.125, err=err, form=2)
        assert int(err) == 4


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_prompt_and_decode_scales_of_any_sign(scale):
    nh, nkv, hd, n = 4, 2, 64, 150
    cache, table = ref.make_cache("int8", nkv, hd, [n], DEV, 3)
    q, err = torch.randn((n, nh * hd), generator=torch.Generator().manual_seed(4)).bfloat16().to(DEV), word()
    keys, values = ref.sequence_rows(cache, table[0], n)
    exact = ref.attend(q.double().view(n, nh, hd), 0, keys, values, scale)
    bound = off_bound(q.double().view(n, nh, hd), 0, keys, values, abs(scale), 0, exact, torch.bfloat16, True)
    # (the bound's weighted sum is the positive scale's; what any weights can do is at most the largest value)
    bound = torch.maximum(bound, exact.abs() * 2.0 ** -8 + 2.0 ** -9 * values.abs().amax(0).repeat_interleave(nh // nkv, 0) * (1 + 40 * abs(scale)))
    tiles, n_tiles = tiles_of([n], [n])
    for form in (1, 2):
        out = torch.empty_like(q)
        ops.attn_prefill_quantized(q, out, *cache_args(cache), table, i32([0]), *tiles, n_tiles, nh, nkv, hd, scale, err=err, form=form)
        check(out.view(n, nh, hd), exact, bound)
    out = torch.empty((1, nh * hd), dtype=torch.bfloat16, device=DEV)
    ops.attn_decode_quantized(q[n - 1:], out, *cache_args(cache), table, i32([0]), i32([n - 1]), 1, nh, nkv, hd, scale, err=err)
    check(out.view(1, nh, hd), exact[n - 1:], bound[n - 1:])
    assert int(err) == 0


@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (16, 4, 128)])
@pytest.mark.parametrize("splits", [1, 4])
def test_prompt_runs_over_and_over_agree(nh, nkv, hd, splits):
    """Hundreds of launches in a row, blocks of one starting where blocks of the last end: every output the same, none reported."""
    totals, news = [600, 130, 333, 520], [90, 65, 129, 31]
    cache, table = ref.make_cache("int8", nkv, hd, totals, DEV, 3, k_size=1.5)
    q = torch.randn((sum(news), nh * hd), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    tiles, n_tiles = tiles_of(totals, news)
    outs, err = torch.zeros((400,) + q.shape, dtype=q.dtype, device=DEV), word()
    args = [*cache_args(cache), table, i32(range(4)), *tiles, n_tiles, nh, nkv, hd, 0.1]
    for out in outs:
        ops.attn_prefill_quantized(q, out, *args, err=err, n_splits=splits)
    assert int(err) == 0 and bool(outs[0].isfinite().all())
    assert bool((outs == outs[:1]).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,form", [("bf16", 2), ("bf16", 1), ("f32", 1)])
def test_query_rows_that_are_no_numbers_stay_to_themselves(fmt, dtype, form):
    """A head's query with a NaN or an infinity gives that head's row not-a-numbers, and changes no other row."""
    nh, nkv, hd, totals, news = 4, 2, 64, [70, 200], [3, 40]
    cache, table = ref.make_cache(fmt, nkv, hd, totals, DEV, 3)
    clean = torch.randn((sum(news), nh, hd), generator=torch.Generator().manual_seed(4)).to(DTYPES[dtype]).to(DEV)
    bad = clean.clone()
    bad[1, 2, 5], bad[1, 0, 63], bad[20, 3, 0] = float("nan"), float("inf"), float("-inf")
    hit = torch.zeros((sum(news), nh), dtype=torch.bool, device=DEV)
    hit[1, 2] = hit[1, 0] = hit[20, 3] = True
    tiles, n_tiles = tiles_of(totals, news)
    outs = []
    for q in (clean, bad):
        out = torch.empty_like(q)
        ops.attn_prefill_quantized(q.view(-1, nh * hd), out.view(-1, nh * hd), *cache_args(cache), table, i32(range(2)), *tiles, n_tiles, nh, nkv, hd, 0.1, err=word(),
                                   form=form)
        outs.append(out)
    assert torch.equal(outs[1].isnan().all(-1), hit) and torch.equal(outs[0][~hit], outs[1][~hit]) and bool(outs[0].isfinite().all())
    pos, outs = i32(n - 1 for n in totals), []
    for q in (clean[:2], bad[:2]):
        out = torch.empty_like(q)
        ops.attn_decode_quantized(q.reshape(2, nh * hd), out.view(2, nh * hd), *cache_args(cache), table, i32(range(2)), pos, 2, nh, nkv, hd, 0.1)
        outs.append(out)
    assert torch.equal(outs[1].isnan().all(-1), hit[:2]) and torch.equal(outs[0][~hit[:2]], outs[1][~hit[:2]]) and bool(outs[0].isfinite().all())


@pytest.mark.parametrize("nkv,hd", [(1, 256), (2, 128)])
def test_offsets_beyond_32_bits(nkv, hd):
    """A cache of more than 2^32 codes whose last pages are used: the same codes and outputs as in a small one."""
    nh, totals, news = 4 * nkv, [200, 70], [200, 70]
    pages = (1 << 32) // (nkv * 64 * hd) + 200
    big = {n: torch.zeros((pages, nkv, 64, hd), dtype=torch.int8, device=DEV) for n in ("k", "v")} | {n: torch.zeros((pages, nkv, 64), device=DEV) for n in ("ks", "vs")}
    small = {n: torch.zeros_like(t[:8]) for n, t in big.items()}
    table = torch.tensor([[0, 3, 5, 1], [7, 2, 6, 4]], dtype=torch.int32, device=DEV)
    qkv = torch.randn((sum(news), (nh + 2 * nkv) * hd), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(DEV)
    pos, seq = i32([*range(200), *range(70)]), i32([0] * 200 + [1] * 70)
    angles = torch.arange(256.0, device=DEV)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, device=DEV) / hd)
    cos, sin, err, (tiles, n_tiles) = angles.cos().contiguous(), angles.sin().contiguous(), word(), tiles_of(totals, news)
    got = []
    for cache, where in ((small, table), (big, table + (pages - 8))):
        q, kept = qkv.clone(), cache_args(cache)
        ops.rope_quantize_append(q, pos, seq, i32([0, 1]), where, cos, sin, *kept, nh, nkv, hd, err)
        rows = [torch.empty((270, nkv, hd), dtype=q.dtype, device=DEV) for _ in range(2)]
        ops.quantized_rows(*kept, pos, seq, i32([0, 1]), where, *rows, err)
        outs = []
        for form in (0, 1):
            outs.append(torch.empty((270, nh * hd), dtype=q.dtype, device=DEV))
            ops.attn_prefill_quantized(q, outs[-1], *kept, where, i32([0, 1]), *tiles, n_tiles, nh, nkv, hd, 0.1, err=err, form=form, n_splits=2)
        step = qkv[[5, 6]].contiguous()
        outs.append(torch.empty((2, nh * hd), dtype=q.dtype, device=DEV))
        ops.attn_decode_rope_quantized(step, outs[-1], *kept, where, i32([0, 1]), i32([200, 70]), cos, sin, 2, nh, nkv, hd, 0.1, err=err)
        assert int(err) == 0
        got.append([q, *rows, *outs] + [t[-8:].clone() for t in cache.values()])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and not any(bool(t[:-8].any()) for t in big.values())
