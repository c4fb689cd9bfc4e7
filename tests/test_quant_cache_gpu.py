"""The 8-bit cache's kernels against plain statements of them (tests/quant_reference.py)."""
import math

import pytest
import torch

from edgelm_b200.csrc import ops
from tests import quant_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def i32(v):
    return torch.tensor(list(v), dtype=torch.int32, device=DEV)


def word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def same(a, b):
    return torch.equal(a.contiguous().view(torch.int8), b.contiguous().view(torch.int8)) if a.element_size() == 1 else \
        bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def cache_args(c):
    return c["k"], c["v"], c["ks"], c["vs"]


def off_bound(q, first, keys, values, scale, window, exact, dtype, given_bf16):
    """How far an output may be, number by number.  With A = sum p |v|: an operand's rounding moves a score by at most
    d = u_q sum |q_i k_i| scale, and every weight by a factor within 1 +- 2 d (numerator and denominator), the weights' own rounding
    by u_w, and the output is rounded once.  float16 terms: u = 2^-11 of one, 2^-22 of two (a bfloat16 query row is exact down to
    2^-14 of its largest number once lifted, taken as 2^-11 all the same); scores and exponents themselves are float32 sums: 2^-20 of
    the sum of their terms' magnitudes, the value's exponent of up to 2^5 and the reference among them.  Weighted rows far below the
    largest: a weight as operand is at most half of float16's smallest step (2^-25) off, and the largest one is 2^14 at least, so every
    key adds up to 2^-39 of the largest weighted row's largest number (matters where that row's own number is zero)."""
    n, nh, hd = q.shape
    g = nh // keys.shape[1]
    size = torch.einsum("nhd,lhd->hnl", q.abs(), keys.abs().repeat_interleave(g, 1)) * scale
    last = first + n
    u = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
    d = u * size.nan_to_num(0.0)[..., :last].amax(-1) + 2.0 ** -20 * (size.nan_to_num(0.0)[..., :last].amax(-1) + 32.0)      # [nh, n]
    a = ref.attend(q, first, keys, values.abs(), scale, window)
    half_ulp = torch.finfo(dtype).eps / 2
    floor = 2.0 ** -39 * last * ref.attend(q, first, keys, values.abs().amax(-1, keepdim=True), scale, window)
    return floor + exact.abs() * half_ulp + a * (2 * d.T[..., None] + 2 * u + 2.0 ** -20)


def check(out, exact, bound):
    out = out.double()
    nan = torch.isnan(exact)
    assert torch.equal(torch.isnan(out), nan), "not-a-numbers in other places"
    off = (out - exact).abs()[~nan]
    worst = (off / bound[~nan].clamp(min=1e-300)).max() if off.numel() else 0.0
    assert worst <= 1.0, f"{float(worst):.2f} of the bound"


# ----------------------------------------------------------------------------------------------------- writing and reading back
def step(lengths, news, nh, nkv, hd, dtype, seed, k_size=1.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(news)
    qkv = torch.randn((T, (nh + 2 * nkv) * hd), generator=g) * k_size
    pos = [p for n, m in zip(lengths, news) for p in range(n - m, n)]
    seq = [b for b, m in enumerate(news) for _ in range(m)]
    return qkv.to(dtype).to(DEV), i32(pos), i32(seq)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hd,nh,nkv", [(16, 3, 1), (32, 2, 2), (48, 4, 2), (64, 9, 3), (80, 5, 5), (128, 4, 1), (240, 2, 1), (256, 3, 3)])
def test_append_writes_what_the_format_says(fmt, dtype, hd, nh, nkv):
    lengths, news = [1, 70, 64, 200], [1, 6, 64, 3]
    cache, table = ref.make_cache(fmt, nkv, hd, lengths, DEV, 7)
    qkv, pos, seq = step(lengths, news, nh, nkv, hd, DTYPES[dtype], 11)
    rows = qkv.view(-1, nh + 2 * nkv, hd)
    rows[0, nh:] = 0                                          # a key and a value of zeros
    rows[1, nh, 3] = float("nan")
    rows[2, nh + nkv, hd - 1] = float("inf")
    rows[3, nh, :] = 1e-30                                    # below what a row's largest magnitude counts as
    rows[4, nh + nkv, :] *= 1e30
    cos, sin = ref.tables(256, hd, DEV)
    slot = i32([2, 0, 3, 1])                                  # sequences in another order than the table's rows
    table = table[torch.argsort(slot.long())].contiguous()
    x = rows.float()
    turned = ref.rotate(x[:, :nh + nkv], cos[pos.long()], sin[pos.long()])
    want = {k: v.clone() for k, v in cache.items()}
    page = table[slot[seq.long()].long(), pos.long() // 64].long()
    for codes, scales, new in (("k", "ks", turned[:, nh:]), ("v", "vs", x[:, nh + nkv:])):
        c, s = ref.quantize(new, fmt)
        want[codes].view(torch.int8)[page, :, pos.long() % 64] = c.view(torch.int8)
        want[scales][page, :, pos.long() % 64] = s
    want_q, rest = turned[:, :nh].to(qkv.dtype), x[:, nh:].clone()
    err = word()
    # the queries to rows of their own first: the projections stay as they were
    other, before, q_out = {k: v.clone() for k, v in cache.items()}, qkv.clone(), torch.zeros((len(pos), nh * hd), dtype=qkv.dtype, device=DEV)
    ops.rope_quantize_append(qkv, pos, seq, slot, table, cos, sin, *cache_args(other), nh, nkv, hd, err, q_out=q_out)
    assert same(qkv, before) and same(q_out, want_q.reshape(len(pos), -1).contiguous())
    ops.rope_quantize_append(qkv, pos, seq, slot, table, cos, sin, *cache_args(cache), nh, nkv, hd, err)
    assert int(err) == 0
    for k in want:
        assert same(cache[k], want[k]) and same(other[k], want[k]), k
    assert same(qkv.view(-1, nh + 2 * nkv, hd)[:, :nh].contiguous(), want_q.contiguous())
    assert same(qkv.view(-1, nh + 2 * nkv, hd)[:, nh:].float(), rest)
    # and back
    for out in (torch.float32, torch.bfloat16):
        keys, values = (torch.full((len(pos), nkv, hd), 7.0, dtype=out, device=DEV) for _ in range(2))
        ops.quantized_rows(*cache_args(cache), pos, seq, slot, table, keys, values, err)
        at = pos.long() % 64
        for got, codes, scales in ((keys, "k", "ks"), (values, "v", "vs")):
            n = cache[codes].view(torch.int8)[page, :, at].view(cache[codes].dtype).float() * cache[scales][page, :, at][..., None]
            assert same(got.float(), n.to(out).float())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_of_few_tokens_writes_what_that_of_many_writes(fmt, dtype):
    nh, nkv, hd = 15, 5, 64
    qkv, pos, seq = step([80], [80], nh, nkv, hd, DTYPES[dtype], 5)
    cos, sin = ref.tables(80, hd, DEV)
    caches, queries, rows = [], [], []
    for piece in (80, 7):
        cache, table = ref.make_cache(fmt, nkv, hd, [80], DEV, 3)
        x = qkv.clone()
        keys, values = (torch.empty((80, nkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
        for a in range(0, 80, piece):
            part = slice(a, min(80, a + piece))
            ops.rope_quantize_append(x[part], pos[part], seq[part], i32([0]), table, cos, sin, *cache_args(cache), nh, nkv, hd, word())
        for a in range(0, 80, piece):
            part = slice(a, min(80, a + piece))
            ops.quantized_rows(*cache_args(cache), pos[part], seq[part], i32([0]), table, keys[part], values[part], word())
        caches.append(cache)
        queries.append(x)
        rows.append((keys, values))
    assert all(same(caches[0][k], caches[1][k]) for k in caches[0]) and same(*queries) and same(rows[0][0], rows[1][0]) and same(rows[0][1], rows[1][1])


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_a_row_is_kept_within_half_a_step(fmt):
    hd, nkv = 64, 2
    cache, table = ref.make_cache(fmt, nkv, hd, [64], DEV, 3)
    qkv, pos, seq = step([64], [64], 2, nkv, hd, torch.float32, 5)
    cos, sin = ref.tables(64, hd, DEV)
    x = qkv.view(64, -1, hd).clone()
    ops.rope_quantize_append(qkv, pos, seq, i32([0]), table, cos, sin, *cache_args(cache), 2, nkv, hd, word())
    keys, values = (torch.empty((64, nkv, hd), device=DEV) for _ in range(2))
    ops.quantized_rows(*cache_args(cache), pos, seq, i32([0]), table, keys, values, word())
    want = x[:, 4:].double()
    amax = want.abs().amax(-1, keepdim=True)
    # int8: half a step of A / 127; e4m3: 2^-4 of the number, or half a step below the smallest normal one (2^-9 of scale A / 448 halved);
    # and float32's own roundings of the factor and the product
    step_ = amax / 254 if fmt == "int8" else torch.maximum(want.abs() * 2.0 ** -4, amax / 448 * 2.0 ** -10)
    assert bool(((values.double() - want).abs() <= step_ + amax * 2.0 ** -21).all())


# ----------------------------------------------------------------------------------------------------- decode
def decode_case(fmt, dtype, nh, nkv, hd, lengths, window=0, splits=None, fused=False, seed=1, spoil=True, change=None, q_pad=0):
    dtype = DTYPES[dtype]
    cache, table = ref.make_cache(fmt, nkv, hd, lengths, DEV, seed, k_size=1.5)
    if spoil:     # what lies behind a sequence's end is not its own: no number at all
        for b, n in enumerate(lengths):
            if n > 0 and n % 64:
                p = int(table[b, n // 64])
                cache["ks"][p, :, n % 64:] = float("nan")
                cache["vs"][p, :, n % 64:] = float("inf")
                if fmt == "fp8":
                    cache["v"].view(torch.int8)[p, :, n % 64:] = 0x7f
                    cache["k"].view(torch.int8)[p, :, n % 64:] = 0x7f
    if change:
        change(cache, table)
    g = torch.Generator().manual_seed(seed + 1)
    B = len(lengths)
    width = (nh + 2 * nkv) * hd if fused else nh * hd
    q = torch.randn((B, width + q_pad), generator=g).to(dtype).to(DEV)
    pos = i32([n - 1 for n in lengths])
    out = torch.full((B, nh * hd + 16), 3.0, dtype=dtype, device=DEV)
    err, scale = word(), 1 / math.sqrt(hd)
    qd = q[:, :width]
    if fused:
        cos, sin = ref.tables(max(max(lengths), 1), hd, DEV)
        at = pos.long().clamp(min=0)
        x = qd.float().view(B, -1, hd)
        turned = ref.rotate(x[:, :nh + nkv], cos[at], sin[at])
        queries, want = turned[:, :nh], {k: v.clone() for k, v in cache.items()}
        for codes, scales, new in (("k", "ks", turned[:, nh:]), ("v", "vs", x[:, nh + nkv:])):
            c, s = ref.quantize(new, fmt)
            for b, n in enumerate(lengths):
                if n > 0:
                    p = int(table[b, (n - 1) // 64])
                    want[codes].view(torch.int8)[p, :, (n - 1) % 64] = c[b].view(torch.int8)
                    want[scales][p, :, (n - 1) % 64] = s[b]
        ops.attn_decode_rope_quantized(qd, out[:, :nh * hd], *cache_args(cache), table, i32(range(B)), pos, cos, sin, B, nh, nkv, hd, scale, n_splits=splits,
                                       err=err, window=window)
        for k in want:
            assert same(cache[k], want[k]), f"the cache's {k} is not what the append writes"
    else:
        queries = qd.float().view(B, nh, hd)
        ops.attn_decode_quantized(qd, out[:, :nh * hd], *cache_args(cache), table, i32(range(B)), pos, B, nh, nkv, hd, scale, n_splits=splits, err=err, window=window)
    assert int(err) == 0
    assert bool((out[:, nh * hd:] == 3.0).all())
    for b, n in enumerate(lengths):
        got = out[b, :nh * hd].view(1, nh, hd)
        if n == 0:
            assert bool((got == 0).all())
            continue
        keys, values = ref.sequence_rows(cache, table[b], n)
        lo = max(0, n - window) if window else 0
        qq = queries[b:b + 1].double()
        exact = ref.attend(qq, n - 1 - lo, keys[lo:], values[lo:], scale, window)
        check(got, exact, off_bound(qq, n - 1 - lo, keys[lo:], values[lo:], scale, window, exact, dtype, not fused))
    return out, cache, table


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 130, 0, 700]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (4, 4, 64), (15, 5, 64), (4, 1, 128), (3, 3, 32), (6, 2, 96), (2, 1, 16), (5, 1, 48), (3, 1, 80), (2, 2, 256),
                                       (8, 1, 64), (9, 1, 64), (24, 2, 112), (7, 1, 192), (2, 1, 208)])
def test_decode_heads_and_lengths(fmt, dtype, nh, nkv, hd):
    for fused in (False, True):
        decode_case(fmt, dtype, nh, nkv, hd, LENGTHS, fused=fused)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8, 16, 40, 128])
@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (4, 1, 128), (11, 1, 256)])
def test_decode_splits(fmt, splits, nh, nkv, hd):
    for fused in (False, True):
        decode_case(fmt, "bf16", nh, nkv, hd, LENGTHS + [3000], splits=splits, fused=fused)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 5000])
@pytest.mark.parametrize("fused", [False, True])
def test_decode_window(window, fused):
    decode_case("int8", "bf16", 9, 3, 64, LENGTHS, window=window, fused=fused)
    decode_case("fp8", "f32", 4, 1, 128, LENGTHS, window=window, fused=fused, splits=3)


def test_decode_long_rows_of_many_tiles():
    # more tiles a warp than a lane holds pages of, with and without splits
    decode_case("int8", "bf16", 4, 1, 64, [64 * 64 * 9 + 5, 40], splits=1)
    decode_case("fp8", "bf16", 3, 1, 256, [64 * 150 + 1, 64 * 33], splits=2, fused=True)


def test_decode_window_does_not_touch_pages_before_it():
    def gone(cache, table):
        table[0, :10] = -1
    dtype = torch.bfloat16
    cache, table = ref.make_cache("int8", 2, 64, [700], DEV, 5)
    q = torch.randn((1, 4 * 64), device=DEV).to(dtype)
    outs = []
    for t in (table, table.clone()):
        if outs:
            t[0, :9] = -1       # pages 0 .. 8 hold keys up to 575; the window of 100 starts at 600
        out, err = torch.empty((1, 256), dtype=dtype, device=DEV), word()
        ops.attn_decode_quantized(q, out, *cache_args(cache), t, i32([0]), i32([699]), 1, 4, 2, 64, 0.125, window=100, err=err)
        assert int(err) == 0
        outs.append(out)
    assert torch.equal(*outs)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_scales_of_all_sizes(fmt, dtype):
    # values whose rows differ by many orders of magnitude, and rows of zeros among them: no weight leaves float16's range
    def change(cache, table):
        g = torch.Generator().manual_seed(9)
        cache["vs"].mul_((10.0 ** (torch.rand(cache["vs"].shape, generator=g) * 40 - 20)).to(DEV))
        cache["v"].view(torch.int8)[:, :, ::7] = 0
        cache["vs"][:, :, ::7] = 2.0 ** -60 / ref.TOP[fmt]
    decode_case(fmt, dtype, 9, 3, 64, [1, 8, 65, 700], change=change, spoil=False)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_decode_a_row_that_is_no_number_reaches_who_sees_it(fmt):
    def change(cache, table):
        cache["vs"][int(table[0, 1]), 0, 5] = float("nan")       # value of position 69, kv head 0
        cache["v"].view(torch.int8)[int(table[0, 1]), 0, 5] = 0
        cache["ks"][int(table[1, 0]), 1, 3] = float("nan")       # key of position 3, kv head 1
        cache["k"].view(torch.int8)[int(table[1, 0]), 1, 3] = 0
    for splits in (1, 4, 24):
        out, _, _ = decode_case(fmt, "bf16", 4, 2, 64, [130, 130, 130], change=change, spoil=False, splits=splits)
        nan = torch.isnan(out[:, :256].view(3, 4, 64)).all(-1)
        assert nan.tolist() == [[True, True, False, False], [False, False, True, True], [False] * 4]
    # outside of the window nobody sees them
    out, _, _ = decode_case(fmt, "bf16", 4, 2, 64, [130, 130, 130], change=change, spoil=False, window=50)
    assert not bool(torch.isnan(out).any())


def test_decode_equal_scores_and_scores_far_apart():
    def far(cache, table):
        cache["ks"].mul_(200.0)
    decode_case("int8", "bf16", 4, 2, 64, [1, 130, 700], spoil=False, change=lambda c, t: c["ks"].zero_())
    cache, table = ref.make_cache("int8", 1, 64, [200], DEV, 5)
    cache["ks"].mul_(1e4)
    keys, values = ref.sequence_rows(cache, table[0], 200)
    q = torch.randn((40, 64), generator=torch.Generator().manual_seed(6)).to(DEV)
    apart = 0
    for row in q.split(1):
        out = torch.empty((1, 64), device=DEV)
        ops.attn_decode_quantized(row, out, *cache_args(cache), table, i32([0]), i32([199]), 1, 1, 1, 64, 0.125)
        s = (keys[:, 0] @ row[0].double()) * 0.125
        if float(s.topk(2).values.diff().abs()) > 100:       # (the others' weights are below 2^-144 of the largest, none as operands)
            apart += 1
            assert torch.allclose(out[0].double(), values[int(s.argmax()), 0], rtol=2.0 ** -20, atol=0)
    assert apart >= 20


def test_decode_rows_lie_where_the_strides_say():
    decode_case("int8", "bf16", 9, 3, 64, LENGTHS, q_pad=24)
    decode_case("fp8", "f32", 9, 3, 64, LENGTHS, q_pad=3, fused=True)
    decode_case("fp8", "bf16", 9, 3, 48, LENGTHS, q_pad=5, fused=True)


def test_decode_scratch():
    # one's own, of the size asked for; a smaller one is refused; results do not depend on what it held
    cache, table = ref.make_cache("int8", 2, 64, [3000, 5, 0], DEV, 3)
    q, outs = torch.randn((3, 4 * 64), device=DEV).bfloat16(), []
    room = ops.quantized_decode_scratch_floats(3, 4, 64, 32)
    assert room == 3 * 4 * 4 * 66 and ops.quantized_decode_scratch_floats(3, 4, 64, 8) == 0
    for fill in (0.0, float("nan"), None):
        scratch = torch.full((room,), fill, device=DEV) if fill is not None else None
        outs.append(torch.empty((3, 256), dtype=torch.bfloat16, device=DEV))
        ops.attn_decode_quantized(q, outs[-1], *cache_args(cache), table, i32(range(3)), i32([2999, 4, -1]), 3, 4, 2, 64, 0.125, n_splits=32, scratch=scratch)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and bool((outs[0][2] == 0).all())
    with pytest.raises(ops.KernelError, match="scratch"):
        ops.attn_decode_quantized(q, outs[0], *cache_args(cache), table, i32(range(3)), i32([2999, 4, -1]), 3, 4, 2, 64, 0.125, n_splits=32,
                                  scratch=torch.empty(room - 1, device=DEV))


def test_decode_repeats_itself_and_leaves_the_rest():
    a = decode_case("fp8", "bf16", 9, 3, 64, [1300, 5, 64], splits=8)[0]
    b = decode_case("fp8", "bf16", 9, 3, 64, [1300, 5, 64], splits=8)[0]
    assert torch.equal(a, b)


def test_decode_in_a_graph_and_on_a_stream_of_its_own():
    nh, nkv, hd, lengths = 9, 3, 64, [130, 700, 64]
    cache, table = ref.make_cache("int8", nkv, hd, lengths, DEV, 3)
    cos, sin = ref.tables(800, hd, DEV)
    qkv = torch.randn((3, (nh + 2 * nkv) * hd), device=DEV).bfloat16()
    pos, slot, err = i32([n - 1 for n in lengths]), i32(range(3)), word()
    out = torch.empty((3, nh * hd), dtype=torch.bfloat16, device=DEV)
    run = lambda o: ops.attn_decode_rope_quantized(qkv, o, *cache_args(cache), table, slot, pos, cos, sin, 3, nh, nkv, hd, 0.125, err=err)   # noqa: E731
    run(out)
    torch.cuda.synchronize()
    graph, captured = torch.cuda.CUDAGraph(), torch.zeros_like(out)
    with torch.cuda.graph(graph):
        run(captured)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, captured)
    qkv.copy_(torch.randn_like(qkv.float()).bfloat16())
    pos += 1                                                     # (the third sequence's new token starts a page that it does not have)
    pos[2] = 63
    graph.replay()
    fresh = torch.zeros_like(out)
    run(fresh)
    torch.cuda.synchronize()
    assert torch.equal(fresh, captured) and not torch.equal(fresh, out) and int(err) == 0
    side, other = torch.cuda.Stream(), torch.zeros_like(out)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(other)
    side.synchronize()
    assert torch.equal(other, fresh)


def test_no_sequences_and_no_tokens():
    cache, table = ref.make_cache("int8", 1, 64, [3], DEV, 3)
    cos, sin = ref.tables(8, 64, DEV)
    none, err = i32([]), word()
    ops.rope_quantize_append(torch.empty((0, 192), device=DEV), none, none, i32([0]), table, cos, sin, *cache_args(cache), 1, 1, 64, err)
    ops.quantized_rows(*cache_args(cache), none, none, i32([0]), table, torch.empty((0, 1, 64), device=DEV), torch.empty((0, 1, 64), device=DEV), err)
    ops.attn_decode_quantized(torch.empty((0, 64), device=DEV), torch.empty((0, 64), device=DEV), *cache_args(cache), table, none, none, 0, 1, 1, 64, 0.1)
    assert int(err) == 0


def test_pages_and_positions_that_are_not_there_are_reported():
    nh, nkv, hd = 2, 1, 64
    cos, sin = ref.tables(128, hd, DEV)
    for bad, table_change, positions in ((2, None, [128, 3]), (2, None, [-1, 3]), (4, -1, [70, 3]), (4, 99, [70, 3])):
        cache, table = ref.make_cache("int8", nkv, hd, [128, 64], DEV, 3)
        if table_change is not None:
            table[0, 1] = table_change
        before = {k: v.clone() for k, v in cache.items()}
        qkv = torch.randn((2, (nh + 2 * nkv) * hd), device=DEV)
        err = word()
        ops.rope_quantize_append(qkv, i32(positions), i32([0, 1]), i32([0, 1]), table, cos, sin, *cache_args(cache), nh, nkv, hd, err)
        assert int(err) == bad
        page = int(table[1, 0])
        for k in cache:     # the good token's row is written, nothing else
            before[k].view(torch.int8 if before[k].element_size() == 1 else torch.float32)[page, :, 3] = \
                cache[k].view(torch.int8 if cache[k].element_size() == 1 else torch.float32)[page, :, 3]
            assert same(cache[k], before[k])
        if positions[0] == 70:
            err = word()
            out = torch.empty((2, nh * hd), device=DEV)
            ops.attn_decode_rope_quantized(qkv, out, *cache_args(cache), table, i32([0, 1]), i32(positions), cos, sin, 2, nh, nkv, hd, 0.1, err=err)
            assert int(err) == 4
            err = word()
            keys, values = (torch.ones((2, nkv, hd), device=DEV) for _ in range(2))
            ops.quantized_rows(*cache_args(cache), i32(positions), i32([0, 1]), i32([0, 1]), table, keys, values, err)
            assert int(err) == 4 and bool((keys[0] == 0).all()) and bool((keys[1] != 0).any())
    # a position behind the rotation table
    cache, table = ref.make_cache("int8", nkv, hd, [192], DEV, 3)
    before, err = cache["k"].clone(), word()
    out = torch.empty((1, nh * hd), device=DEV)
    ops.attn_decode_rope_quantized(torch.randn((1, (nh + 2 * nkv) * hd), device=DEV), out, *cache_args(cache), table, i32([0]), i32([130]), cos, sin, 1, nh, nkv, hd,
                                   0.1, err=err)
    assert int(err) == 2 and same(before, cache["k"])
