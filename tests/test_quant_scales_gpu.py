"""Prompt and decode attention over the 8-bit cache where scales differ within a block of keys, and where the rounding of a key's factor shows."""
import math

import pytest
import torch

import helpers as H
from edgelm_b200.csrc import ops
from tests import quant_reference as ref
from tests.test_quant_cache_gpu import DEV, cache_args, check, i32, off_bound, word
from tests.test_quant_prefill_gpu import tiles_of

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def tcgen05_bound(q, first, keys, values, scale, exact, largest_scale):
    """How far an output of the tcgen05 kernel may be.  A key's tile holds a_j (u_j / 2^k) as float16: u_j / 2^k rounded, then its product with the
    code, 2^-11 each; a lifted query 2^-11 at the most (its numbers below 2^-14 of the row's largest): a score is off by d = 3 x 2^-11 sum |q_i k_i| scale and
    float32's 2^-20 of its terms, every weight by a factor within exp(+-d), numerator and denominator.  Values: twice 2^-11; weights 2^-11; the output
    once.  Weights: the reference lags by up to 2^8, so the largest weight is 2^6 to 2^14 as an operand and a key adds up to 2^-31 of the largest weighted row.  Values far
    below their group's largest scale: half of float16's smallest step, 2^-25 of it."""
    g = q.shape[1] // keys.shape[1]
    size = (torch.einsum("nhd,lhd->hnl", q.abs(), keys.abs().repeat_interleave(g, 1)) * scale).amax(-1)
    d = 3 * 2.0 ** -11 * size + 2.0 ** -20 * (size + 32.0)
    a = ref.attend(q, first, keys, values.abs(), scale)
    floor = 2.0 ** -31 * (first + q.shape[0]) * ref.attend(q, first, keys, values.abs().amax(-1, keepdim=True), scale) + 2.0 ** -25 * largest_scale
    return floor + exact.abs() * torch.finfo(BF16).eps / 2 + a * (torch.expm1(2 * d).T[..., None] + 3 * 2.0 ** -11 + 2.0 ** -20)


def mixed(cache, wild_keys, wild_values, seed=9):
    """Groups of 32 keys of both kinds side by side: scales within 2^3 of one another in the first half of a page, up to 2^14 apart in the second (only
    ever smaller than they were, so that scores stay what they are at the most)."""
    g = torch.Generator().manual_seed(seed)
    for name, wild in (("ks", wild_keys), ("vs", wild_values)):
        steps = torch.randint(0, 4, cache[name].shape, generator=g)
        if wild:
            steps[..., 32:] = torch.randint(0, 15, cache[name][..., 32:].shape, generator=g)
        cache[name].mul_((2.0 ** -steps).to(DEV))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("wild_keys,wild_values", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("nh,nkv,hd,splits", [(4, 2, 64, 1), (8, 1, 128, 1), (3, 1, 80, 3), (2, 2, 16, 8)])
def test_groups_of_both_kinds_in_one_block(fmt, wild_keys, wild_values, nh, nkv, hd, splits):
    total, n, scale = 900, 200, 1 / math.sqrt(hd)
    cache, table = ref.make_cache(fmt, nkv, hd, [total], DEV, 3, k_size=1.5)
    mixed(cache, wild_keys, wild_values)
    q = torch.randn((n, nh * hd), generator=torch.Generator().manual_seed(4)).to(BF16).to(DEV)
    out, err, (tiles, n_tiles) = torch.empty_like(q), word(), tiles_of([total], [n])
    ops.attn_prefill_quantized(q, out, *cache_args(cache), table, i32([0]), *tiles, n_tiles, nh, nkv, hd, scale, err=err, n_splits=splits, form=2)
    assert int(err) == 0
    keys, values = ref.sequence_rows(cache, table[0], total)
    qq = q.double().view(n, nh, hd)
    exact = ref.attend(qq, total - n, keys, values, scale)
    check(out.view(n, nh, hd), exact, tcgen05_bound(qq, total - n, keys, values, scale, exact, float(cache["vs"].max())))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_key_scales_of_all_sizes(fmt, dtype):
    """Spread key scales in the other kernels: decode, and prompts on mma.sync."""
    dtype = {"bf16": BF16, "f32": torch.float32}[dtype]
    nh, nkv, hd, total, n, scale = 9, 3, 64, 700, 90, 0.125
    cache, table = ref.make_cache(fmt, nkv, hd, [total], DEV, 3, k_size=1.5)
    mixed(cache, True, True)
    q = torch.randn((n, nh * hd), generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    keys, values = ref.sequence_rows(cache, table[0], total)
    qq = q.double().view(n, nh, hd)
    exact = ref.attend(qq, total - n, keys, values, scale)
    bound = off_bound(qq, total - n, keys, values, scale, 0, exact, dtype, True)
    out, err, (tiles, n_tiles) = torch.empty_like(q), word(), tiles_of([total], [n])
    ops.attn_prefill_quantized(q, out, *cache_args(cache), table, i32([0]), *tiles, n_tiles, nh, nkv, hd, scale, err=err, form=1)
    check(out.view(n, nh, hd), exact, bound)
    out = torch.empty_like(q)
    ops.attn_decode_quantized(q, out, *cache_args(cache), table.expand(n, -1), i32(range(n)), i32(range(total - n, total)), n, nh, nkv, hd, scale, err=err)
    check(out.view(n, nh, hd), exact, bound)
    assert int(err) == 0


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("hd", [64, 128])
def test_two_keys_of_nearly_the_same_large_score(fmt, hd):
    """Two keys share a row's weight, their scores near 60 and up to 2 apart, their scales different: what the rounding of a key's
    factor (common to all of its products, so that it does not average out) does to the weights stays within the bound."""
    nh, total, n, scale = 2, 200, 128, 1 / math.sqrt(hd)
    cache, table = ref.make_cache(fmt, 1, hd, [total], DEV, 3)
    g = torch.Generator().manual_seed(5)
    row = torch.randn(hd, generator=g)
    top = ref.TOP[fmt]
    for place, (factor, at) in {5: (1.37, 0), 70: (1.91, 1)}.items():      # the same direction, another scale: other bits of the factor
        codes, s = ref.quantize(row * factor, fmt)
        page = int(table[0, place // 64])
        cache["k"].view(torch.int8)[page, 0, place % 64] = codes.view(torch.int8).to(DEV)
        cache["ks"][page, 0, place % 64] = float(s) / factor * (1.0 + 0.03 * at)
    keys, values = ref.sequence_rows(cache, table[0], total)
    size = 60.0 / float((row.double() ** 2).sum() * scale)
    q = (row * size * (1 + 0.02 * torch.randn((n, nh, 1), generator=g))).to(BF16).to(DEV)
    exact = ref.attend(q.double(), total - n, keys, values, scale)
    s = torch.einsum("nhd,lhd->hnl", q.double(), keys.expand(-1, nh, -1))[..., [5, 70]] * scale
    assert bool(((s > 50) & (s < 70)).all()) and bool(((s[..., 1] - s[..., 0]).abs() < 2.5).all())
    out, err, (tiles, n_tiles) = torch.empty((n, nh * hd), dtype=BF16, device=DEV), word(), tiles_of([total], [n])
    ops.attn_prefill_quantized(q.view(n, -1), out, *cache_args(cache), table, i32([0]), *tiles, n_tiles, nh, 1, hd, scale, err=err, form=2)
    assert int(err) == 0
    check(out.view(n, nh, hd), exact, tcgen05_bound(q.double(), total - n, keys, values, scale, exact, float(cache["vs"].max())))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd,lengths", [(9, 3, 64, [130]), (15, 5, 64, [3, 130, 70, 1]), (16, 4, 128, [65]), (4, 1, 256, [17])])
def test_short_sequences_under_a_wide_table(dtype, nh, nkv, hd, lengths):
    """An engine's table is as wide as its pool, and the default split counts by it: most blocks of most clusters have no key, and the fold
    runs over them.  As close to the plain statement as under a table that fits, with scratch that held anything."""
    dtype = {"bf16": BF16, "f32": torch.float32}[dtype]
    B, scale = len(lengths), 1 / math.sqrt(hd)
    cache, table = ref.make_cache("int8", nkv, hd, lengths, DEV, 3, k_size=1.5)
    wide = torch.full((B, 1024), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    splits = ops.quantized_decode_splits(B, nh, nkv, hd, 1024 * 64)
    assert splits > 1
    q = torch.randn((B, nh * hd), generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    room = ops.quantized_decode_scratch_floats(B, nh, hd, splits)
    for t in (table, wide):
        out, err = torch.empty_like(q), word()
        ops.attn_decode_quantized(q, out, *cache_args(cache), t, i32(range(B)), i32(n - 1 for n in lengths), B, nh, nkv, hd, scale, err=err,
                                  scratch=torch.full((max(room, 1),), float("nan"), device=DEV))
        assert int(err) == 0
        for b, n in enumerate(lengths):
            keys, values = ref.sequence_rows(cache, table[b], n)
            qq = q[b:b + 1].double().view(1, nh, hd)
            exact = ref.attend(qq, n - 1, keys, values, scale)
            check(out[b].view(1, nh, hd), exact, off_bound(qq, n - 1, keys, values, scale, 0, exact, dtype, True))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_generated_tokens_are_among_the_best(tmp_path, fmt):
    """bfloat16: every token that captured decode steps choose has a logit within the model's tolerance of the largest, by eager single
    steps that are fed the same tokens."""
    from edgelm_b200 import generate
    from edgelm_b200.engine.engine import Engine, StepEntry
    path = H.make_model_dir(tmp_path, "tiny_d")
    eng = Engine.from_dir(path, dtype="bfloat16", max_tokens=2048, cache_format=fmt)
    eager = Engine.from_dir(path, dtype="bfloat16", max_tokens=2048, cache_format=fmt, use_graphs=False)
    prompts = [H.tokens_for("tiny_d", n, n) for n in (70, 3, 129)]
    for prompt, toks in zip(prompts, generate(None, prompts, n=40, engine=eng, slots=3, ignore_eos=True)):
        slot = eager.open(1)[0]
        logits = eager.step([StepEntry(slot, prompt, [len(prompt) - 1])])[0]
        for t in toks:
            # (two engines' logits, each within the tolerance of the model's largest)
            assert float(logits.max() - logits[t]) <= 2 * H.TOL["bfloat16"] * float(logits.abs().max())
            logits = eager.step([StepEntry(slot, [t], [0])])[0]
        eager.close([slot])
    eager.check_device_errors()
