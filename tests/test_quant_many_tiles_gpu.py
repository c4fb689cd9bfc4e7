"""Prompt attention over the 8-bit cache for steps of very many sequences."""
import pytest
import torch

import helpers as H
from edgelm_b200.csrc import ops
from tests import quant_reference as ref
from tests.test_quant_cache_gpu import DEV, cache_args, i32, word
from tests.test_quant_prefill_gpu import tiles_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,form", [(torch.bfloat16, 2), (torch.bfloat16, 1), (torch.float32, 1)])
def test_more_tiles_than_one_grid_takes(dtype, form):
    """2,500 sequences of one to three tokens, 32 query heads on one kv head: more blocks than a grid's 65,535, and the same bits as in pieces."""
    nh, hd, n = 32, 16, 2500
    news = [1 + i % 3 for i in range(n)]
    totals = [m + i % 5 for i, m in enumerate(news)]
    cache, table = ref.make_cache("int8", 1, hd, totals, DEV, 3)
    q = torch.randn((sum(news), nh * hd), generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    tiles, n_tiles = tiles_of(totals, news)
    out, pieces, err = torch.zeros_like(q), torch.zeros_like(q), word()
    call = lambda o, t, k: ops.attn_prefill_quantized(q, o, *cache_args(cache), table, i32(range(n)), *t, k, nh, 1, hd, 0.25, err=err, n_splits=1, form=form)   # noqa: E731
    call(out, tiles, n_tiles)
    for a in range(0, n, 1000):
        part = [t[a:a + 1000].contiguous() for t in tiles]
        call(pieces, part, part[0].numel())
    assert int(err) == 0 and torch.equal(out, pieces) and bool(out.isfinite().all()) and bool((out != 0).any(1).all())


@pytest.mark.parametrize("dtype,form", [(torch.bfloat16, 2), (torch.bfloat16, 1), (torch.float32, 1)])
def test_the_longest_tile_as_the_caller_knows_it(dtype, form):
    """Blocks counted by the step's longest tile give what blocks for whole tiles give; a number that no tile has is refused."""
    nh, nkv, hd, news = 9, 3, 64, [17, 3, 1, 17, 9]
    totals = [400, 3, 200, 64, 130]
    cache, table = ref.make_cache("fp8", nkv, hd, totals, DEV, 3)
    q = torch.randn((sum(news) + 90, nh * hd), generator=torch.Generator().manual_seed(4)).to(dtype).to(DEV)
    tiles, n_tiles = tiles_of(totals, news)
    outs, err = [], word()
    for window in (0, 100):
        for most in (0, 17, 20, 128):
            outs.append(torch.zeros_like(q))
            ops.attn_prefill_quantized(q, outs[-1], *cache_args(cache), table, i32(range(5)), *tiles, n_tiles, nh, nkv, hd, 0.125, err=err, n_splits=2, form=form,
                                       window=window, max_tile_tokens=most)
            assert torch.equal(outs[-1], outs[len(outs) // 5 * 4])
    assert int(err) == 0 and bool((outs[0][sum(news):] == 0).all())
    for most in (-1, 129):
        with pytest.raises(ops.KernelError, match="1 to 128"):
            ops.attn_prefill_quantized(q, outs[0], *cache_args(cache), table, i32(range(5)), *tiles, n_tiles, nh, nkv, hd, 0.125, max_tile_tokens=most)


def test_an_engine_says_how_long_its_tiles_are(tmp_path, monkeypatch):
    from edgelm_b200.engine.engine import Engine, StepEntry
    eng = Engine.from_dir(H.make_model_dir(tmp_path, "tiny_d"), dtype="bfloat16", max_tokens=4096, cache_format="int8", use_graphs=False)
    told, real = [], ops.attn_prefill_quantized
    monkeypatch.setattr(ops, "attn_prefill_quantized", lambda *a, **kw: (told.append(kw["max_tile_tokens"]), real(*a, **kw)))
    slots = eng.open(8)
    for news in ([17] * 8, [1] * 7 + [5], [300] + [2] * 7):
        told.clear()
        eng.step([StepEntry(s, H.tokens_for("tiny_d", n, i), [n - 1]) for i, (s, n) in enumerate(zip(slots, news))])
        assert told and set(told) == {min(128, max(news))}
    eng.check_device_errors()
