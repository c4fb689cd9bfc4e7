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
