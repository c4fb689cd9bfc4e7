"""The 8-bit cache's host side: what it stores, accounts for, and refuses."""
import pytest
import torch

import edgelm_b200
import helpers as H
from edgelm_b200.cache import CacheError, SequenceCache
from edgelm_b200.config import ConfigError, config_class_for
from edgelm_b200.engine.engine import EngineError
from edgelm_b200.engine.model import DecoderModel
from edgelm_b200.parts.base import KVNeed, NeedSet, StateNeed
from edgelm_b200.presets import preset_config

BOTH = ("int8", "fp8")


@pytest.mark.parametrize("fmt,dtype", [("int8", torch.int8), ("fp8", torch.float8_e4m3fn)])
def test_storage_and_accounts(fmt, dtype):
    needs = [KVNeed(2, 48, formats=BOTH), None, KVNeed(2, 48, formats=BOTH), StateNeed((3,)), NeedSet.of(kv=KVNeed(1, 16, window=100, formats=BOTH), s=StateNeed((2,)))]
    c = SequenceCache(needs, 5 * 64, 256, device="cpu", dtype=torch.bfloat16, max_seqs=2, format=fmt)
    plain = SequenceCache(needs, 5 * 64, 256, device="cpu", dtype=torch.bfloat16, max_seqs=2)
    e = c.entries[0]
    assert e.k.dtype == e.v.dtype == dtype and e.k.shape == (5, 2, 64, 48) and e.k_scale.shape == e.v_scale.shape == (5, 2, 64) and e.k_scale.dtype == torch.float32
    assert c.entries[2].k_scale.data_ptr() != e.k_scale.data_ptr() and c.entries[4]["kv"].group.format == fmt
    assert plain.entries[0].group.format is None and plain.entries[0].k.dtype == torch.bfloat16
    # a byte a number, and 8 bytes of scales for a key row and a value row
    assert c.bytes_per_token() == 2 * 2 * (2 * 48 + 8) + 1 * (2 * 16 + 8)
    assert c.storage_bytes() == sum(t.numel() * t.element_size() for g in c.kv_groups for t in (g.k, g.v, g.k_scale, g.v_scale)) + \
        sum(g.state.numel() * 4 for g in c.state_groups)
    assert any(f"{fmt} codes" in line for line in c.describe()) and not any("codes" in line for line in plain.describe())
    for cache in (c, plain):      # the bookkeeping does not know the difference
        s = cache.open_many(2)
        cache.reserve(s[0], 130)
        cache.advance(s[0], 130)
        cache.reserve_next([s[0]])
        cache.check()
        assert cache.footprint(130) == plain.footprint(130)
        cache.close(s[0])
        cache.check()


def test_needs_that_differ_in_their_formats_alone_are_one():
    assert KVNeed(2, 48, formats=BOTH) == KVNeed(2, 48) and hash(KVNeed(2, 48, formats=BOTH)) == hash(KVNeed(2, 48))


def test_refusals():
    ok = KVNeed(2, 48, formats=BOTH)
    with pytest.raises(CacheError, match="known: int8, fp8"):
        SequenceCache([ok], 64, 64, format="int4")
    for need in (KVNeed(2, 48), KVNeed(2, 48, formats=("int8",)), KVNeed(2, 48, formats=BOTH, pool=8), KVNeed(2, 48, formats=BOTH, values_in_keys=True),
                 KVNeed(2, 48, formats=BOTH, v_head_dim=32), NeedSet.of(a=StateNeed((1,)), b=KVNeed(1, 16))):
        with pytest.raises(CacheError, match="schedule entry 1"):
            SequenceCache([ok, need], 64, 64, format="fp8")
        SequenceCache([ok, need], 64, 64)


def model(cfg_dict):
    return DecoderModel(config_class_for(cfg_dict).from_dict(cfg_dict).plan())


@pytest.mark.parametrize("preset", ["smollm2-135m", "smollm2-360m", "smollm2-1.7b"])
def test_llama_models_take_both_formats(preset):
    m = DecoderModel(preset_config(preset).plan())
    for fmt in BOTH:
        m.check_cache_format(fmt)
        assert 128 in m.tile_sizes(fmt)
        c = SequenceCache(m.cache_needs(), 256, 8192, format=fmt)
        assert c.bytes_per_token() < SequenceCache(m.cache_needs(), 256, 8192, dtype=torch.bfloat16).bytes_per_token() * 0.54


@pytest.mark.parametrize("preset", ["sagizen-576", "vosulorn-576", "redenex-576", "radupel-576", "sarizen-576", "semadra-576"])
def test_models_whose_attention_reads_no_codes_refuse(preset):
    m = DecoderModel(preset_config(preset).plan())
    with pytest.raises((CacheError, ConfigError)):
        m.check_cache_format("int8")
        SequenceCache(m.cache_needs(), 256, 8192, format="int8")


def test_the_command_line_knows_the_formats(capsys):
    from edgelm_b200.cli import build_parser
    assert build_parser().parse_args(["run", "--preset", "x", "--cache", "fp8"]).cache == "fp8"
    assert build_parser().parse_args(["bench", "--preset", "x"]).cache is None
    with pytest.raises(SystemExit):
        build_parser().parse_args(["run", "--cache", "int4"])
    assert H.TINY       # (the tiny models that the engine's tests run)


@pytest.mark.parametrize("kept,asked", [(None, "int8"), ("int8", "fp8")])
def test_a_ready_engine_with_another_format_is_refused(kept, asked):
    class Ready:
        class cache:
            format = kept
    with pytest.raises(EngineError, match=asked):
        edgelm_b200.Session("nowhere", engine=Ready(), cache_format=asked)
    with pytest.raises(EngineError, match=asked):
        edgelm_b200.generate("nowhere", [[1]], engine=Ready(), cache_format=asked)
