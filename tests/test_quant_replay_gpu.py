"""Steps over an 8-bit cache that are replayed from captured graphs: what they give does not hang on which steps came before."""
import numpy as np
import pytest

import helpers as H
from edgelm_b200.engine.engine import Engine, StepEntry

pytestmark = pytest.mark.gpu
FORMATS = ["int8", "fp8"]


@pytest.fixture(scope="module")
def model_dir(tmp_path_factory):
    return H.make_model_dir(tmp_path_factory.mktemp("models"), "tiny_d")


def continued(eng, before, new, salt):
    """Logits of `new` tokens behind `before` others."""
    toks = H.tokens_for("tiny_d", before + new, salt)
    slot = eng.open(1)[0]
    eng.step([StepEntry(slot, toks[:before], [])])
    out = eng.step([StepEntry(slot, toks[before:], list(range(new)))]).cpu().numpy()
    eng.close([slot])
    eng.check_device_errors()
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_shape_captured_at_one_length_is_not_replayed_at_another(model_dir, dtype, fmt):
    """40 new tokens behind 10 (one page: mma.sync), behind 100 and behind 700 (several blocks share the keys): each the same bits as an
    engine without graphs gives, whichever was captured first, and each replayed at its own length."""
    eager = Engine.from_dir(model_dir, dtype=dtype, max_tokens=2048, cache_format=fmt, use_graphs=False)
    for lengths in ((10, 100, 700), (700, 10, 300)):
        eng = Engine.from_dir(model_dir, dtype=dtype, max_tokens=2048, cache_format=fmt)
        for before in lengths:
            for salt in range(3):
                assert np.array_equal(continued(eng, before, 40, salt), continued(eager, before, 40, salt)), (lengths, before, salt)
        kept = [key for key in eng._step_graphs if key[0] == (40,)]
        assert len(kept) == len(lengths)
        for before in lengths:      # (and once more, all of them captured)
            assert np.array_equal(continued(eng, before + 3, 40, 9), continued(eager, before + 3, 40, 9))
        assert [key for key in eng._step_graphs if key[0] == (40,)] == kept
