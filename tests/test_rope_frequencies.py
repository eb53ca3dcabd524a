"""Arguments from which rope_frequencies' "parts" cannot find its pairs are refused (no GPU)."""
import math

import pytest

import cuda_attn


@pytest.mark.parametrize("kw", [dict(base=1.0), dict(base=0.5), dict(base=math.inf), dict(factor=math.inf), dict(original=math.inf), dict(high=math.inf)])
def test_refused(kw):
    with pytest.raises(RuntimeError, match="'parts' takes"):
        cuda_attn.rope_frequencies(64, **{"scaling": "parts", "factor": 4.0, **kw})


def test_base_one_turns_all_pairs_alike():
    f, scale = cuda_attn.rope_frequencies(8, 1.0, scaling="linear", factor=2.0)
    assert f.tolist() == [0.5] * 4 and scale == 1.0
