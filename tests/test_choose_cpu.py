"""Refusals of `LlamaDecoder.choose` that need no GPU."""
import math

import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("temperature", [0, 0.0, -1.0, math.nan])
def test_temperatures_that_give_no_distribution(temperature):
    """Zero, for one, made probabilities of NaN: no word had any, and -1 came back as the token."""
    from alignedkv_b200.llama import LlamaDecoder
    with pytest.raises(RuntimeError, match="temperature"):
        LlamaDecoder.choose(None, torch.zeros(1, 2, 4), None, torch.zeros(1, 2, dtype=torch.long), torch.zeros(1, 2), temperature=temperature)
