"""Refusals of `LlamaDecoder.choose` that need no GPU."""
import math
import types

import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("temperature", [0, 0.0, -1.0, math.nan])
def test_temperatures_that_give_no_distribution(temperature):
    """Zero, for one, made probabilities of NaN: no word had any, and -1 came back as the token."""
    from alignedkv_b200.llama import LlamaDecoder
    with pytest.raises(RuntimeError, match="temperature"):
        LlamaDecoder.choose(None, torch.zeros(1, 2, 4), None, torch.zeros(1, 2, dtype=torch.long), torch.zeros(1, 2), temperature=temperature)


@pytest.mark.parametrize("parents", [[-1, 0, 0], [-1, -1, 0], [[-1, 0, 1], [-1, 0, 0]]])
def test_trees_over_a_paged_cache(parents):
    """Of a tree's path nodes 0, 2, say, the count of 2 would have let the tokens of nodes 0 and 1 enter the cache."""
    from alignedkv_b200.llama import LlamaDecoder
    paged = types.SimpleNamespace(attention="paged")
    with pytest.raises(RuntimeError, match="chains"):
        LlamaDecoder.choose(paged, torch.zeros(1, 3, 4), None, torch.zeros(1, 3, dtype=torch.long), torch.zeros(1, 3), torch.tensor(parents))
