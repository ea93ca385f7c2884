"""What an eviction asks of a layer and leaves of it: votes, masks, snapshots."""
import math

import pytest
import torch

from test_gpu_evict import dense, expect, filled, weigh

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_without_votes(akv_lib):
    """Sums that nobody has formed say nothing about which tokens are heavy: refused, unless `recent` alone decides."""
    layer, _, _, _ = filled(1, 2, 300, 128, seed=1)
    with pytest.raises(RuntimeError, match="weights"):
        layer.evict(128, 64)
    assert (layer.rest_start, layer.cache_len, layer.evictions) == (256, 300, 0) and layer.weights is None
    k, v = (t.clone() for t in dense(layer))
    layer.evict(128, recent=128)
    assert (layer.rest_start, layer.cache_len, layer.evictions) == (128, 172, 1)
    # the second half moved into the first, in order
    assert torch.equal(dense(layer)[0], k[:, :, 128:]) and torch.equal(dense(layer)[1], v[:, :, 128:])
    assert torch.equal(layer.positions[..., :128], torch.arange(128, 256, dtype=torch.int32, device=DEV).expand(1, 2, -1))
    with pytest.raises(RuntimeError, match="weights"):
        layer.evict(64)                               # a window does not vote either


def test_nothing_to_evict(akv_lib):
    """keep == the tokens in the planes: all stay in their places, so masks and older snapshots still hold."""
    layer, k, v, gen = filled(2, 2, 200, 128, seed=2, room=100)
    weigh(layer, gen)
    early = layer.snapshot()
    for i in range(2):
        layer.tree_commit(*(torch.randn(2, 40, 2, 128, device=DEV, generator=gen).half() for _ in range(2)),
                          torch.arange(40, dtype=torch.int32, device=DEV).expand(2, -1).contiguous())
        if i == 0:
            expect(layer, 192, 64)
            late = layer.snapshot()
    q, one = torch.randn(2, 1, 2, 128, device=DEV, generator=gen).half(), torch.ones(1, 1, dtype=torch.bool, device=DEV)
    layer.tree_attention(q, q, q, one, mask=torch.zeros(2, 1, 1, 300, dtype=torch.half, device=DEV))
    layer.decode(q, q, q, mask=torch.zeros(2, 1, 1, 300, dtype=torch.half, device=DEV))
    with pytest.raises(RuntimeError, match="overwritten"):
        layer.restore(early)                          # (a block has filled up since: its residual tokens are gone)
    assert late["evictions"] == layer.evictions == 0


def test_snapshot_over_an_eviction_of_nothing(akv_lib):
    layer, _, _, gen = filled(1, 2, 128, 64, seed=3, room=200)
    weigh(layer, gen)
    snap = layer.snapshot()
    new = lambda n: torch.randn(1, n, 2, 64, device=DEV, generator=gen).half()  # noqa: E731
    layer.tree_commit(new(64), new(64), torch.arange(64, dtype=torch.int32, device=DEV)[None])
    expect(layer, 192, 0)
    layer.restore(snap)
    assert (layer.cache_len, layer.rest_start) == (128, 128)
    weigh(layer, gen)
    layer.tree_commit(new(64), new(64), torch.arange(64, dtype=torch.int32, device=DEV)[None])
    expect(layer, 64, 32)                             # (places count from the start again)
    with pytest.raises(RuntimeError, match="evicted since"):
        layer.restore(snap)
