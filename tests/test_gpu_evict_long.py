"""The selection's forms for long caches: 1024 threads a CTA, and keys that shared memory has no room for."""
import pytest
import torch

from test_gpu_evict import DEV, expect, filled, weigh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,n,keep,recent", [
    (1, 1, 70000, 20032, 5000),          # eight CTAs of over 8192 places
    (37, 4, 8300, 4096, 100),            # a CTA a row, over 8192 places
    (1, 1, 330000, 100032, 20000),       # eight CTAs of more places than they can keep the keys of
    (1, 2, 340010, 64, 64)])
@pytest.mark.parametrize("again", [False, True])
def test_long_selection(akv_lib, B, H, n, keep, recent, again):
    layer, _, _, gen = filled(B, H, n, 64, seed=n)
    weigh(layer, gen)
    if again:            # positions as an earlier eviction left them: of the first `arranged` places every other one had been dropped
        layer.arranged, layer.shift = layer.rest_start // 128 * 64, layer.rest_start // 128 * 64
        layer.positions = torch.full((B, H, layer.L), -5, dtype=torch.int32, device=DEV)
        held = torch.rand(B, H, 2 * layer.arranged, device=DEV, generator=gen).argsort(-1)[..., :layer.arranged]
        layer.positions[..., :layer.arranged] = held.to(torch.int32)
    expect(layer, keep, recent)
