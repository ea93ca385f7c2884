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


@pytest.mark.parametrize("by", ["decode", "attention", "weights"])
@pytest.mark.parametrize("lowest", [-math.inf, -65504.0])
def test_a_padded_batch_is_not_evicted(akv_lib, by, lowest):
    """Survivors lie in places that differ from head to head, where no mask row can take padding away; a sequence with fewer real
    tokens than `keep` would keep some of its padding."""
    B, H, D, n = 2, 2, 128, 300
    from alignedkv_b200.decode import DecodeLayer
    gen = torch.Generator(device=DEV).manual_seed(4)
    layer = DecodeLayer(B, n + 100, H, D, DEV)
    empty = layer.snapshot()
    k, v = (torch.randn(B, n, H, D, device=DEV, generator=gen).half() for _ in range(2))
    layer.prefill(k, v)
    weigh(layer, gen)
    mask = torch.zeros(B, 1, 1, n + 50, dtype=torch.half, device=DEV)
    mask[1, ..., :250] = lowest
    q, one = torch.randn(B, 1, H, D, device=DEV, generator=gen).half(), torch.ones(1, 1, dtype=torch.bool, device=DEV)
    if by == "decode":
        layer.decode(q, q, q, mask=mask)
    elif by == "attention":
        layer.tree_attention(q, q, q, one, mask=mask)
    else:
        layer.tree_weights(q, torch.zeros(B, 1, H, device=DEV), mask=mask)
    before = layer.cache_len
    with pytest.raises(RuntimeError, match="mask"):
        layer.evict(128)
    assert (layer.cache_len, layer.rest_start, layer.evictions) == (before, 256, 0)
    layer.evict(256)                                  # nothing goes: nothing to refuse
    # another prompt in the same layer: no mask has been given for its tokens
    layer.restore(empty)
    layer.prefill(k, v)
    weigh(layer, gen)
    expect(layer, 128, 0)


def test_shift_beyond_32_bits(akv_lib):
    """A position that does not fit the positions' type is refused, not cut."""
    from alignedkv_b200 import cache_ops
    layer, _, _, gen = filled(1, 1, 128, 64, seed=5)
    weigh(layer, gen)
    layer.positions = torch.zeros(1, 1, 128, dtype=torch.int32, device=DEV)
    for shift in (2 ** 31 - 100, 2 ** 31, 2 ** 32, 2 ** 32 + 7, 2 ** 40):
        with pytest.raises(RuntimeError, match="shift"):
            cache_ops.evict(layer, layer.weights, layer.positions, rest_len=0, rest_start=128, keep=64, shift=shift)
    cache_ops.evict(layer, layer.weights, layer.positions, rest_len=0, rest_start=128, keep=64, recent=64, shift=2 ** 31 - 64 - 129)
    assert torch.equal(layer.positions[0, 0, :64].long(), torch.arange(64, 128, device=DEV) + 2 ** 31 - 64 - 129)


def test_padding_without_weight_goes_first(akv_lib):
    """What a program does that knows its padding: -inf as weight, and at least `keep` other tokens everywhere."""
    from alignedkv_b200 import cache_ops
    layer, _, _, gen = filled(2, 2, 640, 64, seed=6)
    weigh(layer, gen, zeros=0.9)
    layer.weights[1, :, :500] = -math.inf
    layer.positions = torch.zeros(2, 2, 640, dtype=torch.int32, device=DEV)
    cache_ops.evict(layer, layer.weights, layer.positions, rest_len=0, rest_start=640, keep=128, recent=30)
    assert bool((layer.positions[1, :, :128] >= 500).all())


@pytest.mark.parametrize("mode", ["exact", "order_free"])
def test_decode_steps_after_an_eviction(akv_lib, mode):
    """The survivors in the order of their places, under the maxima of all tokens that were ever there: bit for bit the steps of a
    cache that was filled so.  (Those maxima decide which planes are read: above the survivors' own they read fewer of them.)"""
    from alignedkv_b200.decode import DecodeLayer
    B, H, D, n = 2, 2, 128, 700
    gen = torch.Generator(device=DEV).manual_seed(8)
    new = lambda *shape: torch.randn(*shape, device=DEV, generator=gen).half()  # noqa: E731
    layer, other = (DecodeLayer(B, 800, H, D, DEV, n_q_heads=4, v_mode=mode) for _ in range(2))
    k, v = new(B, n, H, D), new(B, n, H, D)
    k[:, 100, :, ::8] *= 30                           # a token that is evicted and whose exponents stay
    layer.prefill(k, v)
    weigh(layer, gen)
    layer.weights[..., 100] = -1.0
    layer.evict(256, 64)
    kept_k, kept_v = (t.to(torch.int16).view(torch.half).transpose(1, 2) for t in dense(layer))
    rest = n % 64
    other.prefill(torch.cat([kept_k, k[:, n - rest:]], 1).contiguous(), torch.cat([kept_v, v[:, n - rest:]], 1).contiguous())
    assert bool((layer.k_exp_max >= other.k_exp_max).all()) and not torch.equal(layer.k_exp_max, other.k_exp_max)
    other.k_exp_max.copy_(layer.k_exp_max)
    other.v_exp_max.copy_(layer.v_exp_max)
    for _ in range(80):
        q, k1, v1 = new(B, 1, 4, D), new(B, 1, H, D), new(B, 1, H, D)
        assert torch.equal(layer.decode(q, k1, v1), other.decode(q, k1, v1))


def test_too_many_rows_are_refused_by_name(akv_lib):
    from alignedkv_b200 import cache_ops
    from alignedkv_b200.decode import DecodeLayer
    layer = DecodeLayer(65536, 64, 1, 64, DEV)
    weights, positions = (torch.zeros(65536, 1, 64, dtype=t, device=DEV) for t in (torch.float32, torch.int32))
    with pytest.raises(RuntimeError, match="65535 .* rows"):
        cache_ops.evict(layer, weights, positions, rest_len=0, rest_start=64, keep=64)
