"""Eviction from the plane cache against a plan made by sorting, and a run of drafted tokens, weights, commit and eviction together."""
import math
import types

import numpy as np
import pytest
import torch

from tree_reference import attend64, evict_plan, out_bound, random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dense(layer):
    """Cached tokens of a layer from its planes: k, v [B,H,n,D] (fp16 bits as int16)."""
    n = layer.rest_start
    both = lambda t: torch.stack([t >> 4, t & 15], -1).flatten(-2).to(torch.int32)  # noqa: E731
    word = lambda a, b, c: a.to(torch.int32) << 8 | both(b) << 4 | both(c)  # noqa: E731
    k = word(layer.k_first_8, layer.k_mid_4, layer.k_last_4).transpose(3, 4).flatten(2, 3)[:, :, :n]
    v = word(layer.v_first_8, layer.v_mid_4, layer.v_last_4)[:, :, :n]
    return k, v


def filled(B, H, n, D, seed, room=0):
    from alignedkv_b200.decode import DecodeLayer
    gen = torch.Generator(device=DEV).manual_seed(seed)
    layer = DecodeLayer(B, n + room, H, D, DEV)
    k, v = (torch.randn(B, n, H, D, device=DEV, generator=gen).half() for _ in range(2))
    layer.prefill(k, v)
    return layer, k, v, gen


def weigh(layer, gen, zeros=0.3):
    layer.weights = torch.zeros(layer.B, layer.H, layer.L, device=DEV)
    n = layer.cache_len
    w = torch.exp(2 * torch.randn(layer.B, layer.H, n, device=DEV, generator=gen))
    layer.weights[..., :n] = torch.where(torch.rand(w.shape, device=DEV, generator=gen) < zeros, 0.0, w)


def expect(layer, keep, recent):
    """Runs the eviction and holds everything it leaves behind against the plan."""
    n, rest = layer.rest_start, layer.rest_len
    if layer.positions is None:
        layer.positions = torch.full((layer.B, layer.H, layer.L), -5, dtype=torch.int32, device=DEV)
    k, v = dense(layer)
    hi, vhi, w, pos = (t.clone() for t in (layer.k_first_8, layer.v_first_8, layer.weights, layer.positions))
    top = layer.k_exp_max.clone()
    plan = evict_plan(w.cpu().numpy(), pos.cpu().numpy(), n, keep, recent, layer.arranged, layer.shift)
    layer.evict(keep, recent)
    assert (layer.rest_start, layer.rest_len, layer.cache_len) == (keep, rest, keep + rest)
    src = torch.tensor(np.array([s for s, _ in plan])).to(DEV).view(layer.B, layer.H, keep)
    place = torch.tensor(np.array([p for _, p in plan]).astype(np.int64)).to(DEV).view(layer.B, layer.H, n)
    k2, v2 = dense(layer)
    assert torch.equal(k2, k.gather(2, src[..., None].expand_as(k2))) and torch.equal(v2, v.gather(2, src[..., None].expand_as(v2)))
    assert torch.equal(layer.positions[..., :keep].long(), place.gather(2, src))
    same = lambda a, b: torch.equal(a.view(torch.int32), b.contiguous().view(torch.int32))  # noqa: E731  (NaN is itself)
    assert same(layer.weights[..., :keep].contiguous(), w.gather(2, src))
    assert same(layer.weights[..., keep:keep + rest].contiguous(), w[..., n:n + rest])
    if keep < n:
        assert not bool(layer.weights[..., keep + rest:n + rest].any())
    b = keep // 64
    assert not bool(layer.k_mid_4[:, :, b:].any()) and not bool(layer.k_last_4[:, :, b:].any())
    # behind the survivors: high bytes and V planes as they were
    assert torch.equal(layer.k_first_8[:, :, b:], hi[:, :, b:]) and torch.equal(layer.v_first_8[:, :, keep:], vhi[:, :, keep:])
    assert torch.equal(layer.k_exp_max, top)


@pytest.mark.parametrize("B,H,n,D,keep,recent", [
    (1, 1, 64, 128, 64, 0), (1, 2, 128, 128, 64, 0), (2, 3, 150, 64, 64, 10), (1, 4, 1000, 128, 448, 64), (2, 2, 1100, 128, 1024, 0),
    (1, 2, 1088, 128, 1024, 1024), (3, 1, 320, 128, 64, 64), (1, 2, 5000, 64, 1280, 100), (2, 1, 9000, 128, 8000, 33)])
def test_eviction(akv_lib, B, H, n, D, keep, recent):
    layer, _, _, gen = filled(B, H, n, D, seed=n, room=64)
    weigh(layer, gen)
    expect(layer, keep, recent)


@pytest.mark.parametrize("kind", ["equal", "zero", "special", "ascending", "descending", "negative", "close"])
def test_weights_that_are_hard_to_order(akv_lib, kind):
    layer, _, _, gen = filled(1, 2, 2100, 128, seed=4)
    weigh(layer, gen)
    n = layer.cache_len
    w = layer.weights[..., :n]
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "zero":
        w.copy_(torch.where(torch.rand(w.shape, device=DEV, generator=gen) < 0.5, 0.0, -0.0))
    elif kind == "special":
        u = torch.rand(w.shape, device=DEV, generator=gen)
        w[u < 0.2], w[(u > 0.2) & (u < 0.4)], w[u > 0.9] = math.nan, math.inf, -math.inf
        w[(u > 0.4) & (u < 0.5)] = 1e-40
    elif kind == "ascending":
        w.copy_(torch.arange(n, device=DEV).expand_as(w))
    elif kind == "descending":
        w.copy_(-torch.arange(n, device=DEV).expand_as(w).float())
    elif kind == "negative":
        w.neg_()
    else:
        w.copy_(1 + torch.randint(0, 3, w.shape, device=DEV, generator=gen) * 2.0 ** -23)
    expect(layer, 1024, 7)


def test_again_and_again(akv_lib):
    """Evictions with tokens between them: the last positions stay whichever place they were moved to."""
    from alignedkv_b200.decode import DecodeLayer
    B, H, D = 2, 2, 128
    gen = torch.Generator(device=DEV).manual_seed(9)
    layer = DecodeLayer(B, 700, H, D, DEV)
    layer.prefill(*(torch.randn(B, 500, H, D, device=DEV, generator=gen).half() for _ in range(2)))
    for i, (keep, recent) in enumerate(((256, 128), (320, 300), (192, 64), (192, 0))):
        weigh(layer, gen)
        assert layer.shift + layer.cache_len == 500 + 90 * i
        expect(layer, keep, recent)
        for _ in range(3):
            k, v = (torch.randn(B, 30, H, D, device=DEV, generator=gen).half() for _ in range(2))
            layer.tree_commit(k, v, torch.arange(30, dtype=torch.int32, device=DEV).expand(B, -1).contiguous())
    held = layer.positions[..., :layer.arranged].sort(-1).values
    assert bool((held[..., 1:] > held[..., :-1]).all()), "every position once"


def test_a_run_of_them(akv_lib):
    """Prompt, a window of queries that votes, eviction, drafted trees with weights and commits, ordinary decode steps, eviction."""
    from alignedkv_b200.decode import DecodeLayer
    B, Hq, H, D, n = 2, 8, 2, 128, 900
    gen = torch.Generator(device=DEV).manual_seed(1)
    cpu = torch.Generator().manual_seed(1)
    new = lambda T, heads: torch.randn(B, T, heads, D, device=DEV, generator=gen).half()  # noqa: E731
    layer = DecodeLayer(B, 1200, H, D, DEV, n_q_heads=Hq)
    layer.prefill(new(n, H), new(n, H))

    def cached():
        k, v = (t.to(torch.int16).view(torch.half).transpose(1, 2) for t in dense(layer))
        return torch.cat([k, layer.restk[:, :layer.rest_len]], 1), torch.cat([v, layer.restv[:, :layer.rest_len]], 1)

    def round_(T, accepted):
        q, k, v = new(T, Hq), new(T, H), new(T, H)
        tree = random_tree(cpu, B, T, DEV)
        out, lse = layer.tree_attention(q, k, v, tree, lse=True)
        want, _, mass, size = attend64(q, *cached(), k, v, tree)
        assert bool(((out.double() - want).abs() <= out_bound(want, mass, size, D)).all())
        before = layer.weights.clone() if layer.weights is not None else 0
        gained = (layer.tree_weights(q, lse) - before).sum(-1)
        # what each KV head's rows gave to cached tokens: at most one per row, and what they gave to the tree is not in it
        assert bool((gained <= T * Hq // H * 1.001).all()) and bool((gained > 0).all())
        layer.tree_commit(k, v, torch.arange(accepted, dtype=torch.int32, device=DEV).expand(B, -1).contiguous())

    round_(32, 32)
    layer.evict(512, 64)
    for T, accepted in ((6, 3), (1, 1), (17, 5), (40, 33)):
        round_(T, accepted)
    for _ in range(70):                                            # a block fills up behind the survivors
        q, k, v = new(1, Hq), new(1, H), new(1, H)
        kc, vc = cached()
        out = layer.decode(q, k, v)
        want = attend64(q, kc, vc, k, v, torch.ones(B, 1, 1, dtype=torch.bool, device=DEV))[0]
        assert float((out.double() - want).abs().max()) <= 5e-2 * float(want.abs().max())      # (decode's own approximation)
    assert layer.cache_len == layer.rest_start + layer.rest_len == 512 + 932 % 64 + 42 + 70
    layer.evict(256, 128)
    round_(9, 2)
    with pytest.raises(RuntimeError, match="mask"):
        layer.decode(new(1, Hq), new(1, H), new(1, H), mask=torch.zeros(1, 1, 1, 1200, dtype=torch.half, device=DEV))


def test_restore_and_refusals(akv_lib):
    layer, k, v, gen = filled(1, 2, 300, 128, seed=3, room=100)
    weigh(layer, gen)
    snap = layer.snapshot()
    layer.tree_commit(k[:, :5].contiguous(), v[:, :5].contiguous(), torch.arange(5, dtype=torch.int32, device=DEV)[None])
    layer.weights[..., 300:305] = 3.0
    layer.restore(snap)
    assert layer.cache_len == 300 and not bool(layer.weights[..., 300:].any())
    for keep, recent, text in ((0, 0, "keep"), (100, 0, "keep"), (320, 0, "keep"), (64, 65, "recent"), (64, -1, "recent")):
        with pytest.raises(RuntimeError, match=text):
            layer.evict(keep, recent)
    layer.evict(128)
    with pytest.raises(RuntimeError, match="evicted since"):
        layer.restore(snap)
    from alignedkv_b200 import cache_ops
    with pytest.raises(RuntimeError, match="positions: expected"):
        cache_ops.evict(layer, layer.weights, layer.positions.long(), rest_len=0, rest_start=128, keep=64)
    with pytest.raises(RuntimeError, match="head size"):
        from alignedkv_b200.decode import DecodeLayer
        DecodeLayer(1, 256, 1, 192, DEV).evict(64)


def test_two_evictions_at_once_and_replayed(akv_lib):
    from alignedkv_b200 import cache_ops
    a, _, _, gen = filled(2, 2, 1000, 128, seed=1)
    b, _, _, _ = filled(2, 2, 1000, 128, seed=1)
    weigh(a, gen)
    b.weights, b.positions = a.weights.clone(), torch.zeros(2, 2, 1000, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            cache_ops.evict(b, b.weights, b.positions, rest_len=40, rest_start=960, keep=320, recent=10)
        graph.replay()
    a.evict(320, 10)
    torch.cuda.synchronize()
    b.rest_start = 320
    for x, y in zip(dense(a), dense(b)):
        assert torch.equal(x, y)
    assert torch.equal(a.weights, b.weights) and torch.equal(a.positions[..., :320], b.positions[..., :320])
