"""Attention of drafted tokens over the plane cache, its weights, and the accepted path's way into the cache, against 64-bit forms."""
import math
import types

import pytest
import torch

from tree_reference import attend64, lse_bound, out_bound, random_tree, score_error, weights64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).half().to(DEV)


def make(B, n, Hq, H, D, T, seed=0, room=70, spread=1.0, hot=20.0):
    """A layer that holds n tokens, the dense tokens, and T drafted ones with their queries."""
    from alignedkv_b200.decode import DecodeLayer
    gen = torch.Generator().manual_seed(seed)
    x = types.SimpleNamespace(gen=gen)
    x.kc, x.vc = rand(gen, B, n, H, D), rand(gen, B, n, H, D)
    x.k, x.v, x.q = rand(gen, B, T, H, D), rand(gen, B, T, H, D), rand(gen, B, T, Hq, D, scale=spread)
    for c in (3, 34):
        x.kc[..., c] *= hot
        x.k[..., c] *= hot
    x.tree = random_tree(gen, B, T, DEV)
    x.layer = DecodeLayer(B, n + room, H, D, DEV, n_q_heads=Hq)
    if n:
        x.layer.prefill(x.kc, x.vc)
    return x


def check(x, out, lse, mask=None, tree=None):
    D, n = x.q.shape[-1], x.kc.shape[1]
    want, want_lse, mass, size = attend64(x.q, x.kc, x.vc, x.k, x.v, x.tree if tree is None else tree, mask)
    assert bool(((out.double() - want).abs() <= out_bound(want, mass, size, D)).all())
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and not bool(out[empty].any())
    e = (lse.double() - want_lse)[~empty].abs()
    assert bool((e <= lse_bound(want_lse, size, D, n)[~empty]).all())


CASES = [  # B, cached, query heads, KV heads, D, T
    (1, 0, 1, 1, 128, 1), (1, 1, 2, 2, 128, 1), (2, 63, 4, 4, 128, 2), (1, 64, 4, 2, 128, 3), (2, 65, 4, 1, 128, 4),
    (1, 127, 8, 8, 64, 5), (1, 128, 8, 2, 64, 7), (3, 129, 6, 2, 128, 16), (2, 191, 16, 2, 128, 17), (1, 192, 7, 1, 128, 9),
    (1, 640, 8, 1, 128, 64), (2, 777, 4, 4, 128, 64), (1, 1000, 16, 1, 64, 33), (2, 320, 5, 5, 64, 1), (1, 4160, 4, 2, 128, 12),
    (5, 200, 12, 3, 128, 6), (1, 8192, 2, 1, 128, 31),
]


@pytest.mark.parametrize("B,n,Hq,H,D,T", CASES)
def test_tree_attention(akv_lib, B, n, Hq, H, D, T):
    x = make(B, n, Hq, H, D, T, seed=n + T)
    out, lse = x.layer.tree_attention(x.q, x.k, x.v, x.tree, lse=True)
    check(x, out, lse)
    again = torch.empty_like(x.q)
    assert x.layer.tree_attention(x.q, x.k, x.v, x.tree, out=again) is again
    assert torch.equal(again, out), "the same call twice"
    one = x.layer.tree_attention(x.q, x.k, x.v, x.tree[0].contiguous(), lse=True)
    check(x, *one, tree=x.tree[:1].expand(B, -1, -1))


@pytest.mark.parametrize("spread,hot", [(0.02, 1.0), (12.0, 20.0)])
def test_flat_and_peaked_scores(akv_lib, spread, hot):
    x = make(2, 1500, 4, 2, 128, 10, seed=5, spread=spread, hot=hot)
    check(x, *x.layer.tree_attention(x.q, x.k, x.v, x.tree, lse=True))


def test_scale_and_many_short_sequences(akv_lib):
    from alignedkv_b200 import cache_ops
    x = make(40, 70, 16, 16, 128, 3, seed=8)
    check(x, *x.layer.tree_attention(x.q, x.k, x.v, x.tree, lse=True))
    got = cache_ops.tree_attention(x.layer, x.q, x.k, x.v, x.tree, rest_len=6, rest_start=64, scale=-0.25)
    want, _, mass, size = attend64(x.q, x.kc, x.vc, x.k, x.v, x.tree, scale=-0.25)
    assert bool(((got.double() - want).abs() <= out_bound(want, mass, size, 128)).all())


@pytest.mark.parametrize("n", [64, 70, 200, 1030])
def test_masks_and_rows_that_see_nothing(akv_lib, n):
    """Left padding up to the whole cache, with what is padded not a number; rows of the tree without a token; finite masks."""
    B, T = 4, 6
    x = make(B, n, 4, 2, 128, T, seed=n)
    mask = torch.zeros(B, n, dtype=torch.half, device=DEV)
    mask[1, :n // 2] = -math.inf
    mask[2] = -math.inf
    mask[3] = -65504.0
    mask[3, n // 3] = -1.5
    x.kc[1, :n // 2], x.vc[1, :n // 2] = math.nan, math.inf
    x.kc[2], x.vc[2] = math.inf, math.nan
    from alignedkv_b200.decode import DecodeLayer
    x.layer = DecodeLayer(B, n + 9, 2, 128, DEV, n_q_heads=4)
    x.layer.prefill(x.kc, x.vc)
    tree = x.tree.clone()
    tree[2, 0] = False
    tree[0, 3] = False
    wide = torch.full((B, 1, 1, n + 5), 7.0, dtype=torch.half, device=DEV)
    wide[:, 0, 0, :n] = mask
    check(x, *x.layer.tree_attention(x.q, x.k, x.v, tree, mask=wide, lse=True), mask=mask, tree=tree)
    lowest = torch.full((B, 1, 1, n), -65504.0, dtype=torch.half, device=DEV)
    ok = [0, 3]
    out, lse = x.layer.tree_attention(x.q, x.k, x.v, torch.zeros_like(tree), mask=lowest, lse=True)
    assert bool(torch.isfinite(out[ok]).all()) and bool((lse[ok] < -60000).all())


@pytest.mark.parametrize("D,Hq,H,T", [(128, 4, 4, 20), (128, 8, 2, 9), (64, 6, 2, 40)])
def test_masked_drafts_may_hold_anything(akv_lib, D, Hq, H, T):
    """A drafted token that is not a number or infinite: rows that see it follow the formula, the others do not notice."""
    x = make(2, 100, Hq, H, D, T, seed=T)
    tree = x.tree.clone()
    bad, worse = T // 2, T - 1
    tree[:, :, bad] = False
    x.k[:, bad], x.v[:, bad] = math.nan, math.nan
    x.v[:, worse, :, 5], x.v[:, worse, :, 6] = math.inf, math.nan           # the last node is seen by itself alone
    out, lse = x.layer.tree_attention(x.q, x.k, x.v, tree, lse=True)
    good = torch.ones(T, dtype=torch.bool)
    good[worse] = False
    clean = types.SimpleNamespace(**vars(x))
    clean.k, clean.v = x.k.nan_to_num(0, 0, 0), x.v.nan_to_num(0, 0, 0)
    want, want_lse, mass, size = attend64(clean.q, clean.kc, clean.vc, clean.k, clean.v, tree)
    close = (out.double() - want).abs() <= out_bound(want, mass, size, D)
    assert bool(close[:, good].all())
    seen = out[:, worse]
    assert bool((seen[..., 5] == math.inf).all()) and bool(seen[..., 6].isnan().all())
    rest = [c for c in range(D) if c not in (5, 6)]
    assert bool(close[:, worse][..., rest].all())
    x.k[:, worse] = math.nan
    assert bool(x.layer.tree_attention(x.q, x.k, x.v, tree)[:, worse].isnan().all())


@pytest.mark.parametrize("B,n,Hq,H,D,T", [
    (40, 300, 8, 4, 128, 3), (75, 450, 2, 2, 64, 8), (150, 129, 1, 1, 128, 2),          # more units than SMs: runs that cross units
    (1, 20000, 2, 2, 128, 5), (1, 40000, 1, 1, 64, 16),                                 # few units with many tiles
    (149, 70, 18, 1, 128, 1), (38, 260, 20, 5, 64, 5),                                  # the same with more than 16 rows a unit
    (1, 20000, 9, 1, 128, 2), (5, 1000, 8, 1, 64, 20), (3, 900, 13, 1, 128, 20)])
@pytest.mark.parametrize("masked", [False, True])
def test_work_cut_up_every_way(akv_lib, B, n, Hq, H, D, T, masked):
    """Runs of whole units, parts of units and both; masks that leave tiles whole, in part and not at all, what they take away not a
    number."""
    x = make(B, n, Hq, H, D, T, seed=B + n)
    mask = wide = None
    if masked:
        from alignedkv_b200.decode import DecodeLayer
        mask = torch.zeros(B, n, dtype=torch.half, device=DEV)
        for b in range(B):
            mask[b, :(b * 97 + n // 2) % n] = -math.inf                  # left padding
            mask[b, n - 1 - b % 50] = -math.inf                          # a single token
            mask[b, n // 2 + b % 30] = -2.5                              # one that counts less
        hidden = mask == -math.inf
        x.kc[hidden], x.vc[hidden] = math.inf, math.nan
        x.layer = DecodeLayer(B, n + 3, H, D, DEV, n_q_heads=Hq)
        x.layer.prefill(x.kc, x.vc)
        wide = torch.zeros(B, 1, 1, n + 1, dtype=torch.half, device=DEV)
        wide[:, 0, 0, :n] = mask
    check(x, *x.layer.tree_attention(x.q, x.k, x.v, x.tree, mask=wide, lse=True), mask=mask)


def test_one_token_is_a_decode_step(akv_lib):
    """T = 1: the output of `decode` within its read decisions' error, and after a commit the state it leaves, bit for bit."""
    from alignedkv_b200.decode import DecodeLayer
    x = make(2, 180, 8, 4, 128, 1, seed=3, hot=1.0)
    other = DecodeLayer(2, 250, 4, 128, DEV, n_q_heads=8)
    other.prefill(x.kc, x.vc)
    other.reference = True
    got = x.layer.tree_attention(x.q, x.k, x.v, torch.ones(1, 1, dtype=torch.bool, device=DEV))
    want = other.decode(x.q, x.k, x.v)
    # all planes read: what is left is decode's fp16 scores, probabilities and sums of up to 180 terms in fp16
    assert float((got.float() - want.float()).abs().max()) <= 2e-2 * float(want.float().abs().max())
    x.layer.tree_commit(x.k, x.v, torch.zeros(2, 1, dtype=torch.int32, device=DEV))
    same_state(x.layer, other)


STATE = ("k_first_8", "k_mid_4", "k_last_4", "v_first_8", "v_mid_4", "v_last_4", "k_exp_max", "v_exp_max")


def same_state(a, b):
    assert (a.rest_len, a.rest_start, a.cache_len) == (b.rest_len, b.rest_start, b.cache_len)
    for name in STATE:
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    for name in ("restk", "restv"):
        assert torch.equal(getattr(a, name)[:, :a.rest_len], getattr(b, name)[:, :a.rest_len]), name


@pytest.mark.parametrize("n,T,accepted,D,H", [(0, 1, 1, 128, 2), (0, 64, 64, 128, 1), (1, 64, 63, 128, 3), (60, 9, 4, 64, 2),
                                              (63, 5, 1, 128, 2), (63, 64, 64, 64, 2), (100, 40, 30, 128, 4), (128, 7, 7, 128, 2),
                                              (120, 12, 3, 128, 5)])
def test_commit_is_that_many_steps(akv_lib, n, T, accepted, D, H):
    from alignedkv_b200.decode import DecodeLayer
    B = 3
    x = make(B, n, H, H, D, T, seed=n + accepted)
    other = DecodeLayer(B, n + 70, H, D, DEV)
    if n:
        other.prefill(x.kc, x.vc)
    path = torch.stack([torch.randperm(T, generator=x.gen)[:accepted] for _ in range(B)]).to(torch.int32).to(DEV)
    row = torch.arange(B, device=DEV)
    for i in range(accepted):
        other.decode(x.q[:, :1].contiguous(), x.k[row, path[:, i].long()][:, None].contiguous(),
                     x.v[row, path[:, i].long()][:, None].contiguous())
    behind = {m: getattr(x.layer, m)[:, (n + accepted) % 64:].clone() for m in ("restk", "restv")}
    x.layer.tree_commit(x.k, x.v, path)
    same_state(x.layer, other)
    if n % 64 + accepted < 64:                         # rows behind the last token stay as they were
        for m, was in behind.items():
            assert torch.equal(getattr(x.layer, m)[:, x.layer.rest_len:], was)


def test_commit_clamps_and_repeats(akv_lib):
    x = make(2, 10, 2, 2, 128, 4, seed=2)
    x.layer.tree_commit(x.k, x.v, torch.tensor([[-7, 2, 2, 99]] * 2, dtype=torch.int32, device=DEV))
    assert torch.equal(x.layer.restk[:, 10:14], x.k[:, [0, 2, 2, 3]]) and torch.equal(x.layer.restv[:, 10:14], x.v[:, [0, 2, 2, 3]])


@pytest.mark.parametrize("B,n,Hq,H,D,T", [(1, 1, 2, 2, 128, 1), (2, 64, 4, 1, 128, 2), (1, 127, 8, 2, 64, 5), (2, 193, 6, 2, 128, 17),
                                          (1, 2000, 8, 1, 128, 32), (3, 700, 4, 4, 128, 1),
                                          (1, 300, 8, 1, 128, 64), (1, 260, 16, 1, 64, 40), (1, 130, 12, 1, 128, 64), (2, 1290, 40, 2, 64, 13),
                                          (1, 450, 5, 1, 128, 55), (1, 5000, 1, 1, 128, 1)])
@pytest.mark.parametrize("masked", [False, True])
def test_weights(akv_lib, B, n, Hq, H, D, T, masked):
    x = make(B, n, Hq, H, D, T, seed=n)
    mask = wide = None
    if masked:
        mask = torch.zeros(B, n, dtype=torch.half, device=DEV)
        mask[0, :n // 2] = -math.inf
        mask[0, n // 2] = 0.75
        wide = mask[:, None, None].contiguous()
        if n > 1:
            x.kc[0, 0] = math.nan
            from alignedkv_b200.decode import DecodeLayer
            x.layer = DecodeLayer(B, n + 70, H, D, DEV, n_q_heads=Hq)
            x.layer.prefill(x.kc, x.vc)
    _, lse = x.layer.tree_attention(x.q, x.k, x.v, x.tree, mask=wide, lse=True)
    lse[0, 0, 0] = -math.inf                          # a row that saw nothing has no weight
    got = x.layer.tree_weights(x.q, lse, mask=wide).clone()
    want, size = weights64(x.q, x.kc, lse, mask)
    rows = T * Hq // H
    size = size.nan_to_num(0.0)                       # (what is masked away has no weight)
    bound = want * (score_error(size, D) + (rows + 8) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * 40) + 1e-30
    assert bool(((got[..., :n].double() - want).abs() <= bound).all())
    assert not bool(got[..., n:].any())
    twice = x.layer.tree_weights(x.q, lse, mask=wide)
    if rows <= 512:
        assert torch.equal(twice, got * 2), "sums go on; doubling is exact"
    else:
        # 512 rows are added at a time: got = fl(a + b), twice = fl(fl(got + a) + b).  Three roundings of at most 2^-24 of sums of
        # numbers >= 0 that are at most `twice` (and the rounding itself): under 2^-22 of it
        assert rows <= 1024 and bool(((twice - got * 2).abs() <= twice * 2.0 ** -22).all())


def test_replayed_and_on_a_side_stream(akv_lib):
    """A captured round of attention, weights and commit, replayed on new inputs in the same buffers, and a call on a side stream."""
    x = make(2, 130, 8, 2, 128, 11, seed=6)
    path = torch.tensor([[0, 3, 5], [1, 2, 10]], dtype=torch.int32, device=DEV)
    eager, eager_lse = x.layer.tree_attention(x.q, x.k, x.v, x.tree, lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = x.layer.tree_attention(x.q, x.k, x.v, x.tree)
        x.layer.tree_weights(x.q, eager_lse)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, eager)
    x.layer.weights.zero_()
    from alignedkv_b200 import cache_ops
    counts = dict(rest_len=2, rest_start=128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = cache_ops.tree_attention(x.layer, x.q, x.k, x.v, x.tree, lse=True, **counts)
        cache_ops.tree_weights(x.layer, x.q, lse, x.layer.weights, **counts)
        cache_ops.tree_commit(x.layer, x.k, x.v, path, **counts)
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        x.q.copy_(rand(gen, *x.q.shape))
        graph.replay()
        want, want_lse, mass, size = attend64(x.q, x.kc, x.vc, x.k, x.v, x.tree)
        assert bool(((out.double() - want).abs() <= out_bound(want, mass, size, 128)).all())
        assert torch.equal(x.layer.restk[0, 2:5], x.k[0, [0, 3, 5]]) and torch.equal(x.layer.restv[1, 2:5], x.v[1, [1, 2, 10]])


@pytest.mark.parametrize("B,n,Hq,H,T,masked", [(1, 777, 4, 4, 3, False), (20, 300, 8, 8, 2, True), (2, 900, 16, 2, 20, True)])
def test_captured_twice_side_by_side(akv_lib, B, n, Hq, H, T, masked):
    """Two graphs of the same layer, each with its own outputs, replayed in turn and at once, against the eager call."""
    x = make(B, n, Hq, H, 128, T, seed=n)
    mask = None
    if masked:
        mask = torch.zeros(B, 1, 1, n, dtype=torch.half, device=DEV)
        mask[-1, ..., :n // 2] = -math.inf
    want = x.layer.tree_attention(x.q, x.k, x.v, x.tree, mask=mask, lse=True)
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            got.append(x.layer.tree_attention(x.q, x.k, x.v, x.tree, mask=mask, lse=True))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, lse in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_two_streams_at_once(akv_lib):
    a, b = make(2, 700, 8, 2, 128, 16, seed=1), make(1, 1500, 4, 4, 64, 40, seed=2)
    want = [x.layer.tree_attention(x.q, x.k, x.v, x.tree) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(x.layer.tree_attention(x.q, x.k, x.v, x.tree))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_refusals(akv_lib):
    x = make(2, 70, 4, 2, 128, 5, seed=0)
    L, t = x.layer, x.tree
    with pytest.raises(RuntimeError, match="q: expected"):
        L.tree_attention(x.q.float(), x.k, x.v, t)
    with pytest.raises(RuntimeError, match="query heads"):
        L.tree_attention(x.q[:, :, :3].contiguous(), x.k, x.v, t)
    with pytest.raises(RuntimeError, match="k: expected"):
        L.tree_attention(x.q, x.k[:, :4].contiguous(), x.v, t)
    with pytest.raises(RuntimeError, match="v: expected"):
        L.tree_attention(x.q, x.k, x.v.transpose(1, 2), t)
    with pytest.raises(RuntimeError, match="tree: expected"):
        L.tree_attention(x.q, x.k, x.v, t.half())
    with pytest.raises(RuntimeError, match="tree: expected"):
        L.tree_attention(x.q, x.k, x.v, t[:, :4].contiguous())
    with pytest.raises(RuntimeError, match="mask: expected"):
        L.tree_attention(x.q, x.k, x.v, t, mask=torch.zeros(2, 1, 1, 69, dtype=torch.half, device=DEV))
    with pytest.raises(RuntimeError, match="out: expected"):
        L.tree_attention(x.q, x.k, x.v, t, out=torch.empty(2, 5, 4, 64, dtype=torch.half, device=DEV))
    with pytest.raises(RuntimeError, match="out: overlaps"):
        L.tree_attention(x.q, x.k, x.v, t, out=x.q)
    with pytest.raises(RuntimeError, match="drafted tokens"):
        big = torch.zeros(2, 65, 4, 128, dtype=torch.half, device=DEV)
        L.tree_attention(big, big[:, :, :2].contiguous(), big[:, :, :2].contiguous(), t)
    with pytest.raises(RuntimeError, match="lse: expected"):
        L.tree_weights(x.q, torch.zeros(2, 5, 2, device=DEV))
    with pytest.raises(RuntimeError, match="path: expected"):
        L.tree_commit(x.k, x.v, torch.zeros(2, 2, dtype=torch.int64, device=DEV))
    with pytest.raises(RuntimeError, match="cache is full"):
        for _ in range(2):
            L.tree_commit(x.k, x.v, torch.zeros(2, 64, dtype=torch.int32, device=DEV))
    assert akv_lib.akv_device_error_flag() == 0
