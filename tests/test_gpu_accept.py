"""The choice among drafted tokens against its definition in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def problem(B, T, V, gen, dtype=torch.float32, noise=1.0, tree=False):
    z = 2 * torch.randn(B, T, V, generator=gen)
    y = z + noise * torch.randn(B, T, V, generator=gen)
    up = torch.arange(-1, T - 1)
    if tree:
        up = torch.tensor([-1] + [int(torch.randint(0, max(1, i // 2), (1,), generator=gen)) for i in range(1, T)])
    p, q = z.softmax(-1).to(dtype), y.softmax(-1).to(dtype)
    ids = torch.stack([torch.multinomial(q[:, max(0, int(up[i]))].float(), 1, generator=gen)[:, 0] for i in range(T)], 1)
    return p.to(DEV), q.to(DEV), ids.to(DEV), torch.rand(B, T, generator=gen).to(DEV), up.to(torch.int32).to(DEV)


def check(got, p, q, ids, coins, up):
    path, count, token = got
    B, T, V = p.shape
    assert path.dtype is torch.int32 and count.dtype is torch.int32 and token.dtype is torch.int64
    for b in range(B):
        tree = up if up is None or up.dim() == 1 else up[b]
        want, last = ref.walk64(p[b].cpu(), None if q is None else q[b].cpu(), ids[b].tolist(), [float(c) for c in coins[b].tolist()],
                                list(range(-1, T - 1)) if tree is None else tree.tolist())
        assert path[b].tolist() == want + [-1] * (T - len(want)) and int(count[b]) == len(want) and int(token[b]) == last, b


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 1, 50), (7, 2, 5), (4, 5, 1000), (2, 8, 32000), (3, 64, 33), (2, 3, 131075), (1, 4, 4099), (200, 4, 64)])
def test_chains(dtype, B, T, V):
    from alignedkv_b200 import cache_ops
    gen = torch.Generator().manual_seed(B * 7 + T + V)
    p, q, ids, coins, up = problem(B, T, V, gen, dtype)
    check(cache_ops.accept_drafts(p, q, ids, coins), p, q, ids, coins, None)
    check(cache_ops.accept_drafts(p, q, ids, coins, up), p, q, ids, coins, up)
    check(cache_ops.accept_drafts(p, None, ids, coins), p, None, ids, coins, None)


@pytest.mark.parametrize("noise", [0.0, 0.3, 3.0])
@pytest.mark.parametrize("B,T,V", [(50, 12, 6), (20, 40, 30), (3, 16, 32001), (2, 64, 2000)])
def test_trees(noise, B, T, V):
    """Siblings: residuals of residuals, guesses that repeat."""
    from alignedkv_b200 import cache_ops
    gen = torch.Generator().manual_seed(B + T + V)
    p, q, ids, coins, up = problem(B, T, V, gen, noise=noise, tree=True)
    check(cache_ops.accept_drafts(p, q, ids, coins, up), p, q, ids, coins, up)
    check(cache_ops.accept_drafts(p, None, ids, coins, up), p, None, ids, coins, up)
    each = torch.stack([up.roll(0) if b % 2 else torch.cat([up[:1], torch.zeros(T - 1, dtype=torch.int32, device=DEV)]) for b in range(B)])
    check(cache_ops.accept_drafts(p, q, ids, coins, each), p, q, ids, coins, each)


def test_entries_that_are_no_probabilities_and_indices_that_are_none():
    from alignedkv_b200 import cache_ops
    gen = torch.Generator().manual_seed(3)
    B, T, V = 12, 6, 40
    p, q, ids, coins, up = problem(B, T, V, gen, tree=True)
    p[0, :, ::3], p[1, :, 5], p[2, :, 7], q[3, :, ::2], q[4, :, 1] = -1, math.nan, math.inf, math.nan, math.inf
    p[5] = 0
    q[6] = 0
    ids[7, 1:], ids[8, 2], ids[9, 3] = -1, V, 2 ** 40
    p[10] = q[10]                                   # nothing is ever rejected
    p[11, 0], q[11, 0] = 0, 1.0 / V
    p[11, 0, 9] = 1
    coins[7], coins[8, 0], coins[9, 0], coins[10] = 0, 1.0, 5.0, 1 - 2.0 ** -24
    for b, c in ((0, math.nan), (1, -3.0)):
        coins[b, 0] = c
    check(cache_ops.accept_drafts(p, q, ids, coins, up), p, q, ids, coins, up)
    check(cache_ops.accept_drafts(p, None, ids, coins, up), p, None, ids, coins, up)
    got = cache_ops.accept_drafts(p, q, ids, coins, up)
    assert int(got[2][5]) == -1 and (got[0][:, 0] == 0).all()
    wild = torch.tensor([9, 1, 5, -7, 2 ** 31 - 1, 0], dtype=torch.int32, device=DEV)          # only the last hangs under a node
    check(cache_ops.accept_drafts(p, q, ids, coins, wild), p, q, ids, coins, wild)
    coins[:, 1:] = math.nan                         # compares with nothing: rejected
    assert (cache_ops.accept_drafts(p, q, ids, coins, up)[1] == 1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strides(dtype):
    """Rows out of a wider tensor, on odd addresses; one draft row for all nodes; one target for all sequences."""
    from alignedkv_b200 import cache_ops
    gen = torch.Generator().manual_seed(4)
    B, T, V = 3, 5, 1003
    p, q, ids, coins, up = problem(B, T, V, gen, dtype, tree=True)
    wide = torch.full((B, T + 1, V + 9), 7.0, dtype=dtype, device=DEV)
    wide[:, 1:, 3:V + 3] = p
    p2 = wide[:, 1:, 3:V + 3]
    q2 = q[:, :1].expand(B, T, V)
    check(cache_ops.accept_drafts(p2, q2, ids, coins, up), p2, q2, ids, coins, up)
    p3 = p[:1].expand(B, T, V)
    check(cache_ops.accept_drafts(p3, q, ids, coins, up), p3, q, ids, coins, up)


def test_the_output_has_the_targets_distribution():
    """Two drafts under node 0, drawn from q: what follows node 0 is distributed as p.  200,000 draws per token of five; a frequency's
    standard deviation is at most (1/4 / 200000)^(1/2) = 1.1e-3, of which six are allowed."""
    from alignedkv_b200 import cache_ops
    torch.manual_seed(0)
    n, V = 200000, 5
    p1, q1 = torch.tensor([0.5, 0.2, 0.2, 0.1, 0.0], device=DEV), torch.tensor([0.1, 0.1, 0.3, 0.2, 0.3], device=DEV)
    p, q = p1.expand(n, 3, V), q1.expand(n, 3, V)
    up = torch.tensor([-1, 0, 0], dtype=torch.int32, device=DEV)
    ids = torch.multinomial(q1, 3 * n, replacement=True).view(n, 3)
    coins = torch.rand(n, 3, device=DEV)
    for draft in (q, None):
        path, count, token = cache_ops.accept_drafts(p, draft, ids, coins, up)
        node = path.gather(1, (count - 1).long()[:, None])[:, 0].long()
        first = torch.where(count > 1, ids.gather(1, node[:, None])[:, 0], token)
        freq = torch.bincount(first, minlength=V).double() / n
        assert ((freq - p1.double()).abs() < 6 * 1.2e-3).all(), freq
        # accepted at all: sum min(p, q) = 0.5 the first, then sum min(q, r / Z) = 0.2 of the rest, r / Z = (0.8, 0.2, 0, 0, 0); of guesses
        # sum q p = 0.15 the first, sum q(x) (0.15 - q(x) p(x)) = 0.121 the second
        assert abs(float((count > 1).double().mean()) - (0.6 if draft is not None else 0.271)) < 6 * 1.2e-3


def test_captured_and_on_another_stream():
    from alignedkv_b200 import cache_ops
    gen = torch.Generator().manual_seed(5)
    p, q, ids, coins, up = problem(4, 6, 5000, gen, tree=True)
    cache_ops.accept_drafts(p, q, ids, coins, up)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = cache_ops.accept_drafts(p, q, ids, coins, up)
    for seed in (1, 2):
        p2, q2, ids2, coins2, _ = problem(4, 6, 5000, torch.Generator().manual_seed(seed), tree=True)
        for a, b in ((p, p2), (q, q2), (ids, ids2), (coins, coins2)):
            a.copy_(b)
        g.replay()
        check(got, p, q, ids, coins, up)
