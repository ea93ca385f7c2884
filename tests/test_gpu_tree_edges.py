"""Attention of drafted tokens where its forms meet their edges: equal values, short last units, signs of the scale, long runs."""
import math

import pytest
import torch

from test_gpu_tree import DEV, check, make
from tree_reference import attend64, lse_bound, out_bound, score_error, weights64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,n,Hq,H,D,T", [
    (2, 60, 4, 4, 128, 16), (2, 62, 4, 1, 64, 4), (1, 0, 8, 8, 128, 12), (3, 700, 4, 2, 128, 5),      # up to 16 rows
    (40, 300, 8, 4, 128, 3), (1, 1500, 4, 4, 128, 8),
    (2, 60, 8, 1, 128, 9), (1, 190, 20, 1, 64, 6), (2, 700, 4, 1, 128, 30), (1, 450, 8, 1, 128, 40), (2, 900, 4, 2, 64, 64)])
def test_average_of_equal_values_is_that_value(akv_lib, B, n, Hq, H, D, T):
    """All values 2047/1024, of whose half a step is 2^-12: what probabilities lose on the way to their product has to be missing in
    their sum as well.  The rest is fp32: under n / 8 + 64 additions of 2^-23, so 2^-14 at most, and the value comes out exactly.
    Few different keys, so that many tokens share a probability and lose the same."""
    from alignedkv_b200.decode import DecodeLayer
    x = make(B, n, Hq, H, D, T, seed=n + T, hot=1.0, spread=0.6)
    x.k[:] = x.k[:, :1]
    if n:
        x.kc[:, 1:] = x.kc[:, 1:2]
        x.kc[:, n // 2:] = x.kc[:, n // 2:n // 2 + 1]
    x.vc.fill_(2047 / 1024), x.v.fill_(2047 / 1024)
    x.layer = DecodeLayer(B, n + 3, H, D, DEV, n_q_heads=Hq)
    if n:
        x.layer.prefill(x.kc, x.vc)
    out, lse = x.layer.tree_attention(x.q, x.k, x.v, x.tree, lse=True)
    off = int((out != 2047 / 1024).sum())
    assert off == 0, f"{off} of {out.numel()}"
    _, want, _, size = attend64(x.q, x.kc, x.vc, x.k, x.v, x.tree)
    assert bool(((lse.double() - want).abs() <= lse_bound(want, size, D, n)).all()), "the logarithm is that of the exact sum"


@pytest.mark.parametrize("B,n,Hq,H,D,T", [(1, 700, 37, 1, 128, 7), (2, 300, 257, 1, 64, 1), (1, 130, 74, 2, 128, 7), (40, 200, 53, 1, 64, 5)])
@pytest.mark.parametrize("masked", [False, True])
def test_last_unit_shorter_than_the_others(akv_lib, B, n, Hq, H, D, T, masked):
    """More than 256 rows that do not divide into their units."""
    x = make(B, n, Hq, H, D, T, seed=n)
    mask = wide = None
    if masked:
        mask = torch.zeros(B, n, dtype=torch.half, device=DEV)
        mask[-1, :n // 2 + 7] = -math.inf
        mask[0, n - 1] = -1.25
        wide = mask[:, None, None].contiguous()
    check(x, *x.layer.tree_attention(x.q, x.k, x.v, x.tree, mask=wide, lse=True), mask=mask)


@pytest.mark.parametrize("Hq,H,T", [(4, 2, 3), (8, 1, 3), (8, 1, 20), (8, 1, 40)])
@pytest.mark.parametrize("scale", [-0.25, -1 / math.sqrt(128), 0.0, 0.4])
def test_scales(akv_lib, Hq, H, T, scale):
    """Both signs and none, in the attention's forms (6 to 320 rows) and in the weights."""
    from alignedkv_b200 import cache_ops
    B, n, D = 2, 330, 128
    x = make(B, n, Hq, H, D, T, seed=T, hot=4.0)
    counts = dict(rest_len=n % 64, rest_start=n - n % 64)
    mask = torch.zeros(B, 1, 1, n, dtype=torch.half, device=DEV)
    mask[1, ..., :100] = -math.inf
    mask[1, ..., 200] = -0.5
    for m, m2 in ((None, None), (mask, mask[:, 0, 0])):
        out, lse = cache_ops.tree_attention(x.layer, x.q, x.k, x.v, x.tree, mask=m, scale=scale, lse=True, **counts)
        want, want_lse, mass, size = attend64(x.q, x.kc, x.vc, x.k, x.v, x.tree, m2, scale=scale)
        assert bool(((out.double() - want).abs() <= out_bound(want, mass, size, D)).all())
        assert bool(((lse.double() - want_lse).abs() <= lse_bound(want_lse, size, D, n)).all())
        weights = torch.zeros(B, H, x.layer.L, device=DEV)
        cache_ops.tree_weights(x.layer, x.q, lse, weights, mask=m, scale=scale, **counts)
        w, size = weights64(x.q, x.kc, lse, m2, scale=scale)
        bound = w * (score_error(size, D) + (T * Hq // H + 8) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * 40) + 1e-30
        assert bool(((weights[..., :n].double() - w).abs() <= bound).all())


def test_runs_of_more_than_64_tiles(akv_lib):
    """75 sequences of 131072 tokens: 65 tiles a warp.  What the mask takes away is not a number."""
    from alignedkv_b200.decode import DecodeLayer
    B, n, D = 75, 131072, 64
    gen = torch.Generator(device=DEV).manual_seed(7)
    new = lambda *s: torch.randn(*s, device=DEV, generator=gen, dtype=torch.half)  # noqa: E731
    kc, vc = new(B, n, 1, D), new(B, n, 1, D)
    mask = torch.zeros(B, 1, 1, n, dtype=torch.half, device=DEV)
    for b in range(B):
        mask[b, ..., :b * 1733] = -math.inf
        mask[b, ..., n - 300 + b:n - 290 + b] = -math.inf
        hidden = mask[b, 0, 0] == -math.inf
        kc[b, hidden], vc[b, hidden] = math.inf, math.nan
    layer = DecodeLayer(B, n, 1, D, DEV)
    layer.prefill(kc, vc)
    q, k, v = new(B, 1, 1, D), new(B, 1, 1, D), new(B, 1, 1, D)
    one = torch.ones(1, 1, dtype=torch.bool, device=DEV)
    out, lse = layer.tree_attention(q, k, v, one, mask=mask, lse=True)
    for b in range(B):
        s = slice(b, b + 1)
        want, want_lse, mass, size = attend64(q[s], kc[s], vc[s], k[s], v[s], one[None], mask[s, 0, 0])
        assert bool(((out[s].double() - want).abs() <= out_bound(want, mass, size, D)).all()), b
        assert bool(((lse[s].double() - want_lse).abs() <= lse_bound(want_lse, size, D, n)).all()), b


@pytest.mark.parametrize("B,n,Hq,H,D,T", [
    (1, 127, 4, 4, 128, 64), (1, 63, 1, 1, 64, 64), (2, 191, 2, 2, 128, 16),          # the longest tails: 63 residual and all drafted tokens
    (300, 40, 2, 2, 128, 2), (700, 0, 1, 1, 64, 3), (300, 5, 20, 1, 64, 1), (310, 63, 17, 1, 128, 1), (170, 0, 6, 1, 64, 3)])     # tails alone
def test_tails(akv_lib, B, n, Hq, H, D, T):
    x = make(B, n, Hq, H, D, T, seed=B + n)
    check(x, *x.layer.tree_attention(x.q, x.k, x.v, x.tree, lse=True))


@pytest.mark.parametrize("B,n,Hq,H,D,T", [(200, 10, 20, 1, 64, 1), (200, 150, 20, 1, 128, 1), (40, 70, 10, 1, 128, 3), (200, 10, 2, 1, 64, 2),
                                          (200, 150, 4, 1, 128, 1)])
def test_values_that_are_not_finite_stay_in_their_sequence(akv_lib, B, n, Hq, H, D, T):
    """Every third sequence has an infinite residual (or drafted) value: its rows have it, no other sequence notices."""
    from alignedkv_b200.decode import DecodeLayer
    x = make(B, n, Hq, H, D, T, seed=B)
    x.vc[::3, n - 1, :, 7] = math.inf
    x.v[1::3, 0, :, 9] = -math.inf
    x.layer = DecodeLayer(B, n + 3, H, D, DEV, n_q_heads=Hq)
    x.layer.prefill(x.kc, x.vc)
    tree = torch.ones(B, T, T, dtype=torch.bool, device=DEV)
    out, lse = x.layer.tree_attention(x.q, x.k, x.v, tree, lse=True)
    x.vc[::3, n - 1, :, 7], x.v[1::3, 0, :, 9] = 0.0, 0.0
    want, want_lse, mass, size = attend64(x.q, x.kc, x.vc, x.k, x.v, tree)
    # a probability times infinity is infinite (or, where it is under the smallest fp32 number, not a number)
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd[::3, ..., 7], odd[1::3, ..., 9] = True, True
    last = x.kc[:, -1].double().repeat_interleave(Hq // H, 1)
    seen = torch.einsum("bthd,bhd->bth", x.q.double(), last) / math.sqrt(D) - want_lse
    assert bool(((out.double() - want).abs() <= out_bound(want, mass, size, D))[~odd].all())
    assert bool(((lse.double() - want_lse).abs() <= lse_bound(want_lse, size, D, n)).all())
    there = (seen > -40.0)[::3]
    assert bool((out[::3, ..., 7][there] == math.inf).all()) and not bool(torch.isfinite(out[::3, ..., 7]).any())
    assert not bool(torch.isfinite(out[1::3, ..., 9]).any())
