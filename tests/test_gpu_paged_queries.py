"""Attention over pages: queries that are not finite, pools that another program filled, pages that sequences share."""
import math

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref
from test_gpu_paged import DEV, check, filled, i32, table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("width", [0, 3000])
@pytest.mark.parametrize("T,group", [(1, 4), (5, 4), (2, 1)])
def test_queries_that_are_not_finite(form, width, T, group):
    """A NaN in a query is its row's, wherever the row's tokens are summed; the other rows are what they are without it."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(31)
    lens, H, D = [700, 65, 5], 2, 128
    pool, pages, N = filled(form, 3, H, D, 64, lens, gen)
    pages = torch.cat([pages, torch.full((3, width), -1, dtype=torch.int32, device=DEV)], 1)
    q = torch.randn(3, T, H * group, D, generator=gen).half().to(DEV)
    clean, clean_lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    bad = torch.zeros(3, T, H * group, dtype=torch.bool, device=DEV)
    for b, t, h, d, x in ((0, 0, 0, 3, math.nan), (1, T - 1, H * group - 1, 127, math.nan), (2, T - 1, 0, 64, math.nan)):
        q[b, t, h, d] = x
        bad[b, t, h] = True
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad])
    if form == "fp16":                              # a score of +infinity, as in dense attention
        q[bad] = 0
        q[0, T - 1, 1, 7] = math.inf
        assert paged_ops.paged_attention(pool, q, pages, i32(*lens))[0, T - 1, 1].isnan().all()


@pytest.mark.parametrize("form", ["e4m3", "e2m1"])
@pytest.mark.parametrize("T", [1, 5])
def test_exponents_of_another_programs_pool(form, T):
    """Exponents far from what append writes: keys of 2^-60 to 2^3, values of 2^-100 to 2^0 (every value fits fp16), codes as append left them."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(32)
    lens, H, D = [900, 130], 2, 128
    pool, pages, N = filled(form, 2, H, D, 32, lens, gen)
    some = torch.randint(-60, 1, pool.k_exps.shape, generator=gen).to(torch.int8).to(DEV)
    pool.k_exps.copy_(torch.where(some < -20, some, pool.k_exps.clamp(-20, 3)))
    some = torch.randint(-100, 1, pool.v_exps.shape, generator=gen).to(torch.int8).to(DEV)
    pool.v_exps.copy_(torch.where(some < -30, some, pool.v_exps.clamp(-20, 0)))
    q = (torch.randn(2, T, 4, D, generator=gen) * 0.5).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    check(pool, pages, N, form, q, lens, out, lse, page=32)
    pool.v_exps.fill_(-100)                          # (below fp16's smallest)
    assert not paged_ops.paged_attention(pool, q, pages, i32(*lens)).any()


@pytest.mark.parametrize("form", ref.FORMS)
def test_pages_that_sequences_share(form):
    """A common prompt lies in the pool once; each sequence goes on in pages of its own."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(33)
    B, H, D, page, common = 5, 2, 64, 16, 48
    N = 3 + 3 * B
    pool, order = ref.make_pool(N, page, H, D, form, DEV, gen), table(1, N, N, gen)[0]
    pages = torch.cat([order[:3].expand(B, 3), order[3:].view(B, 3)], 1).contiguous()
    k, v = (torch.randn(1, common, H, D, generator=gen).half().to(DEV) for _ in range(2))
    paged_ops.paged_append(pool, k, v, pages[:1], i32(0))
    own = [1, 16, 0, 33, 48]
    k, v = (torch.randn(B, 48, H, D, generator=gen).half().to(DEV) for _ in range(2))
    paged_ops.paged_append(pool, k, v, pages, i32(*[common] * B), counts=i32(*own))
    lens = [common + n for n in own]
    q = torch.randn(B, 1, 8, D, generator=gen).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    check(pool, pages, N, form, q, lens, out, lse, page=page)
    k, v = paged_ops.paged_read(pool, pages, i32(*lens), 96)
    assert torch.equal(k[:, :common], k[:1, :common].expand(B, -1, -1, -1)) and not v[2, common:].any()
