"""Attention over pages is rounded once: what probabilities lose on the way to their product is made good."""
import math

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref
import test_gpu_paged as paged
from test_gpu_paged import DEV, i32

pytestmark = pytest.mark.gpu

ROWS = [(1, 1), (4, 1), (5, 1), (8, 1), (4, 3), (2, 8), (4, 5), (3, 8), (7, 4), (32, 1), (4, 10), (64, 1)]       # query heads of a KV head, tokens


def tables(pages, page, gen):
    """The table, and the same for long sequences: the work is cut up in another way."""
    return pages, torch.cat([pages, torch.randint(-2 ** 31, 2 ** 31 - 1, (len(pages), 200000 // page), generator=gen).to(torch.int32).to(DEV)], 1)


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group,T", ROWS)
def test_average_of_equal_values_is_that_value(form, D, group, T):
    """All values 2047/1024 (1.875 where a code has fewer bits), of whose half a step is 2^-12: what probabilities lose has to be missing in their sum as well,
    or in neither.  The rest is fp32: under n / 8 + 64 additions of 2^-23, so 2^-14 at most, and the value comes out exactly.  Few different
    keys, so that many tokens share a probability and lose the same."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(D + group * T)
    B, H, page, n = 2, 2, 32, 700
    lens = [n, 70]
    N = B * -(-n // page)
    pool, pages = ref.make_pool(N, page, H, D, form, DEV, gen), paged.table(B, N // B, N, gen)
    value = 2047 / 1024 if form == "fp16" else 1.875
    k = torch.randn(B, n, H, D, generator=gen)
    k[:, 1:n // 2], k[:, n // 2:] = k[:, 1:2], k[:, n // 2:n // 2 + 1]
    paged_ops.paged_append(pool, k.half().to(DEV), torch.full((B, n, H, D), value, dtype=torch.half, device=DEV), pages, i32(0, 0), counts=i32(*lens))
    q = torch.randn(B, T, H * group, D, generator=gen).half().to(DEV)
    for t in tables(pages, page, gen):
        out = paged_ops.paged_attention(pool, q, t, i32(*lens))
        off = int((out != value).sum())
        assert off == 0, f"{off} of {out.numel()}"


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group,T", ROWS)
def test_outputs_are_rounded_once(form, D, group, T):
    """Between the nearest halves of the 64-bit result less and more what fp32 may be off.  Queries have one channel: a score is one exact product and
    three roundings of 2^-24 of it (factor, product, the maximum's difference), twice, since the sum has it too; the exponential 2^-21; a
    probability's two halves 2^-22; additions as in `out_bound`; tokens 2^-24 of the largest below it lose bits under fp16's smallest, 2^-39 of the largest
    each."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(D * 3 + group * T)
    lens, B, H, page = [2, 3, 5, 9, 17, 40, 90], 7, 2, 16
    pool, pages, N = paged.filled(form, B, H, D, page, lens, gen)
    q = torch.zeros(B, T, H * group, D)
    q.scatter_(3, torch.randint(0, D, (B, T, H * group, 1), generator=gen), torch.randn(B, T, H * group, 1, generator=gen) * math.sqrt(D))
    q = q.half().to(DEV)
    k, v = (ref.pool_values(pool, w, form) for w in ("k", "v"))
    for t in tables(pages, page, gen):
        out = paged_ops.paged_attention(pool, q, t, i32(*lens))
        for b, n in enumerate(lens):
            kk, there = ref.sequence(k, pages, b, n, page, N)
            vv, _ = ref.sequence(v, pages, b, n, page, N)
            want, _, mass, size, top = ref.attend64(q[b], kk, vv, there, 1 / math.sqrt(D))
            free = mass * (2 * 3 * 2.0 ** -24 * 2 * size[..., None] + 2.0 ** -20 + 2.0 ** -22 + (n / 16 + 64) * 2.0 ** -23) + n * 2.0 ** -38 * top[..., None]
            low, high = (want - free).half(), (want + free).half()
            assert bool(((low <= out[b]) & (out[b] <= high)).all()), (b, n, int(((out[b] < low) | (out[b] > high)).sum()), out[b].numel())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group,T", ROWS)
def test_infinities_have_no_part_in_what_rounding_took(D, group, T):
    """fp16 pages: a value of infinity comes out as that in the rows that see it and in its channel alone, whatever sign the rest of its probability has;
    two of different signs as NaN.  Tables that take one tile of rows, several by clusters, and several by equal runs."""
    from alignedkv_b200 import paged_ops
    import paged_plan
    gen = torch.Generator().manual_seed(D * 5 + group * T)
    B, H, page, n = paged_plan.B, paged_plan.H, 16, 150
    N = B * -(-n // page)
    pool, pages = ref.make_pool(N, page, H, D, "fp16", DEV, gen), paged.table(B, N // B, N, gen)
    k, v = (torch.randn(B, n, H, D, generator=gen).half().to(DEV) for _ in range(2))
    v[:, n - 1, 0, 3], v[:, 20, 1, 5], v[:, n // 2, 2, 7], v[:, n // 3, 2, 7] = math.inf, -math.inf, math.inf, -math.inf
    v[:, n - 1, 3, 9] = math.nan
    paged_ops.paged_append(pool, k, v, pages, i32(*[0] * B))
    q = (torch.randn(B, T, H * group, D, generator=gen) * 0.3).half().to(DEV)
    odd = torch.zeros(T, H * group, D, device=DEV)
    odd[T - 1, :group, 3], odd[:, group:2 * group, 5] = math.inf, -math.inf
    odd[:, 2 * group:3 * group, 7] = odd[T - 1, 3 * group:, 9] = math.nan
    for table in (n,) + paged_plan.TABLES:
        more = max(0, -(-table // page) - pages.shape[1])
        wide = torch.cat([pages, torch.randint(-2 ** 31, 2 ** 31 - 1, (B, more), generator=gen).to(torch.int32).to(DEV)], 1)
        out = paged_ops.paged_attention(pool, q, wide, i32(*[n] * B))
        clean = torch.where(v.isfinite(), v, 0).double()
        for b in (0, B - 1):
            want, _, mass, size, top = ref.attend64(q[b], k[b].double(), clean[b], torch.ones(n, dtype=torch.bool, device=DEV), 1 / math.sqrt(D))
            assert torch.equal(torch.where(odd == 0, 0, out[b].float()).nan_to_num(7, 8, 9), odd.nan_to_num(7, 8, 9))
            bound = ref.out_bound(want, mass, size, top, D, n)
            assert bool((((out[b].double() - want).abs() <= bound) | (odd != 0)).all())
