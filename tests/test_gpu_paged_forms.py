"""Attention over pages in every form of its kernel: formats, head sizes, tiles of rows, pages smaller than a step, clusters and equal runs."""
import pytest

torch = pytest.importorskip("torch")

import paged_plan
import paged_reference as ref
import test_gpu_paged as paged
from test_gpu_paged import DEV, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", paged_plan.PAGES)
@pytest.mark.parametrize("group,T", paged_plan.ROWS)
def test_attention_in_every_form(form, D, page, group, T):
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(D + 7 * group + T + page)
    B, H, lens = paged_plan.B, paged_plan.H, list(paged_plan.LENS)
    pool, pages, N = paged.filled(form, B, H, D, page, lens, gen)
    pages[8, 2], pages[11, 5:9] = -1, N               # pages that were given up
    q = torch.randn(B, T, H * group, D, generator=gen).half().to(DEV)
    for table in paged_plan.TABLES:
        more = -(-table // page) - pages.shape[1]
        wide = torch.cat([pages, torch.randint(-2 ** 31, 2 ** 31 - 1, (B, more), generator=gen).to(torch.int32).to(DEV)], 1)
        out, lse = paged_ops.paged_attention(pool, q, wide, i32(*lens), lse=True)
        paged.check(pool, pages, N, form, q, lens, out, lse, page=page)
        again, _ = paged_ops.paged_attention(pool, q, wide, i32(*lens), lse=True)
        assert torch.equal(out, again)
