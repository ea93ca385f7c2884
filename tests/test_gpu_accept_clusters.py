"""The choice among drafted tokens by clusters whose CTAs do not start together: SMs that other work holds become free one by one."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_accept as accept

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("B,T,V,tree", [(37, 4, 131072, False), (30, 6, 65540, True), (64, 3, 65536, False)])
def test_beside_other_work(B, T, V, tree):
    """Every call gives the same integers as the definition, alone and while another stream's products hold the SMs."""
    from alignedkv_b200 import cache_ops
    p, q, ids, coins, up = accept.problem(B, T, V, torch.Generator().manual_seed(B + V), tree=tree)
    first = cache_ops.accept_drafts(p, q, ids, coins, up)
    accept.check(first, p, q, ids, coins, up)
    x = torch.randn(4096, 4096, dtype=torch.half, device=DEV)
    y = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        with torch.cuda.stream(side):
            torch.mm(x, x, out=y)
        for _ in range(4):
            got.append(cache_ops.accept_drafts(p, q, ids, coins, up))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, first))
