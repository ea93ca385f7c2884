"""What the operators over pages and the choice among drafts refuse, by name, before anything is launched; the pool stays as it was."""
import types

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def made(form="e2m1", D=128, H=2, page=32):
    gen = torch.Generator().manual_seed(1)
    pool = ref.make_pool(4, page, H, D, form, DEV, gen)
    pages = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([3, 40], dtype=torch.int32, device=DEV)
    k = torch.randn(2, 3, H, D, generator=gen).half().to(DEV)
    q = torch.randn(2, 1, 2 * H, D, generator=gen).half().to(DEV)
    return pool, pages, lens, k, q


def other(pool, **kw):
    return types.SimpleNamespace(**dict(vars(pool), **kw))


def test_pools_and_tables():
    from alignedkv_b200 import paged_ops
    pool, pages, lens, k, q = made()
    calls = (lambda p, t, n: paged_ops.paged_append(p, k, k, t, n), lambda p, t, n: paged_ops.paged_read(p, t, n, 5),
             lambda p, t, n: paged_ops.paged_attention(p, q, t, n))
    bad_pools = [(dict(v_codes=None), "v_codes"), (dict(v_codes=pool.v_codes[:3]), "v_codes"), (dict(k_exps=None), "k_exps"),
                 (dict(v_exps=pool.v_exps.view(torch.uint8)), "v_exps"), (dict(k_scales=pool.k_scales.view(torch.uint8)), "k_scales"),
                 (dict(k_scales=pool.k_scales[..., :4]), "k_scales"), (dict(k_codes=pool.k_codes.transpose(1, 2)), "k_codes|page size"),
                 (dict(k_codes=pool.k_codes.cpu()), "k_codes"), (dict(k_codes=pool.k_codes.float()), "k_codes"), (dict(v_exps=pool.v_exps.cpu()), "v_exps"),
                 (dict(k_codes=pool.k_codes[..., :24].contiguous()), "head size 48"), (dict(k_codes=pool.k_codes[:, :, :24].contiguous()), "page size 24")]
    before = ref.parts(pool)
    for call in calls:
        for kw, text in bad_pools:
            with pytest.raises(RuntimeError, match=text):
                call(other(pool, **kw), pages, lens)
        for t, n, text in ((pages.long(), lens, "pages"), (pages[0], lens, "pages"), (pages.cpu(), lens, "pages"), (pages.t(), lens, "pages"), (None, lens, "pages"),
                           (pages[:, :0], lens, "pages"), (pages, lens.long(), "lens"), (pages, lens[:1], "lens"), (pages, lens.cpu(), "lens"), (pages, [3, 40], "lens"),
                           (pages, lens[:, None], "lens")):
            with pytest.raises(RuntimeError, match=text):
                call(pool, t, n)
    assert all(torch.equal(ref.parts(pool)[n], x) for n, x in before.items())


def test_append_and_read():
    from alignedkv_b200 import paged_ops
    pool, pages, lens, k, q = made("e4m3")
    wide = torch.zeros(2, 3, 2, 136, dtype=torch.half, device=DEV)
    odd = torch.zeros(2 * 3 * 2 * 128 + 4, dtype=torch.half, device=DEV)[4:].view(2, 3, 2, 128)
    apart = torch.zeros(2, 3, 2 * 128 + 4, dtype=torch.half, device=DEV)[..., :256].unflatten(2, (2, 128))
    for x, text in ((k.float(), "k: expected an fp16"), (k[:1], "k: expected"), (k[:, :0], "k: expected"), (k[..., :64], "k: expected"), (k.cpu(), "k: expected"),
                    (wide[..., ::1], "k: expected"), (torch.zeros(2, 3, 2, 256, dtype=torch.half, device=DEV)[..., ::2], "unit stride"), (odd, "16-byte"), (apart, "strides")):
        with pytest.raises(RuntimeError, match=text):
            paged_ops.paged_append(pool, x, k, pages, lens)
    with pytest.raises(RuntimeError, match="v: 2 tokens, k has 3"):
        paged_ops.paged_append(pool, k, k[:, :2], pages, lens)
    for c in (lens.long(), lens[:1], lens.cpu()):
        with pytest.raises(RuntimeError, match="counts"):
            paged_ops.paged_append(pool, k, k, pages, lens, counts=c)
    for most in (0, -3):
        with pytest.raises(RuntimeError, match="most"):
            paged_ops.paged_read(pool, pages, lens, most)


def test_attention():
    from alignedkv_b200 import paged_ops
    pool, pages, lens, k, q = made("fp16")
    z = lambda *s: torch.zeros(s, dtype=torch.half, device=DEV)  # noqa: E731
    for x, text in ((q.float(), "q: expected"), (q[:1], "q: expected"), (q[..., :64], "q: expected"), (q.cpu(), "q: expected"), (z(2, 1, 128, 4).transpose(2, 3), "q: expected"),
                    (z(2, 1, 3, 128), "no multiple"), (z(2, 1, 0, 128), "no multiple"), (z(2, 0, 4, 128), "rows"), (z(2, 33, 4, 128), "66|rows"), (z(2, 1, 130, 128), "65|rows")):
        with pytest.raises(RuntimeError, match=text):
            paged_ops.paged_attention(pool, x, pages, lens)
    with pytest.raises(RuntimeError, match="out"):
        paged_ops.paged_attention(pool, q, pages, lens, out=torch.empty_like(q).float())


def test_choice():
    from alignedkv_b200 import cache_ops
    p = torch.full((2, 3, 50), 0.02, device=DEV)
    ids, coins = torch.zeros(2, 3, dtype=torch.long, device=DEV), torch.zeros(2, 3, device=DEV)
    up = torch.tensor([-1, 0, 1], dtype=torch.int32, device=DEV)
    many = torch.full((1, 65, 5), 0.2, device=DEV)
    for args, text in (((p.double(), None, ids, coins), "target"), ((p[0], None, ids, coins), "target"), ((p.cpu(), None, ids, coins), "target"),
                       ((p.transpose(1, 2), None, ids, coins), "target"), ((p[:, :0], None, ids, coins), "target"), ((p, p[:, :2], ids, coins), "draft"),
                       ((p, p.half(), ids, coins), "draft"), ((p, p.cpu(), ids, coins), "draft"), ((p, None, ids.int(), coins), "ids"), ((p, None, ids[:1], coins), "ids"),
                       ((p, None, ids.t(), coins), "ids"), ((p, None, ids, coins.double()), "coins"), ((p, None, ids, coins[:, :2]), "coins"),
                       ((p, None, ids, coins, up.long()), "parents"), ((p, None, ids, coins, up[:2]), "parents"), ((p, None, ids, coins, up[None]), "parents"),
                       ((p, None, ids, coins, up.cpu()), "parents"), ((many, None, ids, coins), "65 nodes")):
        with pytest.raises(RuntimeError, match=text):
            cache_ops.accept_drafts(*args)
