"""Operators over pages against their definitions in 64 bits: what is held, what is read back, attention of the newest tokens."""
import math
import types

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def table(B, width, n_pages, gen):
    return torch.randperm(n_pages, generator=gen)[:B * width].view(B, width).to(torch.int32).to(DEV)


def rows(gen, *shape):
    """fp16 rows of very different magnitudes, outlying channels, zeros."""
    x = torch.randn(*shape, generator=gen) * torch.exp2(torch.randint(-12, 9, shape[:-1] + (1,), generator=gen).float())
    x[..., 3] *= 20
    x[torch.rand(shape, generator=gen) < 0.05] = 0
    return x.half().to(DEV)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("D,H,page,T,lens,counts", [
    (128, 2, 16, 1, (0, 15, 16), None), (128, 3, 64, 70, (60, 0, 127), (70, 1, 33)), (64, 1, 32, 5, (31, 29, 95), (5, 0, 5)),
    (64, 5, 256, 40, (250, 0, 3), (40, 39, 99)), (128, 1, 128, 300, (0, 7, 1), (300, -3, 129))])
def test_append_and_read(form, D, H, page, T, lens, counts):
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(11 * T + D)
    B, width, N = 3, -(-448 // page), 3 * -(-448 // page) + 2
    pool, pages = ref.make_pool(N, page, H, D, form, DEV, gen), table(B, width, N, gen)
    k, v = rows(gen, B, T, H, D), rows(gen, B, T, H, D)
    before = ref.parts(pool)
    paged_ops.paged_append(pool, k, v, pages, i32(*lens), counts=None if counts is None else i32(*counts))
    new = [min(T, max(0, T if counts is None else c)) for c in (counts or [T] * B)]
    # what was written stands for the nearest values, nothing else has changed
    touched = torch.zeros(N, page, dtype=torch.bool, device=DEV)
    for which, x in (("k", k), ("v", v)):
        values = ref.pool_values(pool, which, form)
        for b in range(B):
            for i in range(new[b]):
                at = lens[b] + i
                j = int(pages[b, at // page])
                touched[j, at % page] = True
                assert torch.equal(values[j, :, at % page], ref.held64(x[b, i], form))
    for name, old in before.items():
        now = ref.parts(pool)[name]
        assert torch.equal(now.transpose(1, 2)[~touched], old.transpose(1, 2)[~touched])
    # ... and is read back, with everything in front of it as the pool holds it (random bytes), zeros behind
    after = [n + c for n, c in zip(lens, new)]
    most = max(after) + 3
    got = paged_ops.paged_read(pool, pages, i32(*after), most)
    for o, which in zip(got, ("k", "v")):
        assert o.shape == (B, most, H, D) and o.dtype is torch.half
        values = ref.pool_values(pool, which, form)
        for b in range(B):
            want, _ = ref.sequence(values, pages, b, after[b], page, N)
            want = ref.read16(want) if form != "fp16" else want.half()
            assert torch.equal(o[b, :after[b]].nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
            assert not o[b, after[b]:].any()


@pytest.mark.parametrize("form", ref.FORMS)
def test_special_rows(form):
    """Zeros, the ends of fp16, middles between codes, values that are not finite."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(5)
    D, page = 64, 16
    x = torch.zeros(16, D)
    x[1] = 65504
    x[2, ::2], x[2, 1::2] = 2.0 ** -24, -2.0 ** -24
    x[3] = torch.arange(D) * 0.25                                 # middles of the coarse codes
    x[4] = torch.tensor([6.0 * 2 ** -7 if i % 16 == 0 else (i % 16) * 0.25 * 2 ** -7 for i in range(D)])
    x[5] = -torch.arange(D) / 8
    x[6], x[6, 5] = 1, math.inf
    x[7], x[7, 63] = 2, math.nan
    x[8], x[8, 0] = 3, -math.inf
    x[9, 17] = 2.0 ** -24                                         # one value, the rest zero
    x[10, 0], x[10, 16:32], x[10, 33] = 60000, 2.0 ** -20, 1.0     # groups too small for a scale beside the largest
    x[11] = 448 * torch.exp2(-torch.arange(D).float() / 4)
    x[12] = 448.5
    x[13] = torch.where(torch.arange(D) % 2 == 0, 224.0, 1.0)
    x[14] = 2688
    x[15] = 2690
    k = x.half().to(DEV).view(1, 16, 1, D)
    pool = ref.make_pool(2, page, 1, D, form, DEV, gen)
    paged_ops.paged_append(pool, k, -k, i32(1).view(1, 1), i32(0))
    for which, y in (("k", k), ("v", -k)):
        got, want = ref.pool_values(pool, which, form)[1, 0], ref.held64(y[0, :, 0], form)
        assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
    o = paged_ops.paged_read(pool, i32(1).view(1, 1), i32(16), 16)[0][0, :, 0]
    if form != "fp16":
        assert o[6:9].isnan().all() and o[1].max() == 65504 and not o.isinf().any()
    else:
        assert torch.equal(o.view(torch.int16), k[0, :, 0].view(torch.int16))


@pytest.mark.parametrize("form", ref.FORMS)
def test_pages_given_up_and_ends_of_the_table(form):
    """Writes to a page outside the pool and behind the table's end are dropped; reads of one are zeros."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(6)
    D, H, page, N = 64, 2, 16, 5
    pool = ref.make_pool(N, page, H, D, form, DEV, gen)
    pages = torch.tensor([[0, -1, 1], [2 ** 31 - 1, 3, N], [-2 ** 31, 2, 4]], dtype=torch.int32, device=DEV)
    k = rows(gen, 3, 48, H, D)
    before = ref.parts(pool)
    lens = i32(0, 5, 40)
    paged_ops.paged_append(pool, k, k, pages, lens)
    touched = torch.zeros(N, page, dtype=torch.bool, device=DEV)
    values = ref.pool_values(pool, "k", form)
    for b, n in enumerate(lens.tolist()):
        for i in range(48):
            if n + i < 48 and 0 <= int(pages[b, (n + i) // 16]) < N:
                j = int(pages[b, (n + i) // 16])
                touched[j, (n + i) % 16] = True
                assert torch.equal(values[j, :, (n + i) % 16], ref.held64(k[b, i], form))
    for name, old in before.items():
        now = ref.parts(pool)[name]
        assert torch.equal(now.transpose(1, 2)[~touched], old.transpose(1, 2)[~touched])
    o, _ = paged_ops.paged_read(pool, pages, i32(2 ** 31 - 1, -7, 48), 60)
    assert not o[0, 16:32].any() and not o[0, 48:].any() and not o[1].any() and not o[2, :16].any()
    assert torch.equal(o[2, 16:32].nan_to_num(7.0), ref.read16(values[2]).transpose(0, 1).nan_to_num(7.0)) or form == "fp16"
    before = ref.parts(pool)
    paged_ops.paged_append(pool, k, k, pages, i32(2 ** 31 - 1, 48, 2 ** 31 - 40))
    assert all(torch.equal(ref.parts(pool)[n], t) for n, t in before.items())


@pytest.mark.parametrize("form", ref.FORMS)
def test_append_of_strided_parts(form):
    """Keys and values as they lie in a fused projection, a head apart, a token broadcast."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(7)
    B, T, H, D, page = 2, 9, 3, 128, 16
    qkv = rows(gen, B, T, 5 + 2 * H, D)
    k, v = qkv[:, :, 5:5 + H], qkv[:, :, 5 + H:]
    pool, pages = ref.make_pool(4, page, H, D, form, DEV, gen), i32(3, 0).view(2, 1)
    paged_ops.paged_append(pool, k, v, pages, i32(2, 5))
    for which, x in (("k", k), ("v", v)):
        values = ref.pool_values(pool, which, form)
        assert torch.equal(values[3, :, 2:11].transpose(0, 1), ref.held64(x[0], form))
        assert torch.equal(values[0, :, 5:14].transpose(0, 1), ref.held64(x[1], form))
    heads_first = rows(gen, B, H, T, D).transpose(1, 2)
    paged_ops.paged_append(pool, heads_first, qkv[:, :1, 5:5 + H].expand(B, T, H, D), pages, i32(0, 0))
    assert torch.equal(ref.pool_values(pool, "k", form)[3, :, :9].transpose(0, 1), ref.held64(heads_first[0], form))
    assert torch.equal(ref.pool_values(pool, "v", form)[0, :, 8], ref.held64(qkv[1, 0, 5:5 + H], form))


# ---------------------------------------------------------------------------------------------- attention
def filled(form, B, H, D, page, lens, gen, spread=1.0, extra=2):
    """A pool of random bytes (of values that are not finite, too) in which the sequences' tokens lie, and its table."""
    from alignedkv_b200 import paged_ops
    width = max(1, -(-max(lens) // page))
    N = B * width + extra
    pool, pages = ref.make_pool(N, page, H, D, form, DEV, gen), table(B, width, N, gen)
    T = max(1, max(lens))
    k = torch.randn(B, T, H, D, generator=gen)
    k[..., [3, 34]] *= 20
    v = torch.randn(B, T, H, D, generator=gen) * torch.exp2(torch.randint(-3, 4, (B, T, H, 1), generator=gen).float() * spread)
    paged_ops.paged_append(pool, k.half().to(DEV), v.half().to(DEV), pages, i32(*[0] * B), counts=i32(*lens))
    return pool, pages, N


def check(pool, pages, N, form, q, lens, out, lse, scale=None, page=None):
    D = q.shape[-1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    k, v = (ref.pool_values(pool, w, form) for w in ("k", "v"))
    for b, n in enumerate(lens):
        kk, there = ref.sequence(k, pages, b, n, page, N)
        vv, _ = ref.sequence(v, pages, b, n, page, N)
        want, want_lse, mass, size, top = ref.attend64(q[b], kk, vv, there, scale)
        bound = ref.out_bound(want, mass, size, top, D, n)
        assert bool(((out[b].double() - want).abs() <= bound).all()), (b, n, float(((out[b].double() - want).abs() / bound).max()))
        none = want_lse == -math.inf
        assert torch.equal(lse[b] == -math.inf, none) and not out[b][none].any()
        err = (lse[b].double() - want_lse).abs()[~none]
        assert bool((err <= ref.lse_bound(want_lse, size, D, n)[~none]).all())


SHAPES = [          # B, H, group, T, D, page, lens
    (1, 1, 1, 1, 128, 16, (1,)), (3, 2, 1, 1, 128, 16, (0, 16, 17)), (4, 1, 4, 1, 128, 64, (15, 63, 64, 65)), (2, 2, 8, 1, 64, 32, (31, 777)),
    (2, 4, 2, 1, 128, 256, (255, 1000)), (1, 2, 7, 1, 128, 64, (4097,)), (3, 1, 4, 5, 128, 64, (3, 70, 200)), (2, 2, 8, 8, 128, 32, (5, 333)),
    (2, 1, 1, 64, 64, 16, (40, 129)), (2, 2, 64, 1, 128, 64, (64, 500)), (5, 3, 3, 3, 64, 128, (0, 1, 2, 127, 600)), (1, 1, 16, 1, 128, 64, (300,)),
    (1, 1, 17, 1, 128, 64, (300,)), (40, 2, 4, 1, 128, 16, tuple(range(40)))]


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("B,H,group,T,D,page,lens", SHAPES)
def test_attention(form, B, H, group, T, D, page, lens):
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(B + 10 * T + D)
    pool, pages, N = filled(form, B, H, D, page, lens, gen)
    q = torch.randn(B, T, H * group, D, generator=gen).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    assert out.shape == q.shape and out.dtype is torch.half and lse.shape == (B, T, H * group)
    check(pool, pages, N, form, q, lens, out, lse, page=page)
    again, _ = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    assert torch.equal(out, again)
    # the same behind a table for long sequences, whose entries behind the last token may be anything: the work is cut up in another way
    wide = torch.cat([pages, torch.randint(-2 ** 31, 2 ** 31 - 1, (B, 200000 // page), generator=gen).to(torch.int32).to(DEV)], 1)
    out, lse = paged_ops.paged_attention(pool, q, wide, i32(*lens), lse=True)
    check(pool, pages, N, form, q, lens, out, lse, page=page)
    again, _ = paged_ops.paged_attention(pool, q, wide, i32(*lens), lse=True)
    assert torch.equal(out, again)


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("B,H,group,D,page,n", [(1, 1, 4, 128, 64, 70001), (1, 8, 4, 128, 256, 20000), (2, 2, 1, 64, 16, 33333)])
def test_attention_over_long_sequences(form, B, H, group, D, page, n):
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(n)
    lens = [n] + [n // 7] * (B - 1)
    pool, pages, N = filled(form, B, H, D, page, lens, gen)
    q = torch.randn(B, 1, H * group, D, generator=gen).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    check(pool, pages, N, form, q, lens, out, lse, page=page)


@pytest.mark.parametrize("form", ref.FORMS)
def test_attention_past_pages_given_up(form):
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(21)
    lens = [500, 130, 64, 200]
    pool, pages, N = filled(form, 4, 2, 128, 32, lens, gen)
    pages[0, 1:9] = -1
    pages[0, 15] = N
    pages[1, 4] = 2 ** 31 - 1
    pages[2] = -5
    pages[3, 0] = -1
    q = torch.randn(4, 3, 8, 128, generator=gen).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    check(pool, pages, N, form, q, lens, out, lse, page=32)
    assert not out[2].any()
    wide = torch.cat([pages, torch.full((4, 3000), -1, dtype=torch.int32, device=DEV)], 1)
    out, lse = paged_ops.paged_attention(pool, q, wide, i32(*lens), lse=True)
    check(pool, pages, N, form, q, lens, out, lse, page=32)


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0])
def test_attention_scales(form, scale):
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(22)
    lens = [100, 33]
    pool, pages, N = filled(form, 2, 2, 64, 16, lens, gen)
    q = (torch.randn(2, 1, 4, 64, generator=gen) * 0.3).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True, scale=scale)
    check(pool, pages, N, form, q, lens, out, lse, scale=scale, page=16)


@pytest.mark.parametrize("form", ref.FORMS)
def test_attention_of_sharp_rows_and_odd_magnitudes(form):
    """One key that dominates; values of a token near zero beside large ones, in front of and behind them; rows of zeros."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(23)
    B, H, D, page, n = 1, 1, 128, 64, 300
    pool, pages = ref.make_pool(6, page, H, D, form, DEV, gen), table(1, 5, 6, gen)
    k, v = torch.randn(1, n, H, D, generator=gen), torch.randn(1, n, H, D, generator=gen)
    q = torch.randn(1, 1, 4, D, generator=gen)
    k[0, 100, 0] = q[0, 0, 0] * 3                   # the first head looks at token 100, whose value is zero
    v[0, 100] = 0
    v[0, 7] *= 2.0 ** -22                           # all but nothing, and almost the most there is
    v[0, 8] *= 2.0 ** 14
    v[0, 200:] = 0
    k[0, 250:] = 0
    k, v, q = k.half().to(DEV), v.clamp(-65000, 65000).half().to(DEV), q.half().to(DEV)
    paged_ops.paged_append(pool, k, v, pages, i32(0))
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(n), lse=True)
    check(pool, pages, 6, form, q, [n], out, lse, page=page)
    # one token, and a few equal ones: their value as it is
    out = paged_ops.paged_attention(pool, q, pages, i32(1))
    want = ref.read16(ref.pool_values(pool, "v", form)[int(pages[0, 0]), 0, 0])
    assert torch.equal(out[0, 0], want.expand(4, D))


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("T", [1, 4])
def test_values_that_are_not_finite(form, T):
    """A query that sees such a token has it in its output; one that does not is untouched, whatever lies behind it."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(24)
    B, H, D, page, n, group = 5, 2, 128, 16, 90, 2
    pool, pages = ref.make_pool(B * 6 + 1, page, H, D, form, DEV, gen), table(B, 6, B * 6 + 1, gen)
    k, v = torch.randn(B, n, H, D, generator=gen).half().to(DEV), torch.randn(B, n, H, D, generator=gen).half().to(DEV)
    q = torch.randn(B, T, H * group, D, generator=gen).half().to(DEV)
    clean = paged_ops.paged_append(pool, k, v, pages, i32(*[0] * B))
    clean = paged_ops.paged_attention(pool, q, pages, i32(*[n] * B))
    v[0, n - 1, 0, 5] = math.inf                    # seen by the newest query alone
    v[1, 40, 1, 7] = math.nan                       # by all, in the second KV head
    k[2, n - 1, 0, 9] = math.nan
    v[3, n - 2, 1, 3] = -math.inf                   # by the two newest
    paged_ops.paged_append(pool, k, v, pages, i32(*[0] * B))
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*[n] * B), lse=True)
    odd = ~out.isfinite()
    for b, first, h, d in ((0, T - 1, 0, 5), (1, 0, 1, 7), (2, T - 1, 0, None), (3, max(0, T - 2), 1, 3)):
        heads = slice(h * group, (h + 1) * group)
        assert not odd[b, :first].any() and torch.equal(out[b, :first], clean[b, :first])
        rest = odd[b].clone()
        assert rest[first:, heads].any()
        if form == "fp16" and d is not None:         # the channel alone, with its infinity
            assert odd[b, first:, heads, d].all()
            rest[first:, heads, d] = False
        else:                                        # a row that is not finite stands for NaN throughout
            assert out[b, first:, heads].isnan().all()
            rest[first:, heads] = False
        assert not rest.any()
    if form == "fp16":
        assert (out[0, -1, :group, 5] == math.inf).all() and (out[3, -1, group:, 3] == -math.inf).all()
    assert torch.equal(out[4], clean[4])
    if form == "fp16":                               # keys that take a token away: a score of -inf has no part
        k[4, :, :, 0], q[4, ..., 0] = 1, 1
        k[4, 20, :, 0] = -math.inf
        paged_ops.paged_append(pool, k, v, pages, i32(*[0] * B))
        out = paged_ops.paged_attention(pool, q, pages, i32(*[n] * B))
        v[4, 20] = 1000
        paged_ops.paged_append(pool, k, v, pages, i32(*[0] * B))
        assert torch.equal(paged_ops.paged_attention(pool, q, pages, i32(*[n] * B))[4], out[4]) and out[4].isfinite().all()


def test_attention_into_a_given_tensor_on_another_stream():
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(25)
    lens = [333, 90]
    pool, pages, N = filled("e4m3", 2, 2, 128, 64, lens, gen)
    q = torch.randn(2, 1, 8, 128, generator=gen).half().to(DEV)
    want = paged_ops.paged_attention(pool, q, pages, i32(*lens))
    out = torch.full_like(q, 7.0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert paged_ops.paged_attention(pool, q, pages, i32(*lens), out=out) is out
    side.synchronize()
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="overlaps"):
        paged_ops.paged_attention(pool, q, pages, i32(*lens), out=q)


@pytest.mark.parametrize("form", ref.FORMS)
def test_captured_steps_follow_the_lengths(form):
    """A captured append and attention, replayed with other lengths, pages and tokens than it was captured with; another graph beside it."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(26)
    B, H, D, page = 2, 2, 128, 16
    lens = [40, 7]
    pool, pages, N = filled(form, B, H, D, page, [130, 130], gen)
    n = i32(*lens)
    k, v, q = (torch.randn(B, 1, h, D, generator=gen).half().to(DEV) for h in (H, H, 4 * H))

    def step():
        paged_ops.paged_append(pool, k, v, pages, n)
        n.add_(1)
        return paged_ops.paged_attention(pool, q, pages, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step()))
    for i, start in enumerate(([0, 0], [15, 100], [127, 63], [128, 64])):
        n.copy_(i32(*start))
        k.normal_(), v.normal_(), q.normal_()
        g, out = graphs[i % 2]
        g.replay()
        after = [s + 1 for s in start]
        assert n.tolist() == after
        want, lse = paged_ops.paged_attention(pool, q, pages, n, lse=True)
        assert torch.equal(out, want)
        check(pool, pages, N, form, q, after, out, lse, page=page)
