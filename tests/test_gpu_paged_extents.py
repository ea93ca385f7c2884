"""Operators over pages and the choice among drafts at the ends of their extents: thousands of sequences, offsets beyond 32 bits, tables much wider than the
sequences, several streams at once."""
import math
import types

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref
from test_gpu_paged import DEV, check, filled, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ref.FORMS)
@pytest.mark.parametrize("B,H,group,T,D", [(1000, 1, 4, 1, 64), (4096, 1, 1, 1, 64), (700, 2, 2, 2, 128)])
def test_thousands_of_sequences(form, B, H, group, T, D):
    """Every one of its own length, many empty: as many as a block has threads and more."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(B)
    lens = [0 if b % 7 == 0 else (b * 37) % 150 for b in range(B)]
    pool, pages, N = filled(form, B, H, D, 16, lens, gen)
    q = torch.randn(B, T, H * group, D, generator=gen).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    some = list(range(0, B, B // 61)) + [B - 1]
    sub = types.SimpleNamespace(**vars(pool))
    check(sub, pages[some], N, form, q[some], [lens[b] for b in some], out[some], lse[some], page=16)
    assert not out[::7].any() and torch.equal(lse[::7], torch.full_like(lse[::7], -math.inf))
    k, v = paged_ops.paged_read(pool, pages, i32(*lens), 150)
    values = ref.pool_values(pool, "v", form)
    for b in some:
        want, _ = ref.sequence(values, pages, b, lens[b], 16, N)
        assert torch.equal(v[b, :lens[b]], ref.read16(want)) and not v[b, lens[b]:].any()


@pytest.mark.parametrize("form", ref.FORMS)
def test_pools_beyond_32_bits(form):
    """Pages whose bytes lie behind 2^32; the rest of the pool is never touched."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(3)
    H, P, D, lens = 8, 256, 128, [700, 300]
    row = {"fp16": 256, "e4m3": 128, "e2m1": 64}[form]
    N = 2 ** 32 // (H * P * row) + 40
    dtype = {"fp16": torch.half, "e4m3": torch.float8_e4m3fn, "e2m1": torch.uint8}[form]
    empty = lambda d, *more: torch.empty((N, H, P) + more, dtype=d, device=DEV)  # noqa: E731
    pool = types.SimpleNamespace(k_exps=None, v_exps=None, k_scales=None, v_scales=None)
    size = D // 2 if form == "e2m1" else D
    pool.k_codes, pool.v_codes = empty(dtype, size), empty(dtype, size)
    if form != "fp16":
        pool.k_exps, pool.v_exps = empty(torch.int8), empty(torch.int8)
    if form == "e2m1":
        pool.k_scales, pool.v_scales = empty(torch.float8_e4m3fn, D // 16), empty(torch.float8_e4m3fn, D // 16)
    pages = torch.tensor([[N - 1, 2, N - 7], [N - 3, N - 20, 0]], dtype=torch.int32, device=DEV)
    k, v = torch.randn(2, 700, H, D, generator=gen).half().to(DEV), torch.randn(2, 700, H, D, generator=gen).half().to(DEV)
    paged_ops.paged_append(pool, k, v, pages, i32(0, 0), counts=i32(*lens))
    got = paged_ops.paged_read(pool, pages, i32(*lens), 700)
    for o, x in zip(got, (k, v)):
        for b, n in enumerate(lens):
            assert torch.equal(o[b, :n], ref.read16(ref.held64(x[b, :n], form)))
    q = torch.randn(2, 1, 4 * H, D, generator=gen).half().to(DEV)
    out, lse = paged_ops.paged_attention(pool, q, pages, i32(*lens), lse=True)
    # the same tokens in a small pool
    used = sorted(set(pages.flatten().tolist()))
    small = types.SimpleNamespace(**{n: None if t is None else (t if t.dtype is not torch.float8_e4m3fn else t.view(torch.uint8))[used].view(t.dtype)
                                     for n, t in vars(pool).items()})
    table = torch.tensor([[used.index(j) for j in r] for r in pages.tolist()], dtype=torch.int32, device=DEV)
    check(small, table, len(used), form, q, lens, out, lse, page=P)


def test_probabilities_beyond_32_bits():
    """Sequences whose rows lie 2^32 elements apart."""
    from alignedkv_b200 import cache_ops
    gen = torch.Generator().manual_seed(4)
    T, V, far = 3, 1000, 2 ** 32 + 8
    buffer = torch.empty(far + T * V, dtype=torch.half, device=DEV)
    p = torch.softmax(torch.randn(2, T, V, generator=gen), -1).half().to(DEV)
    target = buffer.as_strided((2, T, V), (far, V, 1))
    target.copy_(p)
    ids = torch.randint(0, V, (2, T), generator=gen).to(DEV)
    coins = torch.rand(2, T, generator=gen).to(DEV)
    draft = torch.full((2, T, V), 1 / V, dtype=torch.half, device=DEV)
    for d in (draft, None):
        for x, y in zip(cache_ops.accept_drafts(target, d, ids, coins), cache_ops.accept_drafts(p, d, ids, coins)):
            assert torch.equal(x, y)


def test_streams_side_by_side():
    """The same calls on four streams at once, each with its own sequences of a shared pool."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(5)
    lens = [3000, 70, 900, 1500]
    pool, pages, N = filled("e4m3", 4, 2, 128, 64, lens, gen)
    wide = torch.cat([pages, torch.full((4, 3000), -1, dtype=torch.int32, device=DEV)], 1)
    q = torch.randn(4, 1, 8, 128, generator=gen).half().to(DEV)
    parts = [(t[b:b + 1].contiguous(), i32(lens[b]), q[b:b + 1]) for b in range(4) for t in (pages, wide)]
    want = [paged_ops.paged_attention(pool, x, t, n) for t, n, x in parts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    for _ in range(5):
        got = []
        for s, (t, n, x) in zip(streams, parts):
            with torch.cuda.stream(s):
                got.append(paged_ops.paged_attention(pool, x, t, n))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("form", ref.FORMS)
def test_values_that_are_not_finite_behind_a_wide_table(form):
    """Where units are cut into runs: a token that is not finite is in the outputs of those who see it, in no other."""
    from alignedkv_b200 import paged_ops
    gen = torch.Generator().manual_seed(6)
    B, H, D, page, n, T = 3, 2, 128, 32, 700, 3
    lens = [n] * B
    pool, pages, N = filled(form, B, H, D, page, lens, gen)
    wide = torch.cat([pages, torch.full((B, 6000), 1, dtype=torch.int32, device=DEV)], 1)
    q = torch.randn(B, T, 4, D, generator=gen).half().to(DEV)
    clean = paged_ops.paged_attention(pool, q, wide, i32(*lens))
    x = torch.randn(B, 1, H, D, generator=gen).half().to(DEV)
    bad = x.clone()
    bad[0, 0, 0, 3], bad[1, 0, 1, 5] = math.inf, math.nan
    paged_ops.paged_append(pool, x, bad, pages, i32(n - 1, 333, 5), counts=i32(1, 1, 0))
    out = paged_ops.paged_attention(pool, q, wide, i32(*lens))
    assert torch.equal(out[2], clean[2]) and torch.equal(out[0, :2], clean[0, :2]) and out[0, 2, 2:].isfinite().all()
    assert not out[0, 2, :2].isfinite().all() and not out[1, :, 2:].isfinite().all() and out[1, :, :2].isfinite().all()
