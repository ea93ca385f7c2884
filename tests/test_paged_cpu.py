"""Refusals of the operators over pages and of the choice among drafted tokens, before anything is launched; the tests' own forms by hand."""
import ctypes
import math
import types

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref

NULL, SHAPE, ALIGN, OVERFLOW = -1, -2, -3, -4
P = 256


def pool(**kw):
    from alignedkv_b200 import _lib
    a = _lib.Pool(*([64] * 6), 2, 100, 64, 4, 128)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


POOLS = [(dict(k_codes=None), NULL), (dict(v_exps=None), NULL), (dict(k_scales=None), NULL), (dict(format=3), SHAPE), (dict(format=-1), SHAPE),
         (dict(head_dim=96), SHAPE), (dict(head_dim=256), SHAPE), (dict(page_size=8), SHAPE), (dict(page_size=48), SHAPE), (dict(page_size=512), SHAPE),
         (dict(n_pages=0), SHAPE), (dict(n_kv_heads=0), SHAPE), (dict(n_kv_heads=4097), SHAPE), (dict(k_codes=72), ALIGN), (dict(v_scales=68), ALIGN),
         (dict(k_exps=66), ALIGN)]


def append(lib, a, k=P, v=P, strides=(512,) * 6, pages=P, lens=P, counts=P, bsz=2, width=10, tokens=3):
    return lib.akv_paged_append(a, k, v, None if strides is None else (ctypes.c_longlong * 6)(*strides), pages, lens, counts, bsz, width, tokens, None)


def read(lib, a, k=P, v=P, pages=P, lens=P, bsz=2, width=10, most=5):
    return lib.akv_paged_read(a, pages, lens, k, v, bsz, width, most, None)


def attention(lib, a, q=P, out=P, lse=None, pages=P, lens=P, scratch=P, scratch_bytes=1 << 40, bsz=2, width=10, group=4, tokens=1):
    return lib.akv_paged_attention(a, q, pages, lens, out, lse, scratch, scratch_bytes, bsz, width, group, tokens, 1.0, None)


COMMON = [(dict(pages=None), NULL), (dict(lens=None), NULL), (dict(bsz=0), SHAPE), (dict(bsz=4097), SHAPE), (dict(width=0), SHAPE),
          (dict(width=1 << 25), OVERFLOW), (dict(pages=P + 2), ALIGN), (dict(lens=P + 1), ALIGN)]


@pytest.mark.parametrize("run,name", [(append, b"paged_append"), (read, b"paged_read"), (attention, b"paged_attention")])
def test_pools_and_tables(akv_lib, run, name):
    for kw, code in POOLS:
        assert run(akv_lib, pool(**kw)) == code and akv_lib.akv_last_error().startswith(name), kw
    for kw, code in COMMON:
        assert run(akv_lib, pool(), **kw) == code and akv_lib.akv_last_error().startswith(name), kw
    assert run(akv_lib, None) == NULL
    assert run(akv_lib, pool(format=0, k_codes=None)) == NULL and run(akv_lib, pool(format=1, k_exps=None)) == NULL


@pytest.mark.parametrize("kw,code", [(dict(k=None), NULL), (dict(v=None), NULL), (dict(strides=None), NULL), (dict(tokens=0), SHAPE), (dict(tokens=-1), SHAPE),
                                     (dict(k=P + 8), ALIGN), (dict(counts=P + 2), ALIGN), (dict(strides=(512, 512, 4, 512, 512, 512)), ALIGN),
                                     (dict(strides=(512, 512, 512, 512, 129, 512)), ALIGN), (dict(tokens=2 ** 31 - 1), SHAPE)])
def test_append_refuses(akv_lib, kw, code):
    assert append(akv_lib, pool(), **kw) == code


@pytest.mark.parametrize("kw,code", [(dict(k=None), NULL), (dict(v=None), NULL), (dict(most=0), SHAPE), (dict(k=P + 2), ALIGN), (dict(most=2 ** 31 - 1), SHAPE)])
def test_read_refuses(akv_lib, kw, code):
    assert read(akv_lib, pool(), **kw) == code


@pytest.mark.parametrize("kw,code", [(dict(q=None), NULL), (dict(out=None), NULL), (dict(tokens=0), SHAPE), (dict(group=0), SHAPE), (dict(group=65), SHAPE),
                                     (dict(group=8, tokens=9), SHAPE), (dict(tokens=1 << 30, group=1 << 30), SHAPE), (dict(q=P + 8), ALIGN),
                                     (dict(out=P + 8), ALIGN), (dict(lse=P + 2), ALIGN)])
def test_attention_refuses(akv_lib, kw, code):
    assert attention(akv_lib, pool(), **kw) == code


def accept(lib, **kw):
    a = dict(target=P, tb=900, tr=300, draft=P, db=900, dr=300, ids=P, coins=P, parents=None, pb=0, path=P, count=P, token=P, bsz=2, T=3, V=300, type=0)
    a.update(kw)
    return lib.akv_accept_drafts(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(target=None), NULL), (dict(ids=None), NULL), (dict(coins=None), NULL), (dict(path=None), NULL), (dict(count=None), NULL), (dict(token=None), NULL),
    (dict(bsz=0), SHAPE), (dict(T=0), SHAPE), (dict(T=65), SHAPE), (dict(V=0), SHAPE), (dict(V=(1 << 24) + 1), OVERFLOW), (dict(type=3), SHAPE),
    (dict(tb=-1), SHAPE), (dict(dr=-5), SHAPE), (dict(pb=-1, parents=P), SHAPE), (dict(target=P + 2), ALIGN), (dict(draft=P + 1, type=1), ALIGN),
    (dict(ids=P + 4), ALIGN), (dict(token=P + 4), ALIGN), (dict(coins=P + 2), ALIGN), (dict(parents=P + 1), ALIGN)])
def test_accept_refuses(akv_lib, kw, code):
    assert accept(akv_lib, **kw) == code and akv_lib.akv_last_error().startswith(b"accept_drafts")


def host_pool(form="e4m3"):
    return ref.make_pool(2, 16, 1, 64, form, "cpu", torch.Generator().manual_seed(0))


def test_host_tensors_are_refused(akv_lib):
    from alignedkv_b200 import cache_ops, paged_ops
    q, n = torch.zeros(1, 1, 1, 64).half(), torch.zeros(1, dtype=torch.int32)
    for run in (lambda p: paged_ops.paged_append(p, q, q, n.view(1, 1), n), lambda p: paged_ops.paged_read(p, n.view(1, 1), n, 1),
                lambda p: paged_ops.paged_attention(p, q, n.view(1, 1), n)):
        for form in ref.FORMS:
            with pytest.raises(RuntimeError, match="k_codes: expected a CUDA tensor"):
                run(host_pool(form))
    with pytest.raises(RuntimeError, match="target: expected a CUDA tensor"):
        cache_ops.accept_drafts(torch.ones(1, 1, 4), None, torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, 1))


def test_held_values_by_hand():
    x = torch.zeros(1, 16).half()
    x[0, :6] = torch.tensor([448.0, 15.0, 0.0, -17.0, 449.0 / 2, 1.0])
    assert ref.held64(x, "e4m3")[0, :6].tolist() == [448, 15, 0, -16, 224, 1]                       # 17: a middle, to the even code
    x[0, 0] = 450
    assert ref.held64(x, "e4m3")[0, :6].tolist() == [448, 15, 0, -16, 224, 1]                       # e = 1 now: 450 / 2 -> 224
    x = torch.zeros(1, 16).half()
    x[0, :5] = torch.tensor([6.0, -1.25, 1.75, 0.25, 5.0])                                          # scale 1 (e = -8, s = 256)
    assert ref.held64(x, "e2m1")[0, :5].tolist() == [6, -1, 2, 0, 4]
    assert ref.held64(torch.full((1, 16), math.inf).half(), "e2m1").isnan().all()


def test_choice_by_hand():
    p, q = torch.tensor([[0.5, 0.5], [0.25, 0.75]]), torch.tensor([[0.0, 1.0], [0.5, 0.5]])
    assert ref.walk64(p, q, [0, 1], [0.3, 0.49], [-1, 0]) == ([0, 1], 1)                            # accepted below 1/2; then 0.3 of (1/4, 3/4)
    assert ref.walk64(p, q, [0, 1], [0.3, 0.51], [-1, 0]) == ([0], 0)                               # rejected: the residual is (1/2, 0)
    assert ref.walk64(p, None, [0, 1], [0.99, 0.5], [-1, 0]) == ([0], 0)                            # a guess: the row without it
    assert ref.walk64(p * 0, q, [0, 1], [0.5, 0.5], [-1, 0]) == ([0], -1)
