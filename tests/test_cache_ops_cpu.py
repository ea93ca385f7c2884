"""Argument checks of the operators around drafted tokens and eviction: refused before anything is launched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def layer(**kw):
    from alignedkv_b200 import _lib
    a = _lib.Layer(*([64] * 11), 1 << 40, 2, 4, 2, 128, 1000)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


NULL, SHAPE, ALIGN, OVERFLOW = -1, -2, -3, -4
P = 256


@pytest.mark.parametrize("kw,args,code", [
    ({}, dict(q=None), NULL), ({}, dict(tree=None), NULL), (dict(scratch=None), {}, NULL), (dict(k_mid_4=None), {}, NULL),
    (dict(head_dim=96), {}, SHAPE), (dict(head_dim=256), {}, SHAPE), ({}, dict(T=0), SHAPE), ({}, dict(T=65), SHAPE),
    (dict(bsz=0), {}, SHAPE), (dict(group=0), {}, SHAPE), ({}, dict(rest=64), SHAPE), ({}, dict(rest=-1), SHAPE),
    ({}, dict(start=65), SHAPE), ({}, dict(start=-64), SHAPE), ({}, dict(start=960, rest=41), SHAPE), (dict(max_seq_len=2 ** 31 - 1), {}, SHAPE),
    ({}, dict(mask_stride=-2, mask=P), SHAPE), ({}, dict(tree_stride=-1), SHAPE), ({}, dict(k=P + 8), ALIGN),
    (dict(v_first_8=72), {}, ALIGN), (dict(bsz=1 << 20, n_kv_heads=1 << 9), {}, OVERFLOW), (dict(scratch_bytes=100), {}, SHAPE)])
def test_tree_attention_refuses(akv_lib, kw, args, code):
    a = dict(q=P, k=P, v=P, tree=P, tree_stride=0, mask=None, mask_stride=0, out=P, T=5, rest=3, start=128)
    a.update(args)
    rc = akv_lib.akv_tree_attention(layer(**kw), a["q"], a["k"], a["v"], a["tree"], a["tree_stride"], a["mask"], a["mask_stride"],
                                    a["out"], None, a["T"], a["rest"], a["start"], 1.0, None)
    assert rc == code and akv_lib.akv_last_error().startswith(b"tree_attention")
    assert akv_lib.akv_tree_attention(None, P, P, P, P, 0, None, 0, P, None, 1, 0, 0, 1.0, None) == NULL


@pytest.mark.parametrize("kw,args,code", [
    ({}, dict(lse=None), NULL), ({}, dict(weights=None), NULL), ({}, dict(T=65), SHAPE), (dict(head_dim=80), {}, SHAPE)])
def test_tree_weights_refuses(akv_lib, kw, args, code):
    a = dict(lse=P, weights=P, T=5)
    a.update(args)
    assert akv_lib.akv_tree_weights(layer(**kw), P, a["lse"], None, 0, a["weights"], a["T"], 3, 128, 1.0, None) == code


@pytest.mark.parametrize("kw,args,code", [
    ({}, dict(path=None), NULL), (dict(restk=None), {}, NULL), ({}, dict(n=0), SHAPE), ({}, dict(n=65), SHAPE), ({}, dict(T=0), SHAPE),
    ({}, dict(start=960, rest=38, n=3), SHAPE), ({}, dict(path=P + 2), ALIGN), (dict(head_dim=32), {}, SHAPE)])
def test_tree_commit_refuses(akv_lib, kw, args, code):
    a = dict(path=P, T=5, n=2, rest=3, start=128)
    a.update(args)
    assert akv_lib.akv_tree_commit(layer(**kw), P, P, a["path"], a["T"], a["n"], a["rest"], a["start"], None) == code


@pytest.mark.parametrize("kw,args,code", [
    ({}, dict(weights=None), NULL), ({}, dict(positions=None), NULL), ({}, dict(keep=0), SHAPE), ({}, dict(keep=100), SHAPE),
    ({}, dict(keep=256), SHAPE), ({}, dict(recent=65), SHAPE), ({}, dict(recent=-1), SHAPE), ({}, dict(arranged=129), SHAPE),
    ({}, dict(shift=-1), SHAPE), ({}, dict(shift=2 ** 31 - 1), SHAPE), ({}, dict(start=0, keep=64), SHAPE), ({}, dict(weights=P + 2), ALIGN),
    (dict(scratch_bytes=8), {}, SHAPE)])
def test_evict_refuses(akv_lib, kw, args, code):
    a = dict(weights=P, positions=P, rest=3, start=128, keep=64, recent=0, arranged=0, shift=0)
    a.update(args)
    assert akv_lib.akv_evict(layer(**kw), a["weights"], a["positions"], a["rest"], a["start"], a["keep"], a["recent"], a["arranged"],
                             a["shift"], None) == code


def test_scratch_sizes(akv_lib):
    assert akv_lib.akv_tree_scratch_bytes(1, 1, 1, 96, 64, 1) == -1 and akv_lib.akv_tree_scratch_bytes(1, 1, 1, 128, 64, 65) == -1
    assert akv_lib.akv_tree_scratch_bytes(8, 32, 1, 128, 4096, 16) > 0
    assert akv_lib.akv_evict_scratch_bytes(2, 3, 128, 192) == -1 and akv_lib.akv_evict_scratch_bytes(2, 3, 640, 64) >= 2 * 3 * 129 * 4


def test_host_tensors_are_refused(akv_lib):
    """The product has no CPU path: tensors on the host are refused by name."""
    import types
    from alignedkv_b200 import cache_ops
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    c = types.SimpleNamespace(k_first_8=u8(1, 1, 1, 128, 64), k_mid_4=u8(1, 1, 1, 128, 32), k_last_4=u8(1, 1, 1, 128, 32),
                              v_first_8=u8(1, 1, 64, 128), v_mid_4=u8(1, 1, 64, 64), v_last_4=u8(1, 1, 64, 64), k_exp_max=u8(1, 1, 1, 128),
                              v_exp_max=u8(1, 1, 1, 128), restk=torch.zeros(1, 64, 1, 128).half(), restv=torch.zeros(1, 64, 1, 128).half())
    q = torch.zeros(1, 1, 1, 128).half()
    with pytest.raises(RuntimeError, match="k_first_8: expected a CUDA tensor"):
        cache_ops.tree_attention(c, q, q, q, torch.ones(1, 1, dtype=torch.bool), rest_len=0, rest_start=0)


def test_eviction_plan_by_hand():
    """The tests' own plan: a few places by hand."""
    import numpy as np
    from tree_reference import evict_plan
    w, pos = np.array([[5.0, 1.0, 1.0, 7.0, 1.0, 9.0]]), np.zeros((1, 6))
    assert evict_plan(w, pos, 6, 3, 0, 0, 0)[0][0] == [0, 3, 5]
    assert evict_plan(w, pos, 6, 4, 0, 0, 0)[0][0] == [0, 1, 5, 3]            # the first of three equal ones
    assert sorted(evict_plan(w, pos, 6, 3, 2, 0, 0)[0][0]) == [3, 4, 5]
