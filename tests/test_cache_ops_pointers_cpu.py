"""Refusals of the entries around drafted tokens and eviction that keep a kernel from addresses it cannot read: alignments, extents whose
products do not fit."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

SHAPE, ALIGN, OVERFLOW = -2, -3, -4
P = 256
MOST = 2 ** 31 - 1


def layer(**kw):
    from alignedkv_b200 import _lib
    a = _lib.Layer(*([64] * 11), 1 << 40, 2, 4, 2, 128, 1000)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def attention(lib, a, mask=None, lse=None):
    return lib.akv_tree_attention(a, P, P, P, P, 0, mask, 0, P, lse, 5, 3, 128, 1.0, None)


def weights(lib, a, mask=None, lse=P, w=P):
    return lib.akv_tree_weights(a, P, lse, mask, 0, w, 5, 3, 128, 1.0, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="refusals are tried where nothing can be launched")
@pytest.mark.parametrize("run,kw", [(attention, dict(mask=P + 1)), (attention, dict(lse=P + 2)), (weights, dict(mask=P + 1)),
                                    (weights, dict(lse=P + 2)), (weights, dict(w=P + 1)), (weights, dict(w=P + 2))])
def test_alignment(akv_lib, run, kw):
    assert run(akv_lib, layer(), **kw) == ALIGN and b"align" in akv_lib.akv_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="refusals are tried where nothing can be launched")
@pytest.mark.parametrize("kw", [dict(bsz=MOST, n_kv_heads=MOST, group=4), dict(bsz=1 << 30, n_kv_heads=1 << 30, group=16),
                                dict(bsz=MOST, n_kv_heads=MOST, group=MOST), dict(bsz=1, n_kv_heads=1, group=1 << 30)])
def test_rows_beyond_64_bits(akv_lib, kw):
    assert attention(akv_lib, layer(**kw)) == OVERFLOW and weights(akv_lib, layer(**kw)) == OVERFLOW
    assert akv_lib.akv_tree_scratch_bytes(kw["bsz"], kw["n_kv_heads"], kw["group"], 128, 128, 5) == -1


def test_workspaces_beyond_64_bits(akv_lib):
    assert akv_lib.akv_evict_scratch_bytes(MOST, MOST, 1 << 20, 1 << 19) == -1
    assert akv_lib.akv_evict_scratch_bytes(65535, 1, 1 << 20, 1 << 19) == 65535 * (2 * (1 << 19) + (1 << 13) + 1) * 4
    assert akv_lib.akv_tree_scratch_bytes(1, 1, 1, 128, MOST, 5) > 0
