"""Refusals of the entries around drafted tokens and eviction that keep a kernel from addresses it cannot read: alignments."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

ALIGN = -3
P = 256


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
