"""Pages are handed out and taken back on the host; the tables need no GPU."""
import pytest

torch = pytest.importorskip("torch")


def table(**kw):
    from alignedkv_b200.paged import PageTable
    return PageTable(**dict(dict(bsz=3, max_seq_len=100, n_pages=8, page_size=16, device="cpu"), **kw))


def test_pages_are_handed_out_once():
    t = table()
    assert t.pages.shape == (3, 7) and (t.pages == -1).all()
    t.reserve([17, 0, 33])
    assert [len(o) for o in t.owned] == [2, 0, 3] and len(t.free) == 3
    t.advance([17, 0, 33])
    assert t.lens.tolist() == t.lengths == [17, 0, 33] and t.lens.dtype is torch.int32
    t.reserve(15)                                    # 32, 15, 48 tokens: one page more, for the second sequence
    t.advance(15)
    assert [len(o) for o in t.owned] == [2, 1, 3] and t.lens.tolist() == [32, 15, 48]
    used = [p for o in t.owned for p in o]
    assert len(set(used)) == 6 and set(used) | set(t.free) == set(range(8))
    for b, o in enumerate(t.owned):
        assert t.pages[b].tolist() == o + [-1] * (7 - len(o))


def test_refusals_change_nothing():
    t = table()
    t.reserve(20)
    t.advance(20)
    before = t.pages.clone(), list(t.free), list(t.lengths)
    for n, text in ((81, "no room"), ([13, 13, 13], "3 pages are needed, 2 of 8"), ([0, 0, 81], "sequence 2: no room")):
        with pytest.raises(RuntimeError, match=text):
            t.reserve(n)
    with pytest.raises(RuntimeError, match="reserve them first"):
        t.advance([0, 0, 13])
    for n in ([1, 2], [1, 2, -1], -1):
        with pytest.raises(ValueError):
            t.reserve(n)
        with pytest.raises(ValueError):
            t.advance(n)
    assert torch.equal(t.pages, before[0]) and t.free == before[1] and t.lengths == before[2] == t.lens.tolist()
    for kw in (dict(bsz=0), dict(max_seq_len=0), dict(n_pages=0)):
        with pytest.raises(ValueError):
            table(**kw)


def test_released_pages_are_used_again():
    t = table()
    t.reserve([48, 48, 32])
    t.advance([48, 48, 32])
    with pytest.raises(RuntimeError):
        t.reserve([0, 0, 16])
    gone = t.owned[1]
    t.release(1)
    assert t.lengths == [48, 0, 32] == t.lens.tolist() and (t.pages[1] == -1).all()
    t.reserve([0, 0, 16])
    assert t.owned[2][2] == gone[0]                  # the one that was given back last is taken first
    t.release(1)
    assert len(t.free) == 2


def test_reserved_is_not_counted():
    t = table()
    t.reserve(5)
    t.reserve(5)
    assert [len(o) for o in t.owned] == [1, 1, 1] and t.lens.tolist() == [0, 0, 0]
    t.advance([5, 3, 0])
    assert t.lens.tolist() == [5, 3, 0]


def test_layers():
    from alignedkv_b200.paged import PagedLayer
    a = PagedLayer(4, 16, 2, 64, "cpu", "e2m1")
    assert a.k_codes.shape == (4, 2, 16, 32) and a.k_codes.dtype is torch.uint8 and a.v_scales.shape == (4, 2, 16, 4) and a.v_exps.dtype is torch.int8
    b = PagedLayer(4, 16, 2, 64, "cpu")
    assert b.k_codes.dtype is torch.float8_e4m3fn and b.k_exps.shape == (4, 2, 16) and b.k_scales is None
    c = PagedLayer(4, 16, 2, 64, "cpu", "fp16")
    assert c.v_codes.dtype is torch.half and c.v_exps is None
    with pytest.raises(ValueError):
        PagedLayer(4, 16, 2, 64, "cpu", "int8")


def test_a_released_sequence_is_over_until_it_has_tokens_again():
    t = table()
    t.reserve(3)
    t.advance(3)
    t.release(1)
    assert t.over == [False, True, False]
    t.reserve([1, 0, 1])
    with pytest.raises(RuntimeError):
        t.reserve([0, 200, 0])
    assert t.over == [False, True, False]
    t.reserve([0, 5, 0])
    assert t.over == [False] * 3
