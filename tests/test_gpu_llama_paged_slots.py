"""A batch of slots: sequences end, the others go on, new ones take their places."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_llama_paged import DEV, close, decoder, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["fp16", "e4m3", "e2m1"])
@pytest.mark.parametrize("explicit", [False, True])
def test_a_slot_is_used_again(akv_lib, form, explicit):
    """Released, left out for some steps of the others, then given another prompt: that prompt's logits, and the others', as if alone."""
    a = decoder(3, form=form)
    ids, lens = words(3, 40), [40, 25, 31]
    a.prefill(ids, lens)
    others = {}
    for b in (0, 2):
        others[b] = decoder(1, form=form)
        others[b].prefill(ids[b:b + 1, :lens[b]])
    a.table.release(1)
    free = len(a.table.free)
    for i in range(3):
        tok = words(3, seed=20 + i)
        logits = a.step(tok, active=[True, False, True]) if explicit else a.step(tok)
        for b, d in others.items():
            close(logits[b], d.step(tok[b:b + 1])[0], form)
    assert a.table.lengths == [43, 0, 34] == a.table.lens.tolist() and not a.table.owned[1] and len(a.table.free) >= free - 2
    new, one = words(1, 19, seed=30), decoder(1, form=form)
    x = torch.zeros(3, 19, dtype=torch.long, device=DEV)
    x[1] = new[0]
    close(a.prefill(x, [0, 19, 0])[1], one.prefill(new)[0], form)
    for i in range(3):
        tok = words(3, seed=40 + i)
        logits = a.step(tok)
        close(logits[1], one.step(tok[1:2])[0], form)
        for b, d in others.items():
            close(logits[b], d.step(tok[b:b + 1])[0], form)
    assert a.table.lengths == [46, 22, 37]


def test_drafts_of_some(akv_lib):
    a = decoder(3)
    a.prefill(words(3, 30), [30, 12, 7])
    a.table.release(1)
    chain = words(3, 4, seed=4)
    logits = a.verify(chain)
    alone = decoder(1)
    alone.prefill(words(3, 30)[2:, :7])
    close(logits[2], alone.verify(chain[2:])[0])
    with pytest.raises(RuntimeError, match="path"):
        a.accept(torch.tensor([1, 1, 1]))
    coins = torch.rand(3, 4, device=DEV, generator=torch.Generator(device=DEV).manual_seed(7))
    token, counts = a.choose(logits, None, chain, coins)
    assert counts[1] == 0 and counts[0] >= 1 and counts[2] >= 1 and a.table.lengths == [30 + counts[0], 0, 7 + counts[2]] == a.table.lens.tolist()
    assert int(token[1]) == int(chain[1, 0]) and not a.table.owned[1]
    a.verify(chain, active=[False, False, True])
    a.accept(torch.tensor([0, 0, 2]))
    assert a.table.lengths == [30 + counts[0], 0, 9 + counts[2]]
    a.step(chain[:, 0], active=torch.tensor([False, True, False]))          # a new sequence that begins with a step
    assert a.table.lengths == [30 + counts[0], 1, 9 + counts[2]] and a.table.over == [False] * 3


def test_a_full_sequence_does_not_stop_the_others(akv_lib):
    a = decoder(2, L=32)
    a.prefill(words(2, 32), [32, 9])
    with pytest.raises(RuntimeError, match="no room"):
        a.step(words(2))
    a.step(words(2), active=[False, True])
    assert a.table.lengths == [32, 10]
    with pytest.raises(RuntimeError, match="active"):
        a.step(words(2), active=[True])
    for b in (0, 1):
        a.table.release(b)
    a.step(words(2))                                  # all were over: all begin anew
    assert a.table.lengths == [1, 1]
