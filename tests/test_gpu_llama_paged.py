"""`LlamaDecoder` over a cache in pages, and the choice among drafts on its caches.

Two forms of the same computation in fp16 differ by roundings: about 20 a layer pair, each off by at most half a step of the largest value, 2^-11: 1e-2 of
the largest logit.  With e4m3 and e2m1 pages such a difference may also move a value to the next code (2^-4, 2^-2 of it), in few channels of many: 5e-2."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOLERANCE = {"fp16": 1e-2, "e4m3": 5e-2, "e2m1": 5e-2}


def config(kv_heads=2, D=64):
    from alignedkv_b200.llama import LlamaConfig
    return LlamaConfig(hidden_size=4 * D, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=kv_heads, vocab_size=500)


def decoder(B, L=160, form="fp16", attention="paged", kv_heads=2, D=64, **kw):
    from alignedkv_b200.llama import LlamaDecoder
    return LlamaDecoder(config(kv_heads, D), B, L, DEV, seed=1, attention=attention, kv_format=form, page_size=16, **kw)


def words(*shape, seed=3):
    return torch.randint(0, 500, shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def close(x, y, form="fp16"):
    err = float((x.float() - y.float()).abs().max() / y.float().abs().max())
    assert err <= TOLERANCE[form], err


@pytest.mark.parametrize("kv_heads,D", [(4, 64), (2, 128), (1, 64)])
def test_unquantised_pages_are_dense_attention(akv_lib, kv_heads, D):
    a, d = decoder(2, kv_heads=kv_heads, D=D), decoder(2, attention="dense", kv_heads=kv_heads, D=D)
    ids = words(2, 97)
    close(a.prefill(ids), d.prefill(ids))
    for i in range(20):
        tok = words(2, seed=i)
        close(a.step(tok), d.step(tok))
    assert a.table.lengths == [117, 117] == a.table.lens.tolist()


@pytest.mark.parametrize("form", ["fp16", "e4m3", "e2m1"])
def test_a_ragged_batch_is_its_sequences(akv_lib, form):
    """Prompts of different lengths in pieces, then steps: what each sequence gives by itself, its prompt in one piece."""
    lens, ids = [1, 97, 40], words(3, 97)
    batch = decoder(3, form=form)
    pieces = [[1, 50, 0], [0, 47, 33], [0, 0, 7]]
    at, last = [0, 0, 0], [None] * 3
    for piece in pieces:
        x = torch.zeros(3, max(piece), dtype=torch.long, device=DEV)
        for b, n in enumerate(piece):
            x[b, :n] = ids[b, at[b]:at[b] + n]
            at[b] += n
        logits = batch.prefill(x, piece)
        last = [logits[b] if n else last[b] for b, n in enumerate(piece)]
    assert at == lens == batch.table.lengths
    alone = []
    for b, n in enumerate(lens):
        dec = decoder(1, form=form)
        close(last[b], dec.prefill(ids[b:b + 1, :n])[0], form)
        alone.append(dec)
    for i in range(18):                               # (over the ends of pages)
        tok = words(3, seed=10 + i)
        logits = batch.step(tok)
        for b, dec in enumerate(alone):
            close(logits[b], dec.step(tok[b:b + 1])[0], form)


@pytest.mark.parametrize("form", ["fp16", "e4m3", "e2m1"])
def test_a_verified_chain_is_that_many_steps(akv_lib, form):
    a, s = decoder(2, form=form), decoder(2, form=form)
    ids, chain = words(2, 30), words(2, 5, seed=4)
    for d in (a, s):
        d.prefill(ids, [30, 11])
    logits = a.verify(chain)
    for t in range(5):
        close(logits[:, t], s.step(chain[:, t]), form)
    assert a.table.lengths == [30, 11]
    a.accept(torch.tensor([2, 4]))
    assert a.table.lengths == [32, 15] == a.table.lens.tolist()
    # the accepted ones stay, the others are overwritten
    close(a.verify(torch.stack([chain[0, 2:4], chain[1, 3:5]]))[0, 0], logits[0, 2], form)
    one = decoder(1, form=form)
    one.prefill(ids[1:, :11])
    for t in range(4):
        one.step(chain[1:, t])
    close(a.step(words(2, seed=8))[1], one.step(words(2, seed=8)[1:])[0], form)


def test_choices_move_the_sequences_on(akv_lib):
    """Greedy drafts of the model itself are accepted all; others as the operator says, and the caches follow."""
    from alignedkv_b200 import cache_ops
    a, s = decoder(2), decoder(2)
    ids = words(2, 30)
    first = a.prefill(ids, [30, 11]).argmax(-1)
    s.prefill(ids, [30, 11])
    chain, tok = [first], first
    for _ in range(3):
        tok = s.step(tok).argmax(-1)
        chain.append(tok)
    chain = torch.stack(chain, 1)
    logits = a.verify(chain)
    coins = torch.full((2, 4), 0.5, device=DEV)
    token, counts = a.choose(logits, None, chain, coins, temperature=1e-3)           # all but a point at the largest
    assert counts == [4, 4] and a.table.lengths == [34, 15]
    assert torch.equal(token, s.step(chain[:, 3]).argmax(-1))
    # a distribution of the drafts' own
    draft = torch.softmax(torch.randn(2, 4, 500, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)), -1)
    chain = torch.cat([token[:, None], words(2, 3, seed=6)], 1)
    logits = a.verify(chain)
    coins = torch.rand(2, 4, device=DEV, generator=torch.Generator(device=DEV).manual_seed(7))
    want = cache_ops.accept_drafts(torch.softmax(logits.float(), -1), draft, chain, coins)
    token, counts = a.choose(logits, draft, chain, coins)
    assert counts == want[1].tolist() and torch.equal(token, want[2]) and a.table.lengths == [34 + counts[0], 15 + counts[1]]


def test_choices_in_a_tree_over_the_plane_cache(akv_lib):
    """One length for the batch: all go on by the smallest count; a sequence that accepted more has its next node as the next token."""
    from alignedkv_b200 import cache_ops
    a = decoder(3, attention="alignedkv")
    a.prefill(words(3, 30))
    ids, parents = words(3, 6, seed=4), torch.tensor([-1, 0, 0, 1, 2, -1])
    logits = a.verify(ids, parents)
    draft = torch.softmax(logits.float() + 0.3 * torch.randn(3, 6, 500, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)), -1)
    coins = torch.tensor([[0.3, 0.0, 0.5, 0.0, 0.5, 0.0], [0.6] + [1 - 2.0 ** -24] * 5, [0.1, 1 - 2.0 ** -24, 0.0, 0.5, 1 - 2.0 ** -24, 0.0]], device=DEV)
    ids[1, 1:] = logits[1, 0].argmin()                # (seldom accepted)
    path, count, token = cache_ops.accept_drafts(torch.softmax(logits.float(), -1), draft, ids, coins, parents.int().to(DEV))
    got, counts = a.choose(logits, draft, ids, coins, parents)
    n = int(count.min())
    assert counts == [n] * 3 and a.pos == 30 + n and all(c.cache_len == 30 + n for c in a.caches) and not (path == 5).any()
    for b in range(3):
        assert int(got[b]) == (int(ids[b, path[b, n]]) if int(count[b]) > n else int(token[b]))


def test_refusals(akv_lib):
    a = decoder(2, n_pages=4)
    a.prefill(words(2, 20), [20, 16])
    with pytest.raises(RuntimeError, match="pages are needed"):
        a.prefill(words(2, 20), [13, 17])
    assert a.table.lengths == [20, 16]
    with pytest.raises(RuntimeError, match="call verify"):
        a.accept(torch.tensor([1, 1]))
    with pytest.raises(RuntimeError, match="chains"):
        a.verify(words(2, 3), torch.tensor([-1, 0, 0]))
    with pytest.raises(RuntimeError, match="query rows"):
        a.verify(words(2, 33))
    with pytest.raises(RuntimeError, match="prefill: expected"):
        a.prefill(words(2, 3), [4, 0])
    a.verify(words(2, 3), torch.tensor([-1, 0, 1]))
    for bad in (torch.tensor([1, 4]), torch.tensor([[1], [1]]), torch.tensor([1.0, 1.0]), torch.tensor([-1, 0])):
        with pytest.raises(RuntimeError, match="path"):
            a.accept(bad)
    a.accept(torch.tensor([3, 0]))
    assert a.table.lengths == [23, 16]
    with pytest.raises(RuntimeError, match="call verify"):
        a.accept(torch.tensor([1, 1]))
    a.verify(words(2, 3))
    a.step(words(2))
    with pytest.raises(RuntimeError, match="call verify"):
        a.accept(torch.tensor([1, 1]))


def test_a_sequence_that_is_over_makes_room(akv_lib):
    a, b = decoder(2, n_pages=6, form="e4m3"), decoder(1, form="e4m3")
    a.prefill(words(2, 60), [60, 30])
    with pytest.raises(RuntimeError, match="pages are needed"):
        a.prefill(words(2, 40, seed=9), [0, 40])
    a.table.release(0)
    x = words(2, 64, seed=9)
    logits = a.prefill(x, [64, 0])
    close(logits[0], b.prefill(x[:1])[0], "e4m3")
    assert a.table.lengths == [64, 30]


def test_generation(akv_lib):
    a, d = decoder(2, kv_heads=4), decoder(2, attention="dense", kv_heads=4)
    ids = words(2, 33)
    x, y = a.generate(ids, 8), d.generate(ids, 8)
    assert x.shape == y.shape == (2, 8) and (x[:, 0] == y[:, 0]).all()
