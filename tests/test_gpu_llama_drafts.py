"""Drafted tokens of `LlamaDecoder.verify` belong to the state that they were made for, and survive a refused `accept`."""
import pytest
import torch

pytestmark = pytest.mark.gpu
B, S = 2, 70
CHAIN = torch.tensor([-1, 0, 1, 2])


def decoder(room, seed=1):
    from alignedkv_b200.llama import LlamaConfig, LlamaDecoder
    cfg = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1,
                      vocab_size=500)
    gen = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(0, cfg.vocab_size, (B, S + 8), device="cuda", generator=gen)
    dec = LlamaDecoder(cfg, B, S + room, "cuda:0", seed=seed)
    dec.prefill(ids[:, :S])
    return dec, ids


def paths(*nodes):
    return torch.tensor([nodes] * B)


def lengths(dec):
    return [c.cache_len for c in dec.caches] + [dec.pos]


def test_a_step_drops_the_drafts(akv_lib):
    """Keys rotated for the position that a step has taken are not appended behind it."""
    dec, ids = decoder(20)
    dec.verify(ids[:, S:S + 4], CHAIN)
    dec.step(ids[:, S])
    with pytest.raises(RuntimeError, match="call verify"):
        dec.accept(paths(0, 1))
    assert lengths(dec) == [S + 1] * 3
    dec.verify(ids[:, S + 1:S + 5], CHAIN)
    dec.accept(paths(0, 1))
    assert lengths(dec) == [S + 3] * 3


def test_a_roll_back_drops_the_drafts(akv_lib):
    """Caches that were rolled back since: other tokens are cached now, or none at these positions."""
    dec, ids = decoder(20)
    snaps = [c.snapshot() for c in dec.caches]
    dec.step(ids[:, S])
    dec.verify(ids[:, S:S + 4], CHAIN)
    for c, snap in zip(dec.caches, snaps):
        c.restore(snap)
    dec.pos = S
    with pytest.raises(RuntimeError, match="call verify"):
        dec.accept(paths(0))
    assert lengths(dec) == [S] * 3


def test_a_refused_accept_can_be_made_again(akv_lib):
    dec, ids = decoder(3)
    other, _ = decoder(3)
    for d in (dec, other):
        d.verify(ids[:, S:S + 4], CHAIN)
    for bad, text in ((paths(0, 1, 2, 3), "cache is full"), (torch.zeros(1, 2, dtype=torch.int64), "path"),
                      (torch.zeros(B, 0, dtype=torch.int64), "path"), (torch.zeros(B, dtype=torch.int64), "path"),
                      (torch.zeros(B, 2), "path"), (torch.zeros(B, 65, dtype=torch.int64), "path")):
        with pytest.raises(RuntimeError, match=text):
            dec.accept(bad)
        assert lengths(dec) == [S] * 3
    for d in (dec, other):
        d.accept(paths(0, 1, 2))
    assert lengths(dec) == [S + 3] * 3
    for x, y in zip(dec.caches, other.caches):
        assert torch.equal(x.restk, y.restk) and torch.equal(x.restv, y.restv) and torch.equal(x.k_exp_max, y.k_exp_max)
    with pytest.raises(RuntimeError, match="call verify"):
        dec.accept(paths(0))


def test_an_eviction_between_is_fine(akv_lib):
    """Positions go on counting over an eviction, so the drafts stay what they were."""
    dec, ids = decoder(80)
    other, _ = decoder(80)
    for d in (dec, other):
        d.verify(ids[:, S:S + 4], CHAIN, weights=True)
        d.accept(paths(0, 1, 2, 3))
        for i in range(60):
            d.step(ids[:, i])
        d.verify(ids[:, S:S + 4], CHAIN, weights=True)
    dec.evict(64)
    for d in (dec, other):
        d.accept(paths(0, 2))
    assert dec.pos == other.pos == S + 66
    for x, y in zip(dec.caches, other.caches):
        assert x.cache_len == 64 + 6 + 2 and torch.equal(x.restk[:, 6:8], y.restk[:, 6:8]) and torch.equal(x.restv[:, :8], y.restv[:, :8])


def test_wide_indices_are_clamped_like_others(akv_lib):
    dec, ids = decoder(20)
    dec.verify(ids[:, S:S + 4], CHAIN)
    keys = [k for k, _ in dec._drafts[1]]
    dec.accept(torch.tensor([[-2 ** 40 - 3, 2 ** 32 + 1, 7]] * B))
    at = S % 64
    for c, k in zip(dec.caches, keys):
        assert torch.equal(c.restk[:, at:at + 3], k[:, [0, 3, 3]])
