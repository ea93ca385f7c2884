"""Operators around a bit-plane KV cache that a program with drafted tokens and a bounded cache calls, as measurable cases.

  attend    a tree of T drafted tokens attends to the cache and to its own ancestors (`cache_ops.tree_attention`); T = 1 is
            a decode token that is not appended yet.
  observe   the attention weight that such queries give each cached token is added to fp32 sums (`cache_ops.tree_weights`).
  commit    the accepted path of a tree enters the cache: exponent maxima, residual buffer, and the planes of blocks that
            fill up (`cache_ops.tree_commit`).
  evict     each (sequence, KV head) keeps its `keep` heaviest cached tokens; survivors from behind move into the places that
            became free (`cache_ops.evict`).

Keys, values and queries are N(0,1) with four key channels per head scaled by 20, the distribution of this repository's
benchmark.  Planes: fp16 x as high byte, bits 7..4 and bits 3..0; K [B,H,blocks,D,64] with two tokens in a nibble byte, V
[B,H,tokens,D] with two channels in one, the even one in the high nibble.
"""
import math
import random
import types

import torch

own = False

BLOCK = 64
OUTLIER_CHANNELS = (3, 34, 65, 96)
MOST_ROWS = 8 * 32 * 4096        # (sequence, KV head, token) rows of the largest cache that a drawn case reads

BASE = dict(batch=1, heads=32, kv_heads=32, dim=128, tokens=0, drafts=1, masked=False, accepted=0, keep=0, recent=0, again=False)


def listed():
    return [
        # one user's chat with a short tree: a small call, where launches and latency count
        dict(BASE, name="tree-b1-777-t8", kind="attend", tokens=777, drafts=8),
        # the benchmark's layer, 16 drafted tokens per sequence: every head has its own keys
        dict(BASE, name="tree-b8-4096-t16", kind="attend", batch=8, tokens=4096, drafts=16),
        # a left-padded batch of short prompts, one token each: a decode step whose token is not appended yet
        dict(BASE, name="tree-b16-1000-t1-padded", kind="attend", batch=16, tokens=1000, drafts=1, masked=True),
        # grouped queries, an ordinary tree: 48 query rows share a KV head
        dict(BASE, name="tree-gqa-b16-8190-t12", kind="attend", batch=16, kv_heads=8, tokens=8190, drafts=12),
        # a wide tree under grouped queries: 256 query rows per KV head
        dict(BASE, name="tree-gqa-b4-8192-t64", kind="attend", batch=4, kv_heads=8, tokens=8192, drafts=64),
        # one long document, a chain of five drafted tokens
        dict(BASE, name="tree-gqa-b1-131072-t5", kind="attend", kv_heads=8, tokens=131072, drafts=5),
        # weights of a single token per sequence, after its attention
        dict(BASE, name="weights-b8-4096-t1", kind="observe", batch=8, tokens=4096, drafts=1),
        # weights of an observation window: the last 32 prompt tokens vote on the cache before it
        dict(BASE, name="weights-gqa-b4-8190-t32", kind="observe", batch=4, kv_heads=8, tokens=8190, drafts=32),
        # three accepted tokens of one sequence: the smallest call
        dict(BASE, name="commit-b1-n3", kind="commit", tokens=777, drafts=8, accepted=3),
        # a window of 48 tokens of a large batch, which fills a block and begins the next
        dict(BASE, name="commit-gqa-b64-n48", kind="commit", batch=64, kv_heads=8, tokens=1000, drafts=64, accepted=48),
        # half of the benchmark's cache goes, the last 256 positions are safe
        dict(BASE, name="evict-b8-4096-2048", kind="evict", batch=8, tokens=4100, keep=2048, recent=256),
        # a long document cut to an eighth, for the second time
        dict(BASE, name="evict-gqa-b1-131072-16384", kind="evict", kv_heads=8, tokens=131072, keep=16384, recent=1024, again=True),
    ]


def _between(rng: random.Random, low: int, high: int) -> int:
    """Spread over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choices(["attend", "observe", "commit", "evict"], [6, 3, 2, 3])[0]
    group = rng.choice([1, 1, 2, 4, 4, 8])
    heads = rng.choice([8, 32, 32])
    case = dict(BASE, kind=kind, heads=heads, kv_heads=heads // group, dim=rng.choice([64, 128, 128, 128]))
    case["batch"] = _between(rng, 1, 64)
    room = MOST_ROWS // (case["batch"] * case["kv_heads"])
    if kind in ("attend", "observe"):
        case["tokens"] = _between(rng, 16, min(131072, room))
        case["drafts"] = _between(rng, 1, 64)
        # no dearer than the largest listed cases: rows x tokens of the plain form's scores
        while case["batch"] * heads * case["drafts"] * case["tokens"] > 4 * 32 * 64 * 8192:
            case["drafts"] = max(1, case["drafts"] // 2)
            case["tokens"] = max(16, case["tokens"] * 3 // 4)
        case["masked"] = rng.random() < 0.3
        if rng.random() < 0.4:
            case["tokens"] = max(BLOCK, case["tokens"] // BLOCK * BLOCK)
    elif kind == "commit":
        case["tokens"] = _between(rng, 16, min(4096, room))
        case["drafts"] = _between(rng, 1, 64)
        case["accepted"] = rng.randint(1, case["drafts"])
    else:
        case["tokens"] = _between(rng, 4 * BLOCK, min(65536, max(4 * BLOCK, room)))
        blocks = case["tokens"] // BLOCK
        case["keep"] = BLOCK * rng.randint(max(1, blocks // 8), blocks - 1)
        case["recent"] = rng.randint(0, case["keep"] // 2)
        case["again"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _sizes(case):
    group = case["heads"] // case["kv_heads"]
    rest = case["tokens"] % BLOCK
    whole = case["tokens"] - rest
    most = (case["tokens"] + 2 * BLOCK + BLOCK - 1) // BLOCK * BLOCK      # room for what is appended
    return group, whole, rest, most


def _inputs(case, seed):
    """Dense tensors from the seed alone: cached keys and values [B,H,tokens,D], queries, drafts, tree, mask."""
    B, H, D, n, T = case["batch"], case["kv_heads"], case["dim"], case["tokens"], case["drafts"]
    g = torch.Generator(device=_device()).manual_seed(1000003 * seed + 131 * n + B)
    normal = lambda *shape: torch.randn(*shape, device=_device(), generator=g)  # noqa: E731
    hot = torch.ones(D, device=_device())
    hot[[c for c in OUTLIER_CHANNELS if c < D]] = 20.0
    x = types.SimpleNamespace()
    x.kc, x.vc = (normal(B, H, n, D) * hot).half(), normal(B, H, n, D).half()
    x.q = normal(B, T, case["heads"], D).half()
    x.k, x.v = (normal(B, T, H, D) * hot).half(), normal(B, T, H, D).half()
    # a random tree per sequence: node i hangs under an earlier node or under the last cached token; a node sees its ancestors
    u = torch.rand(B, T, device=_device(), generator=g)
    node = torch.arange(T, device=_device())
    parent = (u * (node + 1)).floor().long() - 1
    link = (parent[:, :, None] == node) | torch.eye(T, dtype=torch.bool, device=_device())
    tree = link.float()
    for _ in range(max(1, (T - 1).bit_length())):
        tree = (tree @ tree).clamp_(max=1.0)
    x.tree = tree > 0
    x.mask = None
    if case["masked"]:           # left padding, different for every sequence; the first sequence has none
        pad = torch.randint(0, max(1, n // 2), (B,), device=_device(), generator=g)
        pad[0] = 0
        x.mask = torch.zeros(B, 1, 1, n + T, dtype=torch.half, device=_device())
        x.mask[torch.arange(n + T, device=_device()) < pad[:, None, None, None]] = -math.inf
    # the accepted tokens: `accepted` distinct nodes of each sequence in ascending order
    order = torch.rand(B, T, device=_device(), generator=g).argsort(1)[:, :case["accepted"]]
    x.path = order.sort(1).values.to(torch.int32)
    # accumulated weights: a few heavy tokens, a long tail, and a fifth that nothing ever looked at
    w = torch.exp(2.0 * normal(B, H, n))
    x.weights = torch.where(torch.rand(B, H, n, device=_device(), generator=g) < 0.2, 0.0, w)
    # positions of the tokens that an earlier eviction has moved (`again`): a third had been dropped then
    x.shift = n // 2 if case["again"] else 0
    x.arranged = n // BLOCK * BLOCK // 2 if case["again"] else 0
    x.positions = torch.rand(B, H, x.arranged + x.shift, device=_device(), generator=g).argsort(-1)[..., :x.arranged].to(torch.int32)
    return x


def _nibbles(a, b):
    return (a << 4 | b).to(torch.uint8)


def _planes(x, case):
    """The cache that holds x.kc, x.vc: planes of whole blocks, the rest in the residual buffers."""
    B, H, D = case["batch"], case["kv_heads"], case["dim"]
    _, whole, rest, most = _sizes(case)
    c = types.SimpleNamespace()
    zero = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=_device())  # noqa: E731
    nb = most // BLOCK
    c.k_first_8, c.k_mid_4, c.k_last_4 = zero(B, H, nb, D, BLOCK), zero(B, H, nb, D, BLOCK // 2), zero(B, H, nb, D, BLOCK // 2)
    c.v_first_8, c.v_mid_4, c.v_last_4 = zero(B, H, most, D), zero(B, H, most, D // 2), zero(B, H, most, D // 2)
    k = x.kc[:, :, :whole].reshape(B, H, whole // BLOCK, BLOCK, D).transpose(3, 4).contiguous().view(torch.int16)
    v = x.vc[:, :, :whole].contiguous().view(torch.int16)
    c.k_first_8[:, :, :whole // BLOCK] = (k >> 8).to(torch.uint8)
    c.k_mid_4[:, :, :whole // BLOCK] = _nibbles(k[..., 0::2] >> 4 & 15, k[..., 1::2] >> 4 & 15)
    c.k_last_4[:, :, :whole // BLOCK] = _nibbles(k[..., 0::2] & 15, k[..., 1::2] & 15)
    c.v_first_8[:, :, :whole] = (v >> 8).to(torch.uint8)
    c.v_mid_4[:, :, :whole] = _nibbles(v[..., 0::2] >> 4 & 15, v[..., 1::2] >> 4 & 15)
    c.v_last_4[:, :, :whole] = _nibbles(v[..., 0::2] & 15, v[..., 1::2] & 15)
    c.restk, c.restv = (torch.zeros(B, BLOCK, H, D, dtype=torch.half, device=_device()) for _ in range(2))
    c.restk[:, :rest] = x.kc[:, :, whole:].transpose(1, 2)
    c.restv[:, :rest] = x.vc[:, :, whole:].transpose(1, 2)
    exponent = lambda t: (t.abs().amax(2).view(torch.int16) >> 10 & 31).to(torch.uint8)[:, None]  # noqa: E731
    c.k_exp_max, c.v_exp_max = exponent(x.kc), exponent(x.vc)
    return c


def prepare(case, seed):
    x = _inputs(case, seed)
    group, whole, rest, most = _sizes(case)
    s = types.SimpleNamespace(case=case, cache=_planes(x, case), q=x.q, k=x.k, v=x.v, tree=x.tree, mask=x.mask, path=x.path,
                              shift=x.shift, arranged=x.arranged, whole=whole, rest=rest)
    B, H, n = case["batch"], case["kv_heads"], case["tokens"]
    if case["kind"] == "observe":
        s.lse = _scores(x.q, x.kc, case, x.mask).logsumexp(-1).view(B, H, -1, group).permute(0, 2, 1, 3).reshape(B, -1, H * group).contiguous()
    if case["kind"] in ("observe", "evict"):
        s.weights = torch.zeros(B, H, most, device=_device())
        s.before = torch.zeros_like(s.weights)
        s.before[..., :n] = x.weights
    if case["kind"] == "evict":
        s.positions = torch.zeros(B, H, most, dtype=torch.int32, device=_device())
        s.places = torch.zeros_like(s.positions)
        s.places[..., :x.arranged] = x.positions
    return s


# ---------------------------------------------------------------------------------------------- the plain form
def _halves(hi, mid, low):
    """Words from high bytes and the two nibble planes, whose last axis is half as long."""
    both = lambda t: torch.stack([t >> 4, t & 15], -1).flatten(-2).to(torch.int16)  # noqa: E731
    return (hi.to(torch.int16) << 8 | both(mid) << 4 | both(low)).view(torch.half)


def _keys(c, whole, rest):
    """[B,H,tokens,D] of the cache, fp16."""
    nb = whole // BLOCK
    k = _halves(c.k_first_8[:, :, :nb], c.k_mid_4[:, :, :nb], c.k_last_4[:, :, :nb]).transpose(3, 4).flatten(2, 3)
    return torch.cat([k, c.restk[:, :rest].transpose(1, 2)], 2)


def _values(c, whole, rest):
    v = _halves(c.v_first_8[:, :, :whole], c.v_mid_4[:, :, :whole], c.v_last_4[:, :, :whole])
    return torch.cat([v, c.restv[:, :rest].transpose(1, 2)], 2)


def _rows(q, kv_heads):
    """[B,T,Hq,D] -> [B,Hkv,T*group,D]"""
    B, T, Hq, D = q.shape
    return q.view(B, T, kv_heads, Hq // kv_heads, D).permute(0, 2, 1, 3, 4).reshape(B, kv_heads, -1, D)


def _scores(q, k, case, mask):
    """fp32 scores [B,Hkv,T*group,tokens]"""
    s = _rows(q, case["kv_heads"]).float() @ k.float().transpose(2, 3) / math.sqrt(case["dim"])
    return s if mask is None else s + mask[..., :k.shape[2]].float()


def _attend(s):
    case, c = s.case, s.cache
    B, H, T, D = case["batch"], case["kv_heads"], case["drafts"], case["dim"]
    group = case["heads"] // H
    old = _scores(s.q, _keys(c, s.whole, s.rest), case, s.mask)
    new = _scores(s.q, s.k.transpose(1, 2), case, None)
    seen = s.tree[:, None].repeat_interleave(group, 2)
    score = torch.cat([old, new.masked_fill(~seen, -math.inf)], -1)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    values = torch.cat([_values(c, s.whole, s.rest), s.v.transpose(1, 2)], 2).float()
    o = p @ values / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).view(B, H, T, group).permute(0, 2, 1, 3).reshape(B, T, H * group)
    return o.view(B, H, T, group, D).permute(0, 2, 1, 3, 4).reshape(B, T, H * group, D).half(), lse


def _observe(s):
    case = s.case
    B, H, n = case["batch"], case["kv_heads"], case["tokens"]
    lse = s.lse.view(B, -1, H, case["heads"] // H).permute(0, 2, 1, 3).reshape(B, H, -1, 1)
    p = torch.exp(_scores(s.q, _keys(s.cache, s.whole, s.rest), case, s.mask) - lse)
    s.weights[..., :n] += p.sum(2)
    return s.weights


def _commit(s):
    """`accepted` appends in one: rows of the residual buffer in front of the accepted tokens, whole blocks to the planes."""
    case, c = s.case, s.cache
    B, H, D, n = case["batch"], case["kv_heads"], case["dim"], case["accepted"]
    at = s.path.long()[:, :, None, None].expand(-1, -1, H, D)
    k, v = s.k.gather(1, at), s.v.gather(1, at)
    exponent = lambda t: (t.abs().amax(1, keepdim=True).view(torch.int16) >> 10 & 31).to(torch.uint8)  # noqa: E731
    c.k_exp_max.copy_(torch.maximum(c.k_exp_max, exponent(k)))
    c.v_exp_max.copy_(torch.maximum(c.v_exp_max, exponent(v)))
    rows_k, rows_v = torch.cat([c.restk[:, :s.rest], k], 1), torch.cat([c.restv[:, :s.rest], v], 1)
    full = (s.rest + n) // BLOCK * BLOCK
    if full:
        b0, b1 = s.whole // BLOCK, (s.whole + full) // BLOCK
        w = rows_k[:, :full].view(B, full // BLOCK, BLOCK, H, D).permute(0, 3, 1, 4, 2).contiguous().view(torch.int16)
        c.k_first_8[:, :, b0:b1] = (w >> 8).to(torch.uint8)
        c.k_mid_4[:, :, b0:b1] = _nibbles(w[..., 0::2] >> 4 & 15, w[..., 1::2] >> 4 & 15)
        c.k_last_4[:, :, b0:b1] = _nibbles(w[..., 0::2] & 15, w[..., 1::2] & 15)
        w = rows_v[:, :full].transpose(1, 2).contiguous().view(torch.int16)
        c.v_first_8[:, :, s.whole:s.whole + full] = (w >> 8).to(torch.uint8)
        c.v_mid_4[:, :, s.whole:s.whole + full] = _nibbles(w[..., 0::2] >> 4 & 15, w[..., 1::2] >> 4 & 15)
        c.v_last_4[:, :, s.whole:s.whole + full] = _nibbles(w[..., 0::2] & 15, w[..., 1::2] & 15)
    left = rows_k.shape[1] - full
    first = 0 if full else s.rest         # rows of the residual buffer that do not change are not written
    c.restk[:, first:left], c.restv[:, first:left] = rows_k[:, full + first:], rows_v[:, full + first:]


def _evict(s):
    case, c = s.case, s.cache
    B, H, D, keep, n, rest = case["batch"], case["kv_heads"], case["dim"], case["keep"], s.whole, s.rest
    slot = torch.arange(n, device=_device())
    place = torch.where(slot < s.arranged, s.positions[..., :n], (slot + s.shift).to(torch.int32))
    safe = place >= n + s.shift - case["recent"]
    key = torch.where(safe, math.inf, s.weights[..., :n])
    stays = torch.zeros(B, H, n, dtype=torch.bool, device=_device())
    stays.scatter_(2, key.sort(dim=-1, descending=True, stable=True).indices[..., :keep], True)
    # source of each slot below `keep`: itself, or the i-th survivor from behind for the i-th free slot
    behind = stays[..., keep:]
    to = torch.where(behind, behind.cumsum(-1) - 1, keep)          # (`keep`: a place that nothing reads)
    table = torch.zeros(B, H, keep + 1, dtype=torch.long, device=_device())
    table.scatter_(2, to, slot[keep:].expand(B, H, -1))
    free = ~stays[..., :keep]
    src = torch.where(free, table.gather(2, (free.cumsum(-1) - 1).clamp(min=0)), slot[:keep])
    for name in ("v_first_8", "v_mid_4", "v_last_4"):
        t = getattr(c, name)
        t[:, :, :keep] = t.gather(2, src[..., None].expand(-1, -1, -1, t.shape[-1]))
    nb = n // BLOCK
    flat = lambda t: t[:, :, :nb].transpose(2, 3).flatten(3)  # noqa: E731  [B,H,D,tokens]
    tile = lambda t: t.unflatten(3, (keep // BLOCK, -1)).transpose(2, 3)  # noqa: E731
    both = lambda t: torch.stack([t >> 4, t & 15], -1).flatten(-2)  # noqa: E731
    at = src[:, :, None].expand(-1, -1, D, -1)
    c.k_first_8[:, :, :keep // BLOCK] = tile(flat(c.k_first_8).gather(3, at))
    for name in ("k_mid_4", "k_last_4"):
        t = getattr(c, name)
        x = both(flat(t)).gather(3, at)
        t[:, :, :keep // BLOCK] = tile(_nibbles(x[..., 0::2], x[..., 1::2]))
        t[:, :, keep // BLOCK:nb] = 0
    s.positions[..., :keep] = place.gather(2, src)
    s.weights[..., :keep] = s.weights.gather(2, src)
    tail = s.weights[..., n:n + rest].clone()
    s.weights[..., keep:n + rest] = 0
    s.weights[..., keep:keep + rest] = tail


def run(s):
    case, c = s.case, s.cache
    kind = case["kind"]
    if own:
        from alignedkv_b200 import cache_ops
        if kind == "attend":
            return cache_ops.tree_attention(c, s.q, s.k, s.v, s.tree, rest_len=s.rest, rest_start=s.whole, mask=s.mask, lse=True)
        if kind == "observe":
            cache_ops.tree_weights(c, s.q, s.lse, s.weights, rest_len=s.rest, rest_start=s.whole, mask=s.mask)
            return s.weights
        if kind == "commit":
            cache_ops.tree_commit(c, s.k, s.v, s.path, rest_len=s.rest, rest_start=s.whole)
            return vars(c)
        s.weights.copy_(s.before)
        s.positions.copy_(s.places)
        cache_ops.evict(c, s.weights, s.positions, rest_len=s.rest, rest_start=s.whole, keep=case["keep"], recent=case["recent"],
                        arranged=s.arranged, shift=s.shift)
        return dict(vars(c), weights=s.weights, positions=s.positions)
    if kind == "attend":
        return _attend(s)
    if kind == "observe":
        return _observe(s)
    if kind == "commit":
        _commit(s)
        return vars(c)
    # (the sums of the program's last steps: an eviction changes them)
    s.weights.copy_(s.before)
    s.positions.copy_(s.places)
    _evict(s)
    return dict(vars(c), weights=s.weights, positions=s.positions)


def work(case):
    group, whole, rest, most = _sizes(case)
    B, H, Hq, D, n, T = case["batch"], case["kv_heads"], case["heads"], case["dim"], case["tokens"], case["drafts"]
    if case["kind"] == "attend":
        mask = 2 * B * n if case["masked"] else 0
        return {"bytes": 4 * B * H * (n + T) * D + 4 * B * T * Hq * D + 4 * B * T * Hq + B * T * T + mask,
                "flops": 4 * B * Hq * T * D * (n + T)}
    if case["kind"] == "observe":
        mask = 2 * B * n if case["masked"] else 0
        return {"bytes": 2 * B * H * n * D + 8 * B * H * n + 2 * B * T * Hq * D + 4 * B * T * Hq + mask,
                "flops": 2 * B * Hq * T * D * n}
    if case["kind"] == "commit":
        new, full = case["accepted"], (rest + case["accepted"]) // BLOCK * BLOCK
        left = rest + new - full
        moved = new + (rest if full else 0) + full + (left if full else new)      # rows read and written, K and V
        return {"bytes": 4 * B * H * D * moved + 4 * B * H * D + 4 * B * new, "flops": 0}
    keep = case["keep"]
    moved = keep * (whole - keep) // max(1, whole)                                # survivors from behind, evenly spread
    return {"bytes": B * H * (4 * (whole + rest) + moved * (8 * D + 16) + (whole - keep) * (D + 4)), "flops": 0}


# ---------------------------------------------------------------------------------------------- from the definition, in 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind == "commit":
        return None              # bytes: whole numbers, equal or wrong
    x = _inputs(case, seed)
    B, H, Hq, D, n, T = case["batch"], case["kv_heads"], case["heads"], case["dim"], case["tokens"], case["drafts"]
    group = Hq // H
    if kind == "evict":          # the sums move, they are not computed
        return None
    q = x.q.double() * D ** -0.5
    if kind == "attend":
        out, lse = torch.empty(B, T, Hq, D, dtype=torch.double, device=_device()), torch.empty(B, T, Hq, dtype=torch.double, device=_device())
        for b in range(B):
            add = torch.zeros(n, dtype=torch.double, device=_device()) if x.mask is None else x.mask[b, 0, 0, :n].double()
            hidden = torch.zeros(T, T, dtype=torch.double, device=_device()).masked_fill_(~x.tree[b], -math.inf)
            for h in range(H):
                rows = slice(h * group, (h + 1) * group)
                old = torch.einsum("tgd,nd->gtn", q[b, :, rows], x.kc[b, h].double()) + add
                new = torch.einsum("tgd,nd->gtn", q[b, :, rows], x.k[b, :, h].double()) + hidden
                z = torch.cat([old, new], -1)
                w = torch.softmax(z, -1).nan_to_num(0.0)
                out[b, :, rows] = torch.einsum("gtn,nd->tgd", w, torch.cat([x.vc[b, h], x.v[b, :, h]]).double())
                lse[b, :, rows] = torch.logsumexp(z, -1).t()
        return out, lse
    total = torch.zeros(B, H, _sizes(case)[3], dtype=torch.double, device=_device())
    lse = prepare(case, seed).lse.double()                                       # an input of the call
    for b in range(B):
        for h in range(H):
            rows = slice(h * group, (h + 1) * group)
            z = torch.einsum("tgd,nd->tgn", q[b, :, rows], x.kc[b, h].double())
            if x.mask is not None:
                z += x.mask[b, 0, 0, :n].double()
            total[b, h, :n] = torch.exp(z - lse[b, :, rows, None]).sum((0, 1))
    return total
