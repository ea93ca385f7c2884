"""Operators that a program which serves many users calls around a cache in pages, as measurable cases.

  hold      the keys and values of a piece of a prompt enter the pages (`paged_ops.paged_append`), and the whole of every sequence is
            read back as dense fp16 tensors (`paged_ops.paged_read`), as the dense attention over the piece takes them.
  attend    one new token of every sequence, or a chain of a few drafted ones, attends to the sequence's pages
            (`paged_ops.paged_attention`); its keys and values are in them already.
  choose    which drafted tokens are accepted and what follows them, from the target's and the drafts' probabilities and given random
            numbers (`cache_ops.accept_drafts`).

Sequences of a batch have lengths of their own; their pages lie anywhere in the pool.  A page holds, per KV head, `page` tokens in one of
three formats:
  fp16   as they are
  e4m3   x = code 2^e: a byte per value, an exponent per token and head, the least with max |x| <= 448 2^e
  e2m1   x = code s 2^e: 4 bits per value (the even channel in the lower ones), an e4m3 scale s per 16 channels, the one nearest to their
         largest magnitude over 6, and an exponent per token and head, the least with max |x| <= 2688 2^e
Keys, values and queries are N(0,1) with four key channels per head scaled by 20, the distribution of this repository's benchmark.
"""
import math
import random
import types

import torch

own = False

OUTLIER_CHANNELS = (3, 34, 65, 96)
MOST_ATTENDED = 32 * 8 * 8192            # (sequence, KV head, token) rows of 8 bits or fewer that a drawn case attends to
MOST_PRODUCTS = 32 * 32 * 4096 * 5       # ... and of (sequence, query head, query, token)
MOST_HELD = 16 * 32 * 1000               # rows that a drawn case reads back
MOST_CHOSEN = 64 * 8 * 131072            # probabilities of a drawn case

CACHE = dict(format="e4m3", batch=1, heads=32, kv_heads=32, dim=128, page=64, tokens=0, ragged=False, new=1)
CHOICE = dict(kind="choose", batch=1, drafts=5, vocab=32000, type="float32", tree=False, point=False)


def listed():
    return [
        # a prompt of the reference's example size enters an unquantised cache: a small call, where launches and latency count
        dict(CACHE, name="hold-fp16-b1-29", kind="hold", format="fp16", page=16, tokens=29, new=29),
        # prompts of a batch, multi-head, 8 bits
        dict(CACHE, name="hold-e4m3-b16-1000", kind="hold", batch=16, tokens=1000, ragged=True, new=1000),
        # the second piece of four long prompts under grouped queries, 4 bits
        dict(CACHE, name="hold-e2m1-gqa-b4-8190", kind="hold", format="e2m1", batch=4, kv_heads=8, tokens=8190, ragged=True, new=2047),
        # one user's chat: a decode step of a single sequence of an odd length
        dict(CACHE, name="attend-fp16-b1-777", kind="attend", format="fp16", page=16, tokens=777),
        # short sequences with small heads
        dict(CACHE, name="attend-fp16-b16-1000-d64", kind="attend", format="fp16", batch=16, dim=64, tokens=1000, ragged=True),
        # the benchmark's layer, 8 bits
        dict(CACHE, name="attend-e4m3-b8-4096", kind="attend", batch=8, tokens=4096),
        # the grouped-query serving batch, lengths all over the range
        dict(CACHE, name="attend-e4m3-gqa-b64-8192", kind="attend", batch=64, kv_heads=8, tokens=8192, ragged=True),
        # one long document in 4 bits
        dict(CACHE, name="attend-e2m1-gqa-b1-131072", kind="attend", format="e2m1", kv_heads=8, page=256, tokens=131072),
        # a chain of four drafted tokens behind the newest one: 20 query rows per KV head
        dict(CACHE, name="attend-e2m1-gqa-b32-4096-t5", kind="attend", format="e2m1", batch=32, kv_heads=8, tokens=4096, ragged=True, new=5),
        # a chain of drafts of one sequence: the smallest choice
        dict(CHOICE, name="choose-b1-t5-32000"),
        # a serving batch with a large vocabulary
        dict(CHOICE, name="choose-b64-t8-131072", batch=64, drafts=8, vocab=131072),
        # trees of guessed tokens without probabilities of their own (looked up in the prompt), probabilities in fp16
        dict(CHOICE, name="choose-b8-t32-32000-point", batch=8, drafts=32, type="float16", tree=True, point=True),
    ]


def _between(rng: random.Random, low: int, high: int) -> int:
    """Spread over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choices(["hold", "attend", "choose"], [3, 6, 3])[0]
    if kind == "choose":
        case = dict(CHOICE, type=rng.choice(["float32", "float32", "float16", "bfloat16"]), tree=rng.random() < 0.5, point=rng.random() < 0.3)
        case["vocab"] = _between(rng, 1000, 262144)
        if rng.random() < 0.5:
            case["vocab"] += -case["vocab"] % 8
        case["batch"] = _between(rng, 1, min(256, MOST_CHOSEN // case["vocab"]))
        case["drafts"] = _between(rng, 1, max(1, min(32, MOST_CHOSEN // (case["vocab"] * case["batch"]))))
        return case
    group = rng.choice([1, 1, 2, 4, 4, 8])
    heads = rng.choice([8, 32, 32])
    case = dict(CACHE, kind=kind, format=rng.choice(["fp16", "e4m3", "e4m3", "e2m1", "e2m1"]), heads=heads, kv_heads=heads // group,
                dim=rng.choice([64, 128, 128, 128]), page=rng.choice([16, 32, 64, 64, 128, 256]), ragged=rng.random() < 0.7)
    case["batch"] = _between(rng, 1, 128)
    rows = (MOST_HELD if kind == "hold" else MOST_ATTENDED) // (2 if case["format"] == "fp16" else 1)
    room = max(16, rows // (case["batch"] * case["kv_heads"]))
    if kind == "hold":
        case["tokens"] = _between(rng, 1, min(16384, room))
        case["new"] = _between(rng, 1, case["tokens"])
    else:
        case["tokens"] = _between(rng, 16, min(131072, room))
        case["new"] = rng.choice([1, 1, 1, rng.randint(2, 8)])
        case["tokens"] = min(case["tokens"], max(16, MOST_PRODUCTS // (2 * case["batch"] * heads)))
        case["new"] = max(1, min(case["new"], MOST_PRODUCTS // (2 * case["batch"] * heads * case["tokens"])))
        if rng.random() < 0.3:
            case["tokens"] = max(64, case["tokens"] // 64 * 64)
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _lengths(case):
    """Tokens of each sequence with the new ones: the first has `tokens`, ragged others anything from one on."""
    n = case["tokens"]
    return [1 + math.floor((n - 1) * (b * 0.6180339887498949 % 1.0)) if case["ragged"] and b else n for b in range(case["batch"])]


def _counts(case):
    """New tokens of each sequence (hold): all of a short one are new."""
    return [min(case["new"], n) for n in _lengths(case)]


def _exponent(x, top, add):
    """The least e with max |x| <= top 2^add 2^e over the last axis (top in [1,2)), [..., 1] int32."""
    a = x.float().abs().amax(-1, keepdim=True)
    m, e = torch.frexp(a)
    return torch.where(a == 0, -24, e - 1 + (2 * m > top)).to(torch.int32) - add


def _power(e):
    return (e + 127 << 23).view(torch.float32)


def _held(x, form):
    """fp16 values [..., D] as a page holds them: codes, exponents [...], scales [..., D / 16]."""
    if form == "fp16":
        return x, None, None
    if form == "e4m3":
        e = _exponent(x, 1.75, 8)
        return (x.float() * _power(-e)).to(torch.float8_e4m3fn), e[..., 0].to(torch.int8), None
    e = _exponent(x, 1.3125, 11)
    y = (x.float() * _power(-e)).unflatten(-1, (-1, 16))
    s = (y.abs().amax(-1, keepdim=True) / 6).to(torch.float8_e4m3fn)
    t = s.float()
    a = torch.where(t > 0, y.abs() / t, 0.0)
    # the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6; from the middle of two to the one with an even number
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = (code | torch.signbit(y).to(torch.uint8) << 3).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, e[..., 0].to(torch.int8), s[..., 0]


def _values(codes, exps, scales, form):
    """What codes, exponents and scales stand for, in 32 bits."""
    if form == "fp16":
        return codes.float()
    if form == "e4m3":
        return codes.float() * _power(exps.to(torch.int32))[..., None]
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int32)
    m = n & 7
    a = torch.where(m < 2, m * 0.5, (2 + (m & 1)) * _power((m >> 1) - 2))
    a = torch.where(n > 7, -a, a).unflatten(-1, (-1, 16))
    return (a * scales.float()[..., None]).flatten(-2) * _power(exps.to(torch.int32))[..., None]


def _bytes(t):
    return t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t


def _cache(case, seed, g):
    """A pool with the sequences' tokens in it, pages in any order, and the dense inputs of the call."""
    B, H, D, P, form = case["batch"], case["kv_heads"], case["dim"], case["page"], case["format"]
    lens, dev = _lengths(case), _device()
    width = -(-max(lens) // P)
    s = types.SimpleNamespace(case=case)
    s.most = max(lens)
    s.pages = torch.randperm(B * width + 3, device=dev, generator=g)[:B * width].view(B, width).to(torch.int32)
    s.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    hot = torch.ones(D, device=dev)
    hot[[c for c in OUTLIER_CHANNELS if c < D]] = 20.0
    pool = types.SimpleNamespace()
    for name in ("k", "v"):
        codes, exps, scales = None, None, None
        for b in range(B):                     # (a sequence at a time: the largest cache in 32 bits is not needed at once)
            x = torch.randn(H, width * P, D, device=dev, generator=g)
            if name == "k":
                x *= hot
            x[:, lens[b] - (_counts(case)[b] if case["kind"] == "hold" else 0):] = 0
            parts = _held(x.half(), form)
            if b == 0:
                codes, exps, scales = (None if t is None else torch.zeros((B * width + 3, H, P) + t.shape[2:], dtype=t.dtype, device=dev)
                                       for t in parts)
            for to, t in zip((codes, exps, scales), parts):
                if to is not None:
                    _bytes(to)[s.pages[b].long()] = _bytes(t).unflatten(1, (width, P)).transpose(0, 1)
        setattr(pool, name + "_codes", codes)
        setattr(pool, name + "_exps", exps)
        setattr(pool, name + "_scales", scales)
    s.cache = pool
    if case["kind"] == "hold":
        s.counts = torch.tensor(_counts(case), dtype=torch.int32, device=dev)
        s.before = s.lens - s.counts
        s.k, s.v = (torch.randn(B, case["new"], H, D, device=dev, generator=g) for _ in range(2))
        s.k, s.v = (s.k * hot).half(), s.v.half()
    else:
        s.q = torch.randn(B, case["new"], case["heads"], D, device=dev, generator=g).half()
    return s


def prepare(case, seed):
    g = torch.Generator(device=_device()).manual_seed(1000003 * seed + 131 * case["batch"] + case.get("tokens", case.get("vocab", 0)))
    if case["kind"] != "choose":
        return _cache(case, seed, g)
    B, T, V, dev, dtype = case["batch"], case["drafts"], case["vocab"], _device(), getattr(torch, case["type"])
    s = types.SimpleNamespace(case=case, parents=None)
    up = [i - 1 for i in range(T)]
    if case["tree"]:
        up = [-1] + [math.floor(i * torch.rand(1, generator=torch.Generator().manual_seed(1009 * seed + i)).item() ** 2) for i in range(1, T)]
        s.parents = torch.tensor(up, dtype=torch.int32, device=dev)
    s.target = torch.empty(B, T, V, dtype=dtype, device=dev)
    s.draft = None if case["point"] else torch.empty_like(s.target)
    s.ids = torch.empty(B, T, dtype=torch.long, device=dev)
    gumbel = lambda: -torch.empty(T, V, device=dev).exponential_(generator=g).log_()  # noqa: E731
    row = torch.tensor([max(0, j) for j in up], device=dev)
    for b in range(B):                         # the draft model's logits are the target's with some noise; drafts are drawn from them
        z = 3 * torch.randn(T, V, device=dev, generator=g)
        y = z + torch.randn(T, V, device=dev, generator=g)
        s.target[b] = z.softmax(-1)
        if s.draft is not None:
            s.draft[b] = y.softmax(-1)
        s.ids[b] = (y[row] + gumbel()).argmax(-1)
    s.coins = torch.rand(B, T, device=dev, generator=g)
    return s


# ---------------------------------------------------------------------------------------------- the plain form
def _dense(s, name):
    """[B,H,width * page,D] in 32 bits, everything that the sequences' pages hold."""
    parts = []
    for part in ("_codes", "_exps", "_scales"):
        t = getattr(s.cache, name + part)
        if t is not None:
            x = _bytes(t)[s.pages.long()].transpose(1, 2).flatten(2, 3)
            t = x.view(t.dtype) if x.dtype is not t.dtype else x
        parts.append(t)
    return _values(*parts, s.case["format"])


def _hold(s):
    case = s.case
    P, T = case["page"], case["new"]
    i = torch.arange(T, device=_device())
    at = s.before[:, None] + i
    there = i < s.counts[:, None]
    page = s.pages.gather(1, (at // P).clamp(max=s.pages.shape[1] - 1).long())[there].long()
    slot = (at % P)[there].long()
    for name, x in (("k", s.k), ("v", s.v)):
        for part, t in zip(("_codes", "_exps", "_scales"), _held(x[there], case["format"])):
            if t is not None:
                _bytes(getattr(s.cache, name + part))[page, :, slot] = _bytes(t)
    behind = (torch.arange(s.most, device=_device()) >= s.lens[:, None])[:, :, None, None]
    return tuple(_dense(s, name)[:, :, :s.most].transpose(1, 2).clamp(-65504, 65504).half().masked_fill(behind, 0) for name in ("k", "v"))


def _attend(s):
    case = s.case
    B, H, T, D = case["batch"], case["kv_heads"], case["new"], case["dim"]
    group = case["heads"] // H
    k = _dense(s, "k")
    rows = s.q.float().view(B, T, H, group, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * group, D)
    score = rows @ k.transpose(2, 3) / math.sqrt(D)
    seen = s.lens[:, None] - (T - 1) + torch.arange(T, device=_device())                  # [B,T]: tokens that each query sees
    hidden = torch.arange(k.shape[2], device=_device()) >= seen.repeat_interleave(group, 1)[:, None, :, None]
    del k
    score = score.masked_fill_(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = p @ _dense(s, "v") / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).view(B, H, T, group).permute(0, 2, 1, 3).reshape(B, T, H * group)
    return o.view(B, H, T, group, D).permute(0, 2, 1, 3, 4).reshape(B, T, H * group, D).half(), lse


def _choose(s):
    case = s.case
    B, T, V = case["batch"], case["drafts"], case["vocab"]
    dev = _device()
    every = torch.arange(B, device=dev)
    up = torch.arange(-1, T - 1, device=dev) if s.parents is None else s.parents.long()
    now = torch.zeros(B, dtype=torch.long, device=dev)              # the node that was accepted last
    count = torch.ones(B, dtype=torch.int32, device=dev)
    path = torch.full((B, T), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    taken = torch.zeros(B, dtype=torch.double, device=dev)          # c of r = max(p - c q, 0)
    left = torch.ones(B, dtype=torch.double, device=dev)            # its sum
    gone = torch.zeros(B, V, dtype=torch.bool, device=dev)          # guesses that were rejected here
    rest = lambda c: (s.target[every, now].double() - c[:, None] * s.draft[every, now].double()).clamp_(min=0)  # noqa: E731
    for i in range(1, T):
        asked = up[i] == now
        x = s.ids[:, i]
        p, u = s.target[every, now, x].double(), s.coins[:, i].double()
        if s.draft is None:
            p = torch.where(gone[every, x], 0.0, p)
            good = asked & (u * left < p)
            bad = asked & ~good
            left = torch.where(bad, left - p, left)
            gone[every, x] |= bad
        else:
            q = s.draft[every, now, x].double()
            good = asked & (u * left * q < (p - taken * q).clamp(min=0))
            bad = asked & ~good
            taken = torch.where(bad, taken + left, taken)
            left = torch.where(bad, rest(taken).sum(-1), left)
        path[every, count.clamp(max=T - 1).long()] = torch.where(good, i, path[every, count.clamp(max=T - 1).long()])
        count += good
        now = torch.where(good, i, now)
        taken, left = torch.where(good, 0.0, taken), torch.where(good, 1.0, left)
        gone &= ~good[:, None]
    whole = s.target[every, now].double()
    r = torch.where(gone, 0.0, whole) if s.draft is None else rest(taken)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, whole)
    sums = r.cumsum(-1)
    over = sums > s.coins[:, :1].double() * sums[:, -1:]
    last = V - 1 - (r > 0).flip(-1).to(torch.uint8).argmax(-1)
    token = torch.where(over.any(-1), over.to(torch.uint8).argmax(-1), last)
    return path, count, torch.where(sums[:, -1] > 0, token, -1)


def run(s):
    kind = s.case["kind"]
    if own:
        from alignedkv_b200 import cache_ops, paged_ops
        if kind == "hold":
            paged_ops.paged_append(s.cache, s.k, s.v, s.pages, s.before, counts=s.counts)
            return paged_ops.paged_read(s.cache, s.pages, s.lens, s.most)
        if kind == "attend":
            return paged_ops.paged_attention(s.cache, s.q, s.pages, s.lens, lse=True)
        return cache_ops.accept_drafts(s.target, s.draft, s.ids, s.coins, s.parents)
    return {"hold": _hold, "attend": _attend, "choose": _choose}[kind](s)


def work(case):
    if case["kind"] == "choose":
        # one row of the target's probabilities; one of the drafts', where the walk ends with a rejection; few numbers per node
        size = 4 if case["type"] == "float32" else 2
        rows = 1 if case["point"] or case["drafts"] == 1 else 2
        return {"bytes": case["batch"] * (rows * case["vocab"] * size + case["drafts"] * (12 + 4 + 2 * size) + 16),
                "flops": case["batch"] * case["vocab"] * (1 if rows == 1 else 4)}
    H, D = case["kv_heads"], case["dim"]
    row = {"fp16": 2 * D, "e4m3": D + 1, "e2m1": D // 2 + D // 16 + 1}[case["format"]]
    total = sum(_lengths(case))
    if case["kind"] == "hold":
        new = sum(_counts(case))
        return {"bytes": 2 * H * (new * 2 * D + total * row + case["batch"] * max(_lengths(case)) * 2 * D), "flops": 2 * H * D * (new + total)}
    B, T, Hq = case["batch"], case["new"], case["heads"]
    return {"bytes": 2 * H * total * row + 4 * B * T * Hq * D + 4 * B * T * Hq + 4 * total // case["page"] + 4 * B,
            "flops": 4 * Hq * T * D * total}


# ---------------------------------------------------------------------------------------------- from the definition, in 64 bits
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(x, grid):
    """Index into the ascending grid of what lies nearest to x >= 0, from a middle to the even index; in 64 bits."""
    grid = torch.tensor(grid, dtype=torch.double, device=x.device)
    above = torch.searchsorted(grid, x.contiguous()).clamp(max=len(grid) - 1)
    below = (above - 1).clamp(min=0)
    up, down = grid[above] - x, x - grid[below]
    return torch.where((up < down) | ((up == down) & (above % 2 == 0)) | (x > grid[-1]), above, below)


E4M3 = [(m if e == 0 else 8 + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127]


def _rounded64(x, form):
    """What is read back of fp16 x [n,D]: as its definition says, in 64 bits."""
    if form == "fp16":
        return x.double()
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    grid4, grid2 = (torch.tensor(t, dtype=torch.double, device=x.device) for t in (E4M3, E2M1))
    biggest = 448.0 if form == "e4m3" else 2688.0
    tries = torch.tensor([2.0 ** e for e in range(-40, 12)], dtype=torch.double, device=x.device)
    unit = tries[((tries * biggest) < top).sum(-1, keepdim=True)]
    if form == "e4m3":
        return grid4[_nearest(x.abs() / unit, E4M3)] * x.sign() * unit
    y = (x / unit).unflatten(-1, (-1, 16))
    s = grid4[_nearest(y.abs().amax(-1, keepdim=True) / 6, E4M3)]
    a = torch.where(s > 0, y.abs() / torch.where(s > 0, s, 1.0), 0.0)
    return (grid2[_nearest(a, E2M1)] * y.sign() * s).flatten(-2) * unit


def _stored64(codes, exps, scales, form):
    """Values of one sequence's codes [n,D or D/2] in 64 bits, by tables."""
    if form == "fp16":
        return codes.double()
    raw = codes.view(torch.uint8).long()
    both = lambda grid: torch.tensor(list(grid) + [-v for v in grid], dtype=torch.double, device=raw.device)  # noqa: E731
    unit = 2.0 ** exps.double()[:, None]
    if form == "e4m3":
        return both(E4M3 + [math.nan])[raw] * unit
    pair = torch.empty(raw.shape[0], 2 * raw.shape[1], dtype=torch.long, device=raw.device)
    pair[:, 0::2], pair[:, 1::2] = raw % 16, raw // 16
    scale = both(E4M3 + [math.nan])[scales.view(torch.uint8).long()]
    return both(E2M1)[pair] * scale.repeat_interleave(16, 1) * unit


def _sequence64(s, name, b, h, n):
    """Tokens 0..n-1 of KV head h of sequence b."""
    P = s.case["page"]
    pages = s.pages[b, :-(-n // P)].long()
    get = lambda t: None if t is None else _bytes(t)[pages, h].flatten(0, 1)[:n].contiguous()  # noqa: E731
    return _stored64(*(get(getattr(s.cache, name + part)) for part in ("_codes", "_exps", "_scales")), s.case["format"])


def _walk64(s, b):
    """One sequence's choice: (path, token)."""
    up = [i - 1 for i in range(s.case["drafts"])] if s.parents is None else s.parents.tolist()
    ids, coins = s.ids[b].tolist(), s.coins[b].double().tolist()
    node, path = 0, [0]
    p = s.target[b, 0].double().clone()
    mass = 1.0
    while True:
        q = None if s.draft is None else s.draft[b, node].double()
        r, norm, following = p, mass, None
        for i in [i for i in range(node + 1, len(up)) if up[i] == node]:
            x = ids[i]
            if q is None:
                if coins[i] * norm < float(r[x]):
                    following = i
                    break
                norm -= float(r[x])
                r = r.clone()
                r[x] = 0.0
            else:
                if coins[i] * float(q[x]) * norm < float(r[x]):
                    following = i
                    break
                r = torch.clamp(r - norm * q, min=0.0)
                norm = float(r.sum())
        if following is None:
            break
        node = following
        path.append(node)
        p, mass = s.target[b, node].double().clone(), 1.0
    if float(r.sum()) <= 0.0:
        r = p
    sums = torch.cumsum(r, 0)
    found = torch.nonzero(sums > coins[0] * sums[-1])
    return path, int(found[0]) if len(found) else int(torch.nonzero(r > 0)[-1])


def exact(case, seed):
    s = prepare(case, seed)
    B = case["batch"]
    if case["kind"] == "choose":
        T = case["drafts"]
        path = torch.full((B, T), -1, dtype=torch.int32)
        count, token = torch.zeros(B, dtype=torch.int32), torch.zeros(B, dtype=torch.long)
        for b in range(B):
            nodes, token[b] = _walk64(s, b)
            count[b] = len(nodes)
            path[b, :len(nodes)] = torch.tensor(nodes, dtype=torch.int32)
        return path.to(_device()), count.to(_device()), token.to(_device())
    H, Hq, D, T, form, lens = case["kv_heads"], case["heads"], case["dim"], case["new"], case["format"], _lengths(case)
    if case["kind"] == "hold":
        out = []
        for name, x in (("k", s.k), ("v", s.v)):
            o = torch.zeros(B, s.most, H, D, dtype=torch.double, device=_device())
            for b in range(B):
                new = _counts(case)[b]
                old = lens[b] - new
                for h in range(H):
                    if old:
                        o[b, :old, h] = _sequence64(s, name, b, h, old)
                o[b, old:lens[b]] = _rounded64(x[b, :new].flatten(0, 1), form).view(new, H, D)
            out.append(o.clamp_(-65504, 65504))
        return tuple(out)
    group = Hq // H
    out = torch.zeros(B, T, Hq, D, dtype=torch.double, device=_device())
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.double, device=_device())
    for b in range(B):
        for h in range(H):
            k, v = _sequence64(s, "k", b, h, lens[b]), _sequence64(s, "v", b, h, lens[b])
            for t in range(T):
                n = lens[b] - (T - 1) + t
                if n <= 0:
                    continue
                for g in range(h * group, (h + 1) * group):
                    z = k[:n] @ (s.q[b, t, g].double() / D ** 0.5)
                    out[b, t, g], lse[b, t, g] = torch.softmax(z, 0) @ v[:n], torch.logsumexp(z, 0)
    return out, lse
