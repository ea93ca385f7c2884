"""Plain 64-bit forms of the operators over pages and of the choice among drafted tokens, from their definitions, and error bounds."""
from __future__ import annotations

import math
import types

import torch

E4M3 = [(m if e == 0 else 8 + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127]
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(x, grid):
    """Index into an ascending grid of the value nearest to x >= 0; from a middle to the even index, from beyond the end to the last."""
    g = torch.tensor(grid, dtype=torch.float64, device=x.device)
    middles = (g[1:] + g[:-1]) / 2
    low, high = torch.searchsorted(middles, x.contiguous()), torch.searchsorted(middles, x.contiguous(), right=True)
    return torch.where(low % 2 == 0, low, high)


def _unit(top, biggest):
    """The least power of two u, down to that of fp16's smallest magnitude, with top <= biggest u."""
    top = torch.where(top == 0, 2.0 ** -24, top)
    tries = torch.tensor([2.0 ** e for e in range(-60, 20)], dtype=torch.float64, device=top.device)
    return tries[((tries * biggest) < top).sum(-1, keepdim=True)]


def held64(x, form):
    """What a page stands for that was given fp16 x [..., D]."""
    x = x.double()
    if form == "fp16":
        return x
    top = x.abs().amax(-1, keepdim=True)
    bad = ~x.isfinite().all(-1, keepdim=True)
    x, top = torch.where(bad, 0.0, x), torch.where(bad, 0.0, top)
    grid4, grid2 = (torch.tensor(t, dtype=torch.float64, device=x.device) for t in (E4M3, E2M1))
    unit = _unit(top, 448.0 if form == "e4m3" else 2688.0)
    if form == "e4m3":
        y = grid4[_nearest(x.abs() / unit, E4M3)] * x.sign() * unit
    else:
        z = (x / unit).unflatten(-1, (-1, 16))
        s = grid4[_nearest(z.abs().amax(-1, keepdim=True) / 6, E4M3)]
        a = torch.where(s > 0, z.abs() / torch.where(s > 0, s, 1.0), 0.0)
        y = (grid2[_nearest(a, E2M1)] * z.sign() * s).flatten(-2) * unit
    return torch.where(bad, math.nan, y)


def read16(values):
    """64-bit values as `paged_read` gives them."""
    return torch.where(values.isnan(), values, values.clamp(-65504, 65504)).half()


FORMS = ("fp16", "e4m3", "e2m1")


def make_pool(n_pages, page, heads, dim, form, device, gen):
    """A pool with random bytes in it: anything may lie where nothing was written."""
    row = {"fp16": 2 * dim, "e4m3": dim, "e2m1": dim // 2}[form]
    byte = lambda *s: torch.randint(0, 256, s, generator=gen, dtype=torch.uint8).to(device)  # noqa: E731
    dtype = {"fp16": torch.half, "e4m3": torch.float8_e4m3fn, "e2m1": torch.uint8}[form]
    p = types.SimpleNamespace(k_exps=None, v_exps=None, k_scales=None, v_scales=None)
    p.k_codes, p.v_codes = (byte(n_pages, heads, page, row).view(dtype) for _ in range(2))
    if form != "fp16":
        p.k_exps, p.v_exps = (byte(n_pages, heads, page).view(torch.int8) for _ in range(2))
    if form == "e2m1":
        p.k_scales, p.v_scales = (byte(n_pages, heads, page, dim // 16).view(torch.float8_e4m3fn) for _ in range(2))
    return p


PARTS = ("k_codes", "v_codes", "k_exps", "v_exps", "k_scales", "v_scales")


def parts(pool):
    return {n: getattr(pool, n).view(torch.uint8).clone() if getattr(pool, n).dtype is not torch.half else getattr(pool, n).view(torch.int16).clone()
            for n in PARTS if getattr(pool, n) is not None}


def pool_values(pool, which, form):
    """[pages, H, page, D] in 64 bits: what the codes of a whole pool stand for, by tables."""
    codes, exps, scales = (getattr(pool, which + n) for n in ("_codes", "_exps", "_scales"))
    if form == "fp16":
        return codes.double()
    raw = codes.view(torch.uint8).long()
    both = lambda grid: torch.tensor(grid + [-g for g in grid], dtype=torch.float64, device=raw.device)  # noqa: E731
    unit = torch.tensor([math.nan] + [2.0 ** e for e in range(-127, 128)], dtype=torch.float64, device=raw.device)[exps.long() + 128][..., None]
    if form == "e4m3":
        return both(E4M3 + [math.nan])[raw] * unit
    pair = torch.stack([raw & 15, raw >> 4], -1).flatten(-2)
    return both(E2M1)[pair] * both(E4M3 + [math.nan])[scales.view(torch.uint8).long()].repeat_interleave(16, -1) * unit


def sequence(values, pages, b, n, page, n_pages):
    """(tokens [n,H,D], whether each is there [n]) of sequence b, from pool_values."""
    H, D = values.shape[1], values.shape[3]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=values.device)
    there = torch.zeros(n, dtype=torch.bool, device=values.device)
    for i, j in enumerate(pages[b].tolist()):
        lo, hi = i * page, min(n, (i + 1) * page)
        if lo < hi and 0 <= j < n_pages:
            out[lo:hi] = values[j, :, :hi - lo].transpose(0, 1)
            there[lo:hi] = True
    return out, there


def attend64(q, k, v, there, scale):
    """One sequence: q [T,Hq,D], k, v [n,H,D], there [n] (query t sees the tokens below n - T + 1 + t): out, lse in 64 bits, mass sum_j p_j |v_j|,
    size max_j sum_d |q_d k_jd| |scale|, top max_j |v_j| (per row)."""
    T, Hq, D = q.shape
    H, n = k.shape[1], k.shape[0]
    out, mass = (torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    size, top = torch.zeros_like(lse).fill_(0), torch.zeros_like(lse).fill_(0)
    for t in range(T):
        seen = there[:max(0, n - T + 1 + t)]
        if not bool(seen.any()):
            continue
        for h in range(H):
            rows = slice(h * (Hq // H), (h + 1) * (Hq // H))
            x, kk, vv = q[t, rows].double(), k[:len(seen), h][seen], v[:len(seen), h][seen]
            s = x @ kk.T * scale
            p = torch.softmax(s, -1)
            out[t, rows], mass[t, rows], lse[t, rows] = p @ vv, p @ vv.abs(), torch.logsumexp(s, -1)
            size[t, rows] = (x.abs() @ kk.abs().T).amax(-1) * abs(scale)
            top[t, rows] = vv.abs().max()
    return out, lse, mass, size, top


def score_error(size, D):
    """D fp32 additions (an addition may cut instead of round: 2^-23 of the partial sum each), factors of the score a few steps."""
    return (D + 4) * 2.0 ** -23 * size


def out_bound(out, mass, size, top, D, n):
    """A probability is off by its score's error (twice: it is in the sum too), the exponential's 2^-21 and half an fp16 step (2^-11), which
    the sum of the rounded ones has too (another 2^-11 of the output); probabilities far below the largest lose their lower
    bits at 2^-39 of it (times values of at most twice the largest: a code's rounding up included); n / 16 additions of products, 2^-23 of the partial sums
    each; the output once more half a step, and half of fp16's smallest."""
    return mass * (2.0 ** -11 + 2 * score_error(size, D)[..., None] + 2.0 ** -20 + (n / 16 + 64) * 2.0 ** -23) + out.abs() * 2.0 ** -10 + \
        n * 2.0 ** -38 * top[..., None] + 2.0 ** -25


def lse_bound(lse, size, D, n):
    """The score's error, the sum's additions (one a token, 2^-24 each), a few steps of the logarithm."""
    return score_error(size, D) + (n + 64) * 2.0 ** -24 + 2.0 ** -21 * (1 + lse.abs())


def walk64(target, draft, ids, coins, up):
    """One sequence's choice: target, draft [T,V] (or None), ids, coins, up lists; (path, token)."""
    clean = lambda t: torch.where(t.isfinite() & (t > 0), t, 0.0)  # noqa: E731
    target = clean(target.double())
    draft = None if draft is None else clean(draft.double())
    T, V = target.shape
    node, path = 0, [0]
    while True:
        p = target[node]
        r, norm, following = p.clone(), 1.0, None
        for i in range(1, T):
            if up[i] != node or i <= node:
                continue
            x, here = ids[i], 0 <= ids[i] < V
            rx = float(r[x]) if here else 0.0
            if draft is None:
                if coins[i] * norm < rx:
                    following = i
                    break
                norm -= rx
                if here:
                    r[x] = 0.0
            else:
                qx = float(draft[node, x]) if here else 0.0
                if coins[i] * norm * qx < rx:
                    following = i
                    break
                r = (r - norm * draft[node]).clamp(min=0)
                norm = float(r.sum())
        if following is None:
            break
        node = following
        path.append(node)
    if float(r.sum()) <= 0:
        r = p
    sums = r.cumsum(0)
    if float(sums[-1]) <= 0:
        return path, -1
    coin = coins[0] if coins[0] > 0 else 0.0
    found = (sums > coin * sums[-1]).nonzero()
    return path, int(found[0]) if len(found) else int((r > 0).nonzero()[-1])
