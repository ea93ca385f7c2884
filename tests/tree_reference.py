"""Plain 64-bit forms of the operators around drafted tokens and eviction, from their definitions, and the bounds of their errors."""
from __future__ import annotations

import math

import numpy as np
import torch


def random_tree(gen, B, T, device):
    """Ancestor masks [B,T,T] of random trees: node i hangs under an earlier node or under the last cached token."""
    node = torch.arange(T)
    parent = (torch.rand(B, T, generator=gen) * (node + 1)).floor().long() - 1
    tree = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            j = i
            while j >= 0:
                tree[b, i, j] = True
                j = int(parent[b, j])
    return tree.to(device)


def attend64(q, kc, vc, k, v, tree, mask=None, scale=None):
    """q [B,T,Hq,D], cached kc, vc [B,n,H,D], drafted k, v [B,T,H,D], tree [B,T,T], mask [B,n] additive: out, lse in 64 bits, and what
    the error bounds are made of: sum_j p_j |v_j| like out, and max_j sum_d |q_d k_jd| * scale over present tokens like lse."""
    B, T, Hq, D = q.shape
    H = kc.shape[2]
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, mass = (torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse, size = (torch.zeros(B, T, Hq, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(B):
        for h in range(Hq):
            kk = torch.cat([kc[b, :, h // G], k[b, :, h // G]]).double()
            vv = torch.cat([vc[b, :, h // G], v[b, :, h // G]]).double()
            n = kc.shape[1]
            add = torch.zeros(n, dtype=torch.float64, device=q.device) if mask is None else mask[b].double()
            for t in range(T):
                here = torch.cat([add != -math.inf, tree[b, t]])
                if not bool(here.any()):
                    lse[b, t, h] = -math.inf
                    continue
                x = q[b, t, h].double()
                s = (kk[here] @ x) * scale + torch.cat([add, torch.zeros(T, dtype=torch.float64, device=q.device)])[here]
                p = torch.softmax(s, 0)
                out[b, t, h] = p @ vv[here]
                mass[b, t, h] = p @ vv[here].abs()
                lse[b, t, h] = torch.logsumexp(s, 0)
                size[b, t, h] = (kk[here].abs() @ x.abs()).max() * abs(scale)
    return out, lse, mass, size


def score_error(size, D):
    """Bound of a score's error: D fp32 additions (an addition may cut instead of round: 2^-23 of the partial sum each), the product
    with the factor and log2(e), whose own roundings are a few steps of the score."""
    return (D + 4) * 2.0 ** -23 * size


def out_bound(out, mass, size, D):
    """A probability is off by its score's error (twice: it is in the sum too), the exponential's 2^-21 and half an fp16 step (2^-11); the
    output once more by half a step, and by half of fp16's smallest."""
    return mass * (2.0 ** -11 + 2 * score_error(size, D)[..., None] + 2.0 ** -20) + out.abs() * 2.0 ** -11 + 2.0 ** -25


def lse_bound(lse, size, D, n):
    """The score's error, the sum's additions (one a token within a lane, 2^-24 each; a lane holds a quarter of them), a few steps of
    the logarithm."""
    return score_error(size, D) + (n / 4 + 64) * 2.0 ** -24 + 2.0 ** -21 * (1 + lse.abs())


def weights64(q, kc, lse, mask=None, scale=None):
    """sum over the rows of each KV head of exp(score - lse): [B,H,n], and max_d-sum like `size` [B,H,n]."""
    B, T, Hq, D = q.shape
    H, n = kc.shape[2], kc.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    total, size = (torch.zeros(B, H, n, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(B):
        for h in range(Hq):
            kk = kc[b, :, h // (Hq // H)].double()
            for t in range(T):
                if lse[b, t, h] == -math.inf:
                    continue
                s = kk @ q[b, t, h].double() * scale
                if mask is not None:
                    s = s + mask[b].double()
                    s[mask[b] == -math.inf] = -math.inf
                total[b, h // (Hq // H)] += torch.exp(s - lse[b, t, h].double())
                size[b, h // (Hq // H)] = torch.maximum(size[b, h // (Hq // H)], kk.abs() @ q[b, t, h].double().abs() * abs(scale))
    return total, size


def evict_plan(weights, positions, n, keep, recent, arranged, shift):
    """Source place of every place below keep, [rows][keep], by sorting (numpy, one row at a time)."""
    rows = []
    for w, pos in zip(weights.reshape(-1, weights.shape[-1]), positions.reshape(-1, positions.shape[-1])):
        place = np.where(np.arange(n) < arranged, pos[:n], np.arange(n) + shift)
        rank = sorted(range(n), key=lambda i: (0 if place[i] >= n + shift - recent else 1 if np.isnan(w[i]) else 2,
                                               0.0 if place[i] >= n + shift - recent or np.isnan(w[i]) else -float(w[i]), i))
        kept = set(rank[:keep])
        movers = [i for i in range(keep, n) if i in kept]
        src = list(range(keep))
        for d, m in zip([i for i in range(keep) if i not in kept], movers):
            src[d] = m
        rows.append((src, place))
    return rows
