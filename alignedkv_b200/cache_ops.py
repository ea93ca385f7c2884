"""Operators around the plane cache for programs that draft several tokens at a time and keep their caches bounded.

  tree_attention   a tree of drafted tokens attends to the cache and to its own ancestors
  tree_weights     adds the attention weight that such queries give each cached token to fp32 sums
  tree_commit      the accepted path of the tree enters the cache
  evict            every (sequence, KV head) keeps its heaviest cached tokens

The reference has no counterpart: it decodes one token at a time and never drops one (model/KVCache_AlignedKV.py:81-135).

`cache` is anything with the tensors of a layer as attributes - k_first_8, k_mid_4, k_last_4, v_first_8, v_mid_4, v_last_4,
k_exp_max, v_exp_max, restk, restv, laid out as in `decode.DecodeLayer`, which is one - and `rest_start`, `rest_len` say how many
tokens are in the planes and in the residual buffers.  `DecodeLayer` offers the same operators as methods that keep those counts.
Everything is launched on torch's current stream of the tensors' device; nothing synchronises.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import _lib
from .extension._planes import cdiv, column_block

__all__ = ["tree_attention", "tree_weights", "tree_commit", "evict"]

_nothing = contextlib.nullcontext()
MOST_DRAFTED = 64


def _need(name: str, t, shape: tuple, dtype: torch.dtype, index: int) -> int:
    """The address of t, a contiguous tensor of that shape and type on that CUDA device."""
    if type(t) is not torch.Tensor and not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype is not dtype or \
            t.get_device() != index or not t.is_contiguous():
        raise RuntimeError(f"{name}: expected a contiguous {dtype} tensor of shape {shape} on cuda:{index}")
    return t.data_ptr()


class _Call:
    """A cache's tensors, checked, as the library takes them; a context in which its device is the current one.  (The checks are most of
    what a call on a short cache costs, so they are few: one look at shape, type, device and layout of each tensor that is used.)"""
    __slots__ = ("device", "index", "B", "H", "D", "L", "ptrs", "tokens")

    def __init__(self, cache, rest_len: int, rest_start: int, maxima: bool = False):
        f8 = cache.k_first_8
        if not isinstance(f8, torch.Tensor) or not f8.is_cuda or f8.dim() != 5 or f8.shape[4] != column_block:
            raise RuntimeError(f"k_first_8: expected a CUDA tensor of shape [B, H, blocks, D, {column_block}]")
        self.device = f8.device
        self.index = dev = f8.get_device()
        B, H, nmb, D, _ = f8.shape
        self.B, self.H, self.D = B, H, D
        self.L = L = cache.v_first_8.shape[2] if cache.v_first_8.dim() == 4 else -1
        if D != 128 and D != 64:
            raise RuntimeError(f"head size {D}: these operators cover 64 and 128")
        if nmb != cdiv(L, column_block):
            raise RuntimeError(f"k_first_8 has {nmb} blocks, v_first_8 {L} tokens")
        u8, nk, nv, ex, rs = torch.uint8, (B, H, nmb, D, column_block // 2), (B, H, L, D // 2), (B, 1, H, D), (B, column_block, H, D)
        self.ptrs = [
            _need("k_first_8", f8, (B, H, nmb, D, column_block), u8, dev), _need("k_mid_4", cache.k_mid_4, nk, u8, dev),
            _need("k_last_4", cache.k_last_4, nk, u8, dev), _need("v_first_8", cache.v_first_8, (B, H, L, D), u8, dev),
            _need("v_mid_4", cache.v_mid_4, nv, u8, dev), _need("v_last_4", cache.v_last_4, nv, u8, dev),
            _need("k_exp_max", cache.k_exp_max, ex, u8, dev) if maxima else None,
            _need("v_exp_max", cache.v_exp_max, ex, u8, dev) if maxima else None,
            _need("restk", cache.restk, rs, torch.half, dev), _need("restv", cache.restv, rs, torch.half, dev)]
        self.tokens = rest_start + rest_len
        if rest_start % column_block or not 0 <= rest_len < column_block or rest_start < 0 or self.tokens > L:
            raise RuntimeError(f"{rest_start} tokens in planes of {L} and {rest_len} residual ones: expected whole blocks of "
                               f"{column_block} and at most {column_block - 1}")

    def queries(self, q: torch.Tensor) -> tuple:
        """(drafted tokens, query heads) of q [B,T,Hq,D]."""
        if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[0] != self.B or q.shape[3] != self.D or \
                q.dtype is not torch.half or q.get_device() != self.index or not q.is_contiguous():
            raise RuntimeError(f"q: expected a contiguous fp16 tensor of shape [{self.B}, T, Hq, {self.D}] on {self.device}")
        T, Hq = q.shape[1], q.shape[2]
        if not 1 <= T <= MOST_DRAFTED:
            raise RuntimeError(f"q: {T} drafted tokens, expected 1 to {MOST_DRAFTED}")
        if Hq % self.H or Hq == 0:
            raise RuntimeError(f"q: {Hq} query heads are no multiple of {self.H} KV heads")
        return T, Hq

    def mask(self, mask) -> tuple:
        if mask is None:
            return None, 0
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.half or mask.device != self.device or mask.dim() != 4 or \
                mask.shape[1:3] != (1, 1) or mask.shape[0] not in (1, self.B) or mask.shape[3] < self.tokens or \
                (mask.stride(3) != 1 and mask.shape[3] > 1):
            raise RuntimeError(f"mask: expected a CUDA fp16 tensor of shape [{self.B} or 1, 1, 1, >= {self.tokens}] with a unit "
                               "stride along the positions")
        return mask.data_ptr(), (mask.stride(0) if mask.shape[0] == self.B else 0)

    def layer(self, group: int, scratch: torch.Tensor | None):
        return ctypes.byref(_lib.Layer(*self.ptrs, None if scratch is None else scratch.data_ptr(),
                                       0 if scratch is None else scratch.numel(), self.B, self.H, group, self.D, self.L))

    def here(self):
        return _nothing if torch.cuda.current_device() == self.index else torch.cuda.device(self.index)


def tree_attention(cache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tree: torch.Tensor, *, rest_len: int,
                   rest_start: int, mask: torch.Tensor | None = None, scale: float | None = None, lse: bool = False,
                   out: torch.Tensor | None = None):
    """Attention output [B,T,Hq,D] of T drafted tokens (1 to 64) that are not in the cache.

    q [B,T,Hq,D], k and v [B,T,Hkv,D] fp16; query head i reads KV head i // (Hq / Hkv).  tree: bool [T,T] or [B,T,T], True where
    the drafted token of the row sees that of the column (itself among them: nothing is implied).  Every row sees the whole cache,
    except where `mask` - the additive fp16 row of `DecodeLayer.decode`, [B,1,1,n] or [1,1,1,n] with n >= the cached tokens - is
    -inf; a token taken away by either has no part in the output, whatever its values are.  A row that sees nothing is zero.

    All planes are read: the output is that of dense attention over the cached fp16 values, with fp32 scores (times `scale`, by
    default D**-0.5), softmax and sums and one rounding to fp16.  (`DecodeLayer.decode` skips plane rows by its read decisions,
    rounds scores to fp16 and adds a mask there; the two agree within the decisions' error, not bit for bit.)

    lse=True also returns the logarithm of the rows' sums of exponentials, fp32 [B,T,Hq] (-inf where nothing is seen), which
    `tree_weights` takes.  The cache is not changed; `tree_commit` appends the accepted tokens."""
    c = _Call(cache, rest_len, rest_start)
    T, Hq = c.queries(q)
    k_ptr, v_ptr = _need("k", k, (c.B, T, c.H, c.D), torch.half, c.index), _need("v", v, (c.B, T, c.H, c.D), torch.half, c.index)
    if not isinstance(tree, torch.Tensor) or tree.dtype is not torch.bool or tree.get_device() != c.index or \
            not tree.is_contiguous() or tree.shape != (T, T) and tree.shape != (c.B, T, T):
        raise RuntimeError(f"tree: expected a contiguous bool tensor of shape [{T}, {T}] or [{c.B}, {T}, {T}] on {c.device}")
    if out is None:
        out = torch.empty_like(q)
    else:
        begin = _need("out", out, tuple(q.shape), torch.half, c.index)
        if any(begin < t.data_ptr() + 2 * t.numel() and t.data_ptr() < begin + 2 * out.numel() for t in (q, k, v)):
            raise RuntimeError("out: overlaps q, k or v")
    mask_ptr, mask_stride = c.mask(mask)
    group, lib = Hq // c.H, _lib.load()
    sums = q.new_empty((c.B, T, Hq), dtype=torch.float32) if lse else None
    with c.here():
        ws = torch.empty(max(0, lib.akv_tree_scratch_bytes(c.B, c.H, group, c.D, rest_start, T)), dtype=torch.uint8, device=c.device)
        rc = lib.akv_tree_attention(
            c.layer(group, ws), q.data_ptr(), k_ptr, v_ptr, tree.data_ptr(), T * T if tree.dim() == 3 else 0,
            mask_ptr, mask_stride, out.data_ptr(), sums.data_ptr() if lse else None, T, rest_len, rest_start,
            1.0 / math.sqrt(c.D) if scale is None else scale, _lib.raw_stream(c.index))
    _lib.check("tree_attention", rc)
    return (out, sums) if lse else out


def tree_weights(cache, q: torch.Tensor, lse: torch.Tensor, weights: torch.Tensor, *, rest_len: int, rest_start: int,
                 mask: torch.Tensor | None = None, scale: float | None = None) -> None:
    """weights[b,h,t] += sum over the query rows of KV head h of exp(score(row, t) - lse[row]) for every cached token t.

    q as in `tree_attention`, which gives lse fp32 [B,T,Hq] (its normalisation includes the drafted tokens); mask and scale as
    there.  weights: fp32 [B,Hkv,max_seq_len]; entries behind the cached tokens are left alone.  The sums are formed in one order
    (four interleaved ones over the rows, 512 rows at a time): the same call on the same state gives the same bits."""
    c = _Call(cache, rest_len, rest_start)
    T, Hq = c.queries(q)
    _need("lse", lse, (c.B, T, Hq), torch.float32, c.index)
    _need("weights", weights, (c.B, c.H, c.L), torch.float32, c.index)
    mask_ptr, mask_stride = c.mask(mask)
    with c.here():
        rc = _lib.load().akv_tree_weights(
            c.layer(Hq // c.H, None), q.data_ptr(), lse.data_ptr(), mask_ptr, mask_stride, weights.data_ptr(), T, rest_len,
            rest_start, 1.0 / math.sqrt(c.D) if scale is None else scale, _lib.raw_stream(c.index))
    _lib.check("tree_weights", rc)


def tree_commit(cache, k: torch.Tensor, v: torch.Tensor, path: torch.Tensor, *, rest_len: int, rest_start: int) -> None:
    """Append the drafted tokens path[b, 0], path[b, 1], ... of every sequence b to the cache.

    k, v [B,T,Hkv,D] as given to `tree_attention` (T 1 to 64); path int32 [B,n], n 1 to 64, node indices in the order in which they
    are appended (an index outside the tree is clamped into it; every sequence accepts the same number of tokens).  The cache is
    then what n steps of `DecodeLayer.decode` would have left: exponent maxima, residual rows, and the planes of a block that
    fills up.  The caller's counts become (rest_len + n) % 64 and rest_start + 64 if a block was filled."""
    c = _Call(cache, rest_len, rest_start, maxima=True)
    if not isinstance(k, torch.Tensor) or k.dim() != 4 or not 1 <= k.shape[1] <= MOST_DRAFTED:
        raise RuntimeError(f"k: expected a tensor of shape [B, T, H, D] with T 1 to {MOST_DRAFTED}")
    T = k.shape[1]
    k_ptr, v_ptr = _need("k", k, (c.B, T, c.H, c.D), torch.half, c.index), _need("v", v, (c.B, T, c.H, c.D), torch.half, c.index)
    if not isinstance(path, torch.Tensor) or path.dim() != 2 or not 1 <= path.shape[1] <= MOST_DRAFTED:
        raise RuntimeError(f"path: expected a tensor of shape [{c.B}, n] with n 1 to {MOST_DRAFTED}")
    n = path.shape[1]
    path_ptr = _need("path", path, (c.B, n), torch.int32, c.index)
    if c.tokens + n > c.L:
        raise RuntimeError(f"cache is full ({c.L} tokens): no room for {n} behind {c.tokens}")
    with c.here():
        rc = _lib.load().akv_tree_commit(c.layer(1, None), k_ptr, v_ptr, path_ptr, T, n, rest_len, rest_start,
                                         _lib.raw_stream(c.index))
    _lib.check("tree_commit", rc)


def evict(cache, weights: torch.Tensor, positions: torch.Tensor, *, rest_len: int, rest_start: int, keep: int, recent: int = 0,
          arranged: int = 0, shift: int = 0) -> None:
    """Reduce the rest_start tokens in the planes to `keep` (a positive multiple of 64) per (sequence, KV head), in place.

    weights fp32 [B,Hkv,max_seq_len] (`tree_weights`): the heaviest tokens stay, of equal ones those in the lower places; NaN counts
    as more than infinity.  Tokens at the last `recent` positions (at most `keep`) stay whatever their weight, residual tokens
    are not touched.  The i-th survivor in a place >= keep moves into the i-th place < keep that became free, its weight with it:
    attention does not ask for the order of cached tokens, and moving only those touches each once.

    positions int32 [B,Hkv,max_seq_len]: the sequence position of the token in each place, which an eviction writes for the
    places below `keep`.  Places from `arranged` on hold tokens in order, place p that at position p + shift: (0, 0) before the
    first eviction, after one (keep, shift + rest_start - keep).

    There is no mask: padding is a token like the others - masked queries give it no weight, and the lowest places win among equals - and what
    survives of it is no longer where a mask row could take it away.  Padding whose weight is set to -inf, and which is not among
    the `recent` positions, goes first; a caller then has to know that every sequence has `keep` other tokens in the planes.

    Afterwards: rest_start = keep; K nibble planes behind it are zero as the K writers expect; the residual tokens' weights follow
    at keep.., zeros behind them.  Exponent maxima stay, those of the tokens that go among them: `DecodeLayer.decode` then takes the read
    decisions of a cache that still had those tokens.  Where one of them had a channel's largest exponent, products of other channels
    look smaller beside it, and fewer of their planes are read than in a cache that was filled with the survivors alone."""
    c = _Call(cache, rest_len, rest_start)
    _need("weights", weights, (c.B, c.H, c.L), torch.float32, c.index)
    _need("positions", positions, (c.B, c.H, c.L), torch.int32, c.index)
    if keep <= 0 or keep % column_block or keep > rest_start:
        raise RuntimeError(f"keep: {keep}, expected a positive multiple of {column_block} of at most {rest_start}")
    most = 2 ** 31 - 1 - column_block - c.L          # (positions are 32-bit numbers)
    if not 0 <= recent <= keep or not 0 <= arranged <= rest_start or not 0 <= shift <= most:
        raise RuntimeError(f"recent {recent} [0..keep], arranged {arranged} [0..{rest_start}], shift {shift} [0..{most}]")
    lib = _lib.load()
    with c.here():
        ws = torch.empty(max(0, lib.akv_evict_scratch_bytes(c.B, c.H, rest_start, keep)), dtype=torch.uint8, device=c.device)
        rc = lib.akv_evict(c.layer(1, ws), weights.data_ptr(), positions.data_ptr(), rest_len, rest_start, keep, recent, arranged,
                           shift, _lib.raw_stream(c.index))
    _lib.check("evict", rc)
