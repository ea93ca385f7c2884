"""Operators over a cache in pages: sequences with lengths of their own, quantised as they are written.

  paged_append      keys and values of new tokens enter the pages
  paged_read        what the pages hold, as dense fp16 tensors
  paged_attention   the newest tokens of every sequence attend to it

The reference has no counterpart: its cache is one tensor per layer with one length for the whole batch (extension/k_cache_file.py:34-53,
extension/v_cache_file.py:35-54).

`cache` is anything with a layer's pool as attributes, of which `paged.PagedLayer` is one:
  k_codes, v_codes    [pages, H, page_size, D] torch.half (as they are) or torch.float8_e4m3fn, or [pages, H, page_size, D / 2] torch.uint8 (e2m1, the
                      even channel in the lower 4 bits)
  k_exps, v_exps      int8 [pages, H, page_size], for e4m3 and e2m1: the codes of a row are multiplied by 2**exp
  k_scales, v_scales  float8_e4m3fn [pages, H, page_size, D / 16], for e2m1: a factor per 16 channels
D is 64 or 128, page_size a power of two from 16 to 256.  Of a row x of D values, e4m3: exp is the least integer with max |x| <= 448 * 2**exp;
e2m1: the least with max |x| <= 2688 * 2**exp, and a scale is max |x| * 2**-exp / 6 over its channels; every rounding goes to the nearest value, ties
to even.  A row with a value that is not finite stands for NaN throughout (exp -128), except in a pool of torch.half.  (Appended exponents are
-35 to 8; of pools that something else fills, attention takes -100 to 100.)

pages int32 [B, width]: position t of sequence b lies in page pages[b, t // page_size].  An entry outside 0..pages-1 is a page that was given
up (-1, say): its tokens have no part in attention, are read as zeros, and what would be written there is dropped.  Entries behind a
sequence's last token are not looked at.  lens int32 [B], on the device: nothing here waits for it, and a captured graph replays with
what it holds then.  A length beyond the table counts as the table's, a negative one as 0.

Everything is launched on torch's current stream of the pool's device; nothing synchronises.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from .cache_ops import _need, _run

__all__ = ["paged_append", "paged_read", "paged_attention"]

MOST_ROWS = 64
_PAGES = (16, 32, 64, 128, 256)
_FORMATS = {torch.half: 0, torch.float8_e4m3fn: 1, torch.uint8: 2}
_Strides = ctypes.c_longlong * 6


def _two(name: str, a, b, shape: tuple, dtype: torch.dtype, index: int) -> tuple:
    """The addresses of k_<name> and v_<name>, contiguous tensors of that shape and type on that device: one look at both."""
    if isinstance(a, torch.Tensor) and isinstance(b, torch.Tensor) and a.shape == shape and b.shape == shape and a.dtype is dtype and \
            b.dtype is dtype and a.get_device() == index and b.get_device() == index and a.is_contiguous() and b.is_contiguous():
        return a.data_ptr(), b.data_ptr()
    return _need("k_" + name, a, tuple(shape), dtype, index), _need("v_" + name, b, tuple(shape), dtype, index)       # (says which and why)


class _Call:
    """A pool's tensors and a batch's table, checked, as the library takes them.  (As in `cache_ops`, the checks are most of what a call on few
    tokens costs: one expression each.)"""
    __slots__ = ("device", "index", "B", "W", "H", "D", "P", "pool", "pages", "lens")

    def __init__(self, cache, pages, lens):
        k, v = cache.k_codes, cache.v_codes
        if not isinstance(k, torch.Tensor) or not k.is_cuda or k.dim() != 4 or (form := _FORMATS.get(k.dtype)) is None:
            raise RuntimeError("k_codes: expected a CUDA tensor of shape [pages, H, page_size, row], torch.half, torch.float8_e4m3fn or torch.uint8")
        dtype, shape = k.dtype, k.shape
        self.index, self.device = dev, _ = k.get_device(), k.device
        N, H, P, row = shape
        D = 2 * row if form == 2 else row
        if D != 128 and D != 64:
            raise RuntimeError(f"head size {D}: these operators cover 64 and 128")
        if P not in _PAGES:
            raise RuntimeError(f"page size {P}: expected a power of two from 16 to 256")
        self.H, self.D, self.P = H, D, P
        ke = ve = ks = vs = None
        kp, vp = _two("codes", k, v, shape, dtype, dev)
        if form:
            ke, ve = _two("exps", cache.k_exps, cache.v_exps, (N, H, P), torch.int8, dev)
            if form == 2:
                ks, vs = _two("scales", cache.k_scales, cache.v_scales, (N, H, P, D // 16), torch.float8_e4m3fn, dev)
        if not isinstance(pages, torch.Tensor) or pages.dim() != 2 or pages.dtype is not torch.int32 or pages.get_device() != dev or \
                not pages.is_contiguous() or not pages.numel():
            raise RuntimeError(f"pages: expected a contiguous {torch.int32} tensor of shape [B, width] on cuda:{dev}")
        self.B, self.W = B, _ = pages.shape
        self.pages = pages.data_ptr()
        if not isinstance(lens, torch.Tensor) or lens.dtype is not torch.int32 or lens.get_device() != dev or lens.dim() != 1 or \
                lens.shape[0] != B or not lens.is_contiguous():
            raise RuntimeError(f"lens: expected a contiguous {torch.int32} tensor of shape ({B},) on cuda:{dev}")
        self.lens = lens.data_ptr()
        self.pool = _lib.Pool(kp, vp, ke, ve, ks, vs, form, N, P, H, D)


@functools.lru_cache(maxsize=256)
def _scratch_bytes(index: int, form: int, P: int, H: int, D: int, B: int, W: int, group: int, T: int) -> int:
    """Bytes of the attention's workspace on that device."""
    with torch.cuda.device(index):
        return _lib.load().akv_paged_scratch_bytes(ctypes.byref(_lib.Pool(None, None, None, None, None, None, form, 1, P, H, D)), B, W, group, T)


def _rows(name: str, x, c: _Call) -> tuple:
    """(address, tokens, strides of batch, token and head) of x [B,T,H,D] fp16, whose rows of D are contiguous and begin on 16-byte boundaries."""
    if isinstance(x, torch.Tensor) and x.dim() == 4 and x.dtype is torch.half and x.get_device() == c.index:
        (B, T, H, D), (b, t, h, unit), begin = x.shape, x.stride(), x.data_ptr()
        if B == c.B and H == c.H and D == c.D and T and unit == 1 and not begin & 15:
            if B == 1:
                b = 0
            if T == 1:
                t = 0
            if H == 1:
                h = 0
            if (b | t | h) & 7:
                raise RuntimeError(f"{name}: strides {tuple(x.stride())} do not keep its rows on 16-byte boundaries")
            return begin, T, b, t, h
    raise RuntimeError(f"{name}: expected an fp16 tensor of shape [{c.B}, T, {c.H}, {c.D}] on cuda:{c.index} with a unit stride along the channels, on a "
                       "16-byte boundary")


def paged_append(cache, k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, lens: torch.Tensor, *,
                 counts: torch.Tensor | None = None) -> None:
    """Keys and values of new tokens enter the pages, quantised as the pool holds them.

    k, v [B,T,H,D] fp16, of any strides that keep rows of D together and on 16-byte boundaries (a part of a fused projection, say).  The first
    counts[b] (int32 [B]; by default all T) tokens of sequence b go to positions lens[b], lens[b] + 1, ...; what would lie behind the
    table's end is dropped.  Nothing else in the pool changes.  lens stays: the caller adds what was appended.  Positions that
    two sequences share (pages of a common prompt) must not be appended to; where two tokens have one place, either may be left there,
    or parts of both."""
    c = _Call(cache, pages, lens)
    k_ptr, T, *of_k = _rows("k", k, c)
    v_ptr, Tv, *of_v = _rows("v", v, c)
    if Tv != T:
        raise RuntimeError(f"v: {Tv} tokens, k has {T}")
    count_ptr = None if counts is None else _need("counts", counts, (c.B,), torch.int32, c.index)
    _run("paged_append", c.index, _lib.load().akv_paged_append, ctypes.byref(c.pool), k_ptr, v_ptr, _Strides(*of_k, *of_v), c.pages, c.lens, count_ptr,
         c.B, c.W, T)


def paged_read(cache, pages: torch.Tensor, lens: torch.Tensor, most: int) -> tuple:
    """(k, v) fp16 [B,most,H,D]: positions 0..most-1 of every sequence as the pages hold them, zeros at and behind lens[b].

    The value of a code is rounded once, to fp16; beyond fp16's range to its largest."""
    c = _Call(cache, pages, lens)
    if most < 1:
        raise RuntimeError(f"most: {most} tokens, expected at least 1")
    k = torch.empty(c.B, most, c.H, c.D, dtype=torch.half, device=c.device)
    v = torch.empty_like(k)
    _run("paged_read", c.index, _lib.load().akv_paged_read, ctypes.byref(c.pool), c.pages, c.lens, k.data_ptr(), v.data_ptr(), c.B, c.W, most)
    return k, v


def paged_attention(cache, q: torch.Tensor, pages: torch.Tensor, lens: torch.Tensor, *, scale: float | None = None, lse: bool = False,
                    out: torch.Tensor | None = None):
    """Attention output [B,T,Hq,D] of the T newest tokens of every sequence.

    q [B,T,Hq,D] fp16; their keys and values are in the pages and counted by lens (`paged_append` comes first).  Query t sees the
    positions below lens[b] - (T - 1) + t: a decode step with T = 1, a chain of drafted tokens with more.  Query head i reads KV head
    i // (Hq / H); T * (Hq / H) is at most 64.  A row that sees nothing - an empty sequence, a query before its sequence's first
    token, nothing but pages that were given up - is zero.

    The output is that of dense attention over the values that the codes stand for, with fp32 scores (times `scale`, by default
    D**-0.5), softmax and sums and one rounding to fp16.  What lies in the pages behind lens[b] has no part in it, whatever it is.
    lse=True also returns the logarithm of the rows' sums of exponentials, fp32 [B,T,Hq] (-inf where nothing is seen)."""
    c = _Call(cache, pages, lens)
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.dtype is not torch.half or q.get_device() != c.index or not q.is_contiguous():
        raise RuntimeError(f"q: expected a contiguous fp16 tensor of shape [{c.B}, T, Hq, {c.D}] on {c.device}")
    B, T, Hq, D = q.shape
    if B != c.B or D != c.D:
        raise RuntimeError(f"q: expected a contiguous fp16 tensor of shape [{c.B}, T, Hq, {c.D}] on {c.device}")
    if Hq % c.H or Hq == 0:
        raise RuntimeError(f"q: {Hq} query heads are no multiple of {c.H} KV heads")
    group = Hq // c.H
    if not 1 <= T * group <= MOST_ROWS:
        raise RuntimeError(f"q: {T} tokens of {group} query heads per KV head, expected 1 to {MOST_ROWS} rows")
    if out is None:
        out = torch.empty_like(q)
    else:
        begin = _need("out", out, tuple(q.shape), torch.half, c.index)
        if begin < q.data_ptr() + 2 * q.numel() and q.data_ptr() < begin + 2 * out.numel():
            raise RuntimeError("out: overlaps q")
    sums = torch.empty(B, T, Hq, dtype=torch.float32, device=c.device) if lse else None
    size = _scratch_bytes(c.index, c.pool.format, c.P, c.H, D, B, c.W, group, T)
    ws = torch.empty(size, dtype=torch.uint8, device=c.device) if size > 0 else None
    _run("paged_attention", c.index, _lib.load().akv_paged_attention, ctypes.byref(c.pool), q.data_ptr(), c.pages, c.lens, out.data_ptr(),
         sums.data_ptr() if lse else None, None if ws is None else ws.data_ptr(), size, B, c.W, group, T,
         1.0 / math.sqrt(D) if scale is None else scale)
    return (out, sums) if lse else out
