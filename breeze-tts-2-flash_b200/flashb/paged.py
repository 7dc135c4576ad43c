"""Many readings on the pages of one cache: rows of any length, any number of new tokens of each in a step
(``include/flashb.h``, "paged cache").

A server that decodes many streams, feeds prompts in chunks beside them and lets streams come and go cannot give each the
longest row's cache.  Here slot j of row b lies in page ``table[b, j // page]`` of a shared pool, and a step's tokens are
the rows' runs one after the other:

  ``append``   qkv projections -> head norms, rotary positions, K and V into their pages; returns q
  ``attend``   attention of those tokens over their rows' pages, causal, optionally with a window and sink tokens

``table`` [B, W] int32 (-1 where a row has no page: its slots are not visible, and nothing is written there), ``lengths``
[B] int64: how many slots of each row are in use, the step's tokens among them; ``offsets`` [B + 1] int64: row b's tokens
are offsets[b] .. offsets[b + 1] - 1 of the step's (not decreasing; None: one token a row).  All of them are on the device
and read there, so every call is graph-capturable; tokens behind offsets[B] are left as they are, so that a graph may be
captured for more tokens than a step has.  In a step of at most one token a row leave idle rows out of ``table`` and
``lengths`` and call without ``offsets``: the form of single tokens is more exact and quicker (128 rows to 8192 slots, a
quarter of them idle: 133 us, as runs 150).  bf16, head_dim 128, GQA groups of 1, 2, 4 or 8; fp32 scores, softmax statistics
and sums, rounded once; the weights enter the product with V as two bf16 parts (one token a row: the error of fp32 weights)
or one (runs: 1.2 to 1.4 times that).  The form and the workspace of ``attend`` go by the table's width: give it no more
columns than the longest row needs (``table[:, :n]``).  Outputs may not share memory with inputs (``append``'s q in place of
its projections is the exception).  No reference counterpart: the reference's cache is one request's
(``flash/backbone.py``).

Calls run on the current stream of the cache's device, whichever device is current; workspaces come from torch's allocator
on that stream.
"""
import ctypes
import math

import torch

from . import _native
from ._native import FbPagedCache, check
from .longform import D, _BF16, _I64, _current, _ensure, _on, _raw_stream, _refuse, _span

_I32 = torch.int32
_HEAD = (D,)
_SCALING = D ** -0.5
_lib = None


def _bind():
    global _lib
    _lib = _native.lib()
    return _lib


class PagedCache:
    """A pool of pages, used in place: ``keys`` / ``values`` [pages, NKV, page, 128] bf16 with unit inner stride and other
    strides that are multiples of 8 elements (so also a view of [pages, page, NKV, 128]); ``page`` a power of two from 16
    on.  Build it once, use it every step."""

    def __init__(self, keys, values):
        for t, n in ((keys, 'keys'), (values, 'values')):
            _ensure(t.is_cuda and t.dtype == _BF16 and t.dim() == 4 and t.shape[3] == D and t.stride(3) == 1,
                    f'{n}: [pages, NKV, page, 128] bf16 CUDA with unit inner stride')
        _ensure(keys.shape == values.shape and keys.device == values.device, 'keys and values differ in shape or device')
        P, H, n = keys.shape[:3]
        _ensure(P >= 1 and H >= 1 and n >= 16 and n & (n - 1) == 0, f'{P} pages of {n} slots: a power of two from 16 on')
        self.keys, self.values = keys, values
        self.device, self.index = keys.device, keys.get_device()
        self.pages, self.NKV, self.page = P, H, n
        d = FbPagedCache(pages=P, NKV=H, page=n, k=keys.data_ptr(), v=values.data_ptr())
        # the stride of an axis of one entry is never used
        st = [s if m > 1 else D * i for t in (keys, values) for s, m, i in zip(t.stride(), t.shape[:3], (n, n, 1))]
        d.k_sb, d.k_sh, d.k_sl, d.v_sb, d.v_sh, d.v_sl = st
        self.desc = d
        self._ref = ctypes.byref(d)
        self._ws = {}

    @classmethod
    def empty(cls, pages, NKV, page=64, device='cuda'):
        """A zeroed pool."""
        return cls(*(torch.zeros(pages, NKV, page, D, dtype=_BF16, device=device) for _ in range(2)))


class Rotary:
    """Rotary positions of the first ``dim`` dims of a head (a multiple of 16 up to 128): pair i turns by position x
    freq[i] radians, freq[i] = base^(-2 i / dim).  ``layout`` 'half': pairs (i, i + dim / 2), 'interleaved': (2 i, 2 i + 1).

    ``scaling`` for contexts longer than those of the training:
      dict(kind='linear', factor=f)                  positions divided by f
      dict(kind='ntk', factor=f)                     base times f^(dim / (dim - 2)): the fastest pair as it was, the
                                                     slowest divided by f
      dict(kind='yarn', factor=f, original=n)        pairs that make ``fast`` (32) turns and more in n positions as they
                                                     were, those of ``slow`` (1) or fewer divided by f, a ramp between;
                                                     amplitude 0.1 ln f + 1
    ``freq`` [dim / 2] gives the radians per position themselves, ``amplitude`` the factor of the rotated dims."""

    def __init__(self, dim=D, base=1e4, layout='half', scaling=None, freq=None, amplitude=None, device='cuda'):
        _ensure(0 < dim <= D and dim % 16 == 0, f'rotary: {dim} dims (a multiple of 16 up to {D})')
        _ensure(layout in ('half', 'interleaved'), f'rotary: layout {layout!r}')
        _ensure(base > 1, f'rotary: base {base}')
        self.dim, self.layout = dim, layout
        amp = 1.0
        if freq is None:
            freq, amp = self._freq(dim, float(base), dict(scaling or {}))
        else:
            _ensure(scaling is None, 'rotary: freq and scaling')
            freq = torch.as_tensor(freq, dtype=torch.float64).cpu()
            _ensure(freq.shape == (dim // 2,), f'rotary: freq [{dim // 2}]')
        _ensure(bool(torch.isfinite(freq).all()), 'rotary: freq not finite')
        self.freq = freq
        self.amplitude = float(amp if amplitude is None else amplitude)
        _ensure(math.isfinite(self.amplitude), 'rotary: amplitude not finite')
        self.turns = (freq / (2 * math.pi)).to(device)
        _ensure(self.turns.is_cuda, 'rotary: a CUDA device')
        self.device, self._index = self.turns.device, self.turns.get_device()
        self._args = (self.turns.data_ptr(), dim, int(layout == 'interleaved'), self.amplitude)

    @staticmethod
    def _freq(dim, base, how):
        kind = how.pop('kind', None)
        _ensure(kind is not None or not how, f'rotary: scaling {sorted(how)} without a kind')
        f = float(how.pop('factor', 1.0))
        _ensure(kind in (None, 'linear', 'ntk', 'yarn'), f'rotary: scaling {kind!r}')
        _ensure(f > 0 and math.isfinite(f), f'rotary: factor {f}')
        if kind == 'ntk':
            base *= f ** (dim / (dim - 2))
        i = torch.arange(dim // 2, dtype=torch.float64)
        freq = torch.tensor(base, dtype=torch.float64) ** (-2 * i / dim)
        amp = 1.0
        if kind == 'linear':
            freq = freq / f
        elif kind == 'yarn':
            n, fast, slow = how.pop('original', 0), how.pop('fast', 32.0), how.pop('slow', 1.0)
            _ensure(n > 0 and fast > slow > 0, f'rotary: {n} positions, {fast} and {slow} turns')

            def pair(turns):                              # which pair makes that many turns in n positions
                return dim * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))
            lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
            ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            freq = freq * (1 - ramp) + freq / f * ramp
            amp = 0.1 * math.log(f) + 1 if f > 1 else 1.0
        _ensure(not how, f'rotary: scaling {sorted(how)}')
        return freq, amp


# The checks below are what a call of some microseconds spends its time on: attributes once, devices by index.
def _step(index, table, lengths, offsets, T):
    """The step's (table, its row stride, rows, width, lengths, offsets) as the library takes them."""
    if table.dtype is not _I32 or table.get_device() != index or table.dim() != 2:
        _refuse('table: [B, W] int32 on the cache\'s device')
    B, W = table.shape
    tb, tw = table.stride()
    if B < 1 or W < 1 or (tw != 1 and W > 1):
        _refuse('table: [B, W] with unit inner stride, not empty')
    if lengths.dtype is not _I64 or lengths.get_device() != index or lengths.shape != (B,) or not lengths.is_contiguous():
        _refuse('lengths: [B] int64 on the cache\'s device')
    if offsets is None:
        if T != B:
            _refuse(f'{T} tokens of {B} rows without offsets')
        return table.data_ptr(), tb if B > 1 else W, B, W, lengths.data_ptr(), None
    if offsets.dtype is not _I64 or offsets.get_device() != index or offsets.shape != (B + 1,) or not offsets.is_contiguous():
        _refuse('offsets: [B + 1] int64 on the cache\'s device')
    return table.data_ptr(), tb if B > 1 else W, B, W, lengths.data_ptr(), offsets.data_ptr()


def _tokens(t, name, index, T=None, H=None):
    """(tokens, heads, token stride, head stride) of [T, heads, 128] bf16."""
    if t.dtype is not _BF16 or t.get_device() != index or t.dim() != 3:
        _refuse(f'{name}: [T, heads, 128] bf16 on the cache\'s device')
    n, h, d = t.shape
    st, sh, sd = t.stride()
    if d != D or sd != 1 or (T is not None and (n != T or h != H)):
        _refuse(f'{name}: {f"[{T}, {H}, 128]" if T is not None else "[T, heads, 128]"} with unit inner stride')
    return n, h, st if n > 1 else h * D, sh if h > 1 else D


def _norm(w, name, index):
    if w.dtype is not _BF16 or w.get_device() != index or w.shape != _HEAD or not w.is_contiguous():
        _refuse(f'{name}: [128] bf16 on the cache\'s device')
    return w.data_ptr()


def append(qkv, cache, table, lengths, *, offsets=None, rotary=None, q_norm=None, k_norm=None, eps=1e-6, positions=None,
           out=None):
    """The step's raw projections ``qkv`` [T, (NH + 2 NKV) 128] bf16 (unit inner stride): q and k heads through their RMS
    norms (weights ``q_norm`` / ``k_norm`` [128] bf16, or neither) and ``rotary``, K and V to their slots of ``cache``.
    Returns q [T, NH, 128] bf16 (``out``: where; the q heads of ``qkv`` itself are allowed).

    Row b's run ends at slot lengths[b] - 1; ``positions`` [T] int64 (None: the slot) is what rotates.  In fp32, rounded
    once; the angle is reduced in 64 bits (off by 2^-20 radians at position 2^31).  Slots outside a row's pages are skipped.
    No two tokens may have the same slot."""
    index = cache.index
    if _current() != index:
        with _on(index):
            return append(qkv, cache, table, lengths, offsets=offsets, rotary=rotary, q_norm=q_norm, k_norm=k_norm, eps=eps,
                          positions=positions, out=out)
    if qkv.dtype is not _BF16 or qkv.get_device() != index or qkv.dim() != 2:
        _refuse('qkv: [T, (NH + 2 NKV) 128] bf16 on the cache\'s device')
    T, n = qkv.shape
    ld, one = qkv.stride()
    NH = n // D - 2 * cache.NKV
    if NH < 1 or n % D or one != 1:
        _refuse(f'qkv: [T, {n}] with unit inner stride, 128 a head, 2 x {cache.NKV} heads of them keys and values')
    step = _step(index, table, lengths, offsets, T)
    qn = None if q_norm is None else _norm(q_norm, 'q_norm', index)
    kn = None if k_norm is None else _norm(k_norm, 'k_norm', index)
    if rotary is None:
        rot = _NO_ROTARY
    else:
        rot = rotary._args
        if rotary._index != index:
            _refuse('rotary: on another device')
    if positions is not None and (positions.dtype is not _I64 or positions.get_device() != index or
                                  positions.shape != (T,) or not positions.is_contiguous()):
        _refuse('positions: [T] int64 on the cache\'s device')
    if out is None:
        out = qkv.new_empty((T, NH, D))
        st, sh = NH * D, D
    else:
        _, _, st, sh = _tokens(out, 'out', index, T, NH)
    if T == 0:
        return out
    rc = (_lib or _bind()).flashb_paged_append(
        cache._ref, *step, T, qkv.data_ptr(), ld if T > 1 else n, NH, qn, kn, eps, *rot,
        None if positions is None else positions.data_ptr(), out.data_ptr(), st, sh, _raw_stream(index))
    if rc:
        check(rc)
    return out


_NO_ROTARY = (None, 0, 0, 1.0)


def attend(query, cache, table, lengths, *, offsets=None, window=None, sinks=0, scaling=None, out=None):
    """Attention of the step's tokens over their rows' pages: ``query`` [T, NH, 128] bf16 (strides that are positive
    multiples of 8 elements; 16-byte aligned).  Returns out [T, NH, 128] bf16.

    Row b's run ends at slot lengths[b] - 1 (lengths past the row's pages count as those).  The token at slot p sees slot j
    when j <= p and, with a ``window``, j > p - window or j < ``sinks``; slots of pages that are not there (-1) are not
    seen; a token that sees none gives 0.  Slots that are not seen may hold anything, NaN included; entries of pages that
    no token sees are not read.  ``scaling`` > 0 (None: 128^-0.5).  The same inputs give the same bits.  Without ``offsets``
    out is contiguous."""
    index = cache.index
    if _current() != index:
        with _on(index):
            return attend(query, cache, table, lengths, offsets=offsets, window=window, sinks=sinks, scaling=scaling,
                          out=out)
    T, NH, q_st, q_sh = _tokens(query, 'query', index)
    step = _step(index, table, lengths, offsets, T)
    if window is None and sinks == 0:
        window = 0
    else:
        window, sinks = _span(window, sinks)
    if out is None:
        out = query.new_empty((T, NH, D))
        o_st, o_sh = NH * D, D
    else:
        _, _, o_st, o_sh = _tokens(out, 'out', index, T, NH)
        if offsets is None and not out.is_contiguous():
            _refuse('out: contiguous without offsets')
    if T == 0:
        return out
    lib = _lib or _bind()
    B, W = step[2], step[3]
    key = (B, W, T, NH, window, sinks, offsets is None)   # the workspace's size follows from the shapes alone
    n = cache._ws.get(key)
    if n is None:
        n = (lib.flashb_paged_decode_ws_floats(cache._ref, B, W, NH, window, sinks) if offsets is None else
             lib.flashb_paged_attend_ws_floats(cache._ref, B, W, T, NH, window, sinks))
        if n >= 0:
            if len(cache._ws) >= 256:                     # steps of ever other sizes
                cache._ws.clear()
            cache._ws[key] = n
    ws, wp = None, None
    if n > 0:
        ws = query.new_empty(2 * n)                       # bf16: two a float
        wp = ws.data_ptr()
    if scaling is None:
        scaling = _SCALING
    if offsets is None:
        rc = lib.flashb_paged_decode(cache._ref, *step[:5], query.data_ptr(), q_st, q_sh, NH, window, sinks, scaling, wp, n,
                                     out.data_ptr(), _raw_stream(index))
    else:
        rc = lib.flashb_paged_attend(cache._ref, *step, T, query.data_ptr(), q_st, q_sh, NH, window, sinks, scaling, wp, n,
                                     out.data_ptr(), o_st, o_sh, _raw_stream(index))
    if rc:
        check(rc)
    return out
