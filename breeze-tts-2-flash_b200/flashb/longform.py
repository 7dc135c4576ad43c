"""Long speech on a bounded cache: attention with a sliding window and sink tokens, a KV cache held in 4 bits, and
eviction by accumulated attention weight (``include/flashb.h``, "long speech").

The streaming decode appends one slot a frame to a bf16 cache and attends over all of it.  A reading of an hour outgrows
the cache and, long before, the time a frame may take.  Three ways to bound both, which combine:

  window + sinks   ``decode`` / ``prefill`` with ``window``: the last ``window`` slots and each row's first ``sinks``
  4 bits           ``KV4Cache``: 72 bytes a head and token instead of 256; ``store``, ``read``, ``decode``
  eviction         ``decode(..., acc=)`` adds up each slot's attention weight, ``evict`` keeps the best slots

Row b of a cache holds its keys in slots [starts[b], lengths[b]) (int64 tensors on the device, ``starts`` None = 0: the
left padding of the prompt), so every call is graph-capturable and needs no host read.  The token at slot p sees slot j
when starts[b] <= j <= p and (j > p - window or j < starts[b] + sinks); the output without a visible slot is 0.  Slots
that are not visible may hold anything, NaN included.  bf16 queries, head_dim 128, GQA groups of 1, 2, 4 or 8; fp32
scores, softmax and sums, rounded to bf16 once.  No reference counterpart: the reference's cache holds the whole
sequence in bf16 (``flash/backbone.py``).

Calls run on the current stream of the cache's device; workspaces come from torch's allocator on that stream.
"""
import ctypes
import math

import torch

from . import _native
from ._native import FB_ERR_ARG, FbKVCache, FlashbError, check

D = 128


def _ensure(cond, msg):
    if not cond:
        raise FlashbError(FB_ERR_ARG, msg)


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


class KVCache:
    """A bf16 cache: ``keys`` / ``values`` [B, NKV, S, 128] (any strides that are multiples of 8 elements, unit inner
    stride), used in place -- for example a layer's ``StaticCache`` tensors.  Build it once, use it every step."""

    bits = 16

    def __init__(self, keys, values):
        for t, n in ((keys, 'keys'), (values, 'values')):
            _ensure(t.is_cuda and t.dtype == torch.bfloat16 and t.dim() == 4 and t.shape[3] == D and t.stride(3) == 1,
                    f'{n}: [B, NKV, S, 128] bf16 CUDA with unit inner stride')
        _ensure(keys.shape == values.shape and keys.device == values.device, 'keys and values differ in shape or device')
        self.keys, self.values = keys, values
        self._set(keys, values)

    def _set(self, k, v, ks=None, vs=None, k_scale=1.0, v_scale=1.0):
        self.device = k.device
        self.B, self.NKV, self.S = k.shape[:3]
        st = list(k.stride()[:3]) + list(v.stride()[:3])
        # the stride of an axis of one entry is never used
        for i in range(6):
            if k.shape[i % 3] == 1:
                st[i] = k.shape[3] if i % 3 == 2 else 0
        d = FbKVCache(bits=self.bits, B=self.B, NKV=self.NKV, S=self.S, k=k.data_ptr(), v=v.data_ptr(), k_scale=k_scale,
                      v_scale=v_scale)
        d.k_sb, d.k_sh, d.k_sp, d.v_sb, d.v_sh, d.v_sp = st
        if ks is not None:
            d.ks, d.vs = ks.data_ptr(), vs.data_ptr()
            ss = list(ks.stride()[:3]) + list(vs.stride()[:3])
            for i in range(6):
                if ks.shape[i % 3] == 1:
                    ss[i] = ks.shape[3] if i % 3 == 2 else 0
            d.ks_sb, d.ks_sh, d.ks_sp, d.vs_sb, d.vs_sh, d.vs_sp = ss
        self.desc = d
        self._ref = ctypes.byref(d)


class KV4Cache(KVCache):
    """A cache in 4 bits: e2m1 codes ``kq`` / ``vq`` [B, NKV, S, 64] uint8 (two per byte, the even element in the low
    half) with an e4m3 scale per 16 values, ``ks`` / ``vs`` [B, NKV, S, 8] uint8.  A value stands for code x scale x
    tensor scale; ``k_scale`` / ``v_scale`` are powers of two (1 covers block maxima of 0.1 to 2688)."""

    bits = 4

    def __init__(self, kq, ks, vq, vs, k_scale=1.0, v_scale=1.0):
        for t, n, w in ((kq, 'kq', D // 2), (vq, 'vq', D // 2), (ks, 'ks', D // 16), (vs, 'vs', D // 16)):
            _ensure(t.is_cuda and t.dtype == torch.uint8 and t.dim() == 4 and t.shape[3] == w and t.stride(3) == 1,
                    f'{n}: [B, NKV, S, {w}] uint8 CUDA with unit inner stride')
            _ensure(t.shape[:3] == kq.shape[:3] and t.device == kq.device, f'{n}: rows, heads or slots differ')
        for x, n in ((k_scale, 'k_scale'), (v_scale, 'v_scale')):
            _ensure(0 < x < float('inf') and math.frexp(x)[0] == 0.5, f'{n}: a power of two')
        self.kq, self.ks, self.vq, self.vs = kq, ks, vq, vs
        self._set(kq, vq, ks, vs, float(k_scale), float(v_scale))

    @classmethod
    def empty(cls, B, NKV, S, device='cuda', k_scale=1.0, v_scale=1.0):
        """An empty (zeroed) cache of B rows, NKV heads and S slots."""
        t = [torch.zeros(B, NKV, S, w, dtype=torch.uint8, device=device) for w in (D // 2, D // 16) * 2]
        return cls(*t, k_scale=k_scale, v_scale=v_scale)

    def _slots(self, slots, L):
        _ensure(slots.dtype == torch.int64 and slots.device == self.device and slots.shape[-1] == L and
                slots.stride(-1) in (1, L) and (slots.dim() == 1 or slots.shape == (self.B, L)),
                'slots: [L] or [B, L] int64 on the cache\'s device')
        return slots.stride(0) if slots.dim() == 2 and self.B > 1 else 0

    def store(self, k, v, slots):
        """Stores bf16 heads ``k`` / ``v`` [B, NKV, L, 128] at ``slots`` ([L], or [B, L]: one list per row; distinct
        within a row, those outside the cache are skipped).  To nearest, ties to even, as in exact arithmetic."""
        for t, n in ((k, 'k'), (v, 'v')):
            _ensure(t.dtype == torch.bfloat16 and t.device == self.device and t.dim() == 4 and t.shape[0] == self.B and
                    t.shape[1] == self.NKV and t.shape[3] == D and t.stride(3) == 1 and t.shape[2] == k.shape[2],
                    f'{n}: [B, NKV, L, 128] bf16 on the cache\'s device')
        L = k.shape[2]
        sb = self._slots(slots, L)
        if L == 0:
            return
        check(_native.lib().flashb_kv4_store(self._ref, k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v),
                                             slots.data_ptr(), sb, L, _stream(self.device)))

    def read(self, slots):
        """The values at ``slots`` ([L] or [B, L]) as (k, v), each [B, NKV, L, 128] bf16 (0 outside the cache)."""
        L = slots.shape[-1]
        sb = self._slots(slots, L)
        out = torch.empty(2, self.B, self.NKV, L, D, dtype=torch.bfloat16, device=self.device)
        k, v = out[0], out[1]
        if L:
            check(_native.lib().flashb_kv4_read(self._ref, slots.data_ptr(), sb, L, k.data_ptr(), v.data_ptr(),
                                                _stream(self.device)))
        return k, v


def _strides(t):
    """(batch, head, position) strides in elements, 0 (the row for the position) where the axis has one entry."""
    s, n = t.stride(), t.shape
    return (s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else D)


def _rows(t, name, B, dev):
    _ensure(t.dtype == torch.int64 and t.device == dev and t.shape == (B,) and (B == 1 or t.stride(0) == 1),
            f'{name}: [B] int64 on the cache\'s device')
    return t.data_ptr()


def _acc(t, name, cache, least):
    _ensure(t.dtype == torch.float32 and t.device == cache.device and t.dim() == 3 and t.shape[0] == cache.B and
            t.shape[1] == cache.NKV and t.shape[2] >= least and t.stride(2) == 1,
            f'{name}: [B, NKV, {least}] fp32 on the cache\'s device with unit stride per slot')
    return t.data_ptr(), t.stride(0), t.stride(1)


def decode(query, cache, lengths, *, starts=None, window=None, sinks=0, scaling=None, acc=None, acc_out=None,
           decay=1.0, out=None):
    """Attention of one token per row, the one at slot ``lengths[b] - 1``: ``query`` [B, NH, 1, 128] bf16 over a
    ``KVCache`` or ``KV4Cache``.  Returns out [B, 1, NH, 128] bf16.

    ``window`` (None: all) and ``sinks`` choose the visible slots.  With ``acc`` [B, NKV, S] fp32 the weight of every
    slot, summed over the query heads of its group, is added: acc_out = decay acc + weight (``acc_out`` None: in place).
    The same inputs give the same bits."""
    dev, B = cache.device, cache.B
    _ensure(query.dtype == torch.bfloat16 and query.device == dev and query.dim() == 4 and query.shape[0] == B and
            query.shape[2] == 1 and query.shape[3] == D and query.stride(3) == 1,
            'query: [B, NH, 1, 128] bf16 on the cache\'s device')
    _ensure(window is None or window >= 1, 'window: at least 1, or None')
    NH = query.shape[1]
    w = 0 if window is None else int(window)
    lib = _native.lib()
    if acc is not None:
        ap = _acc(acc, 'acc', cache, cache.S)
        op = ap if acc_out is None else _acc(acc_out, 'acc_out', cache, cache.S)
    else:
        _ensure(acc_out is None, 'acc_out without acc')
        ap = op = (None, 0, 0)
    if out is None:
        out = torch.empty(B, 1, NH, D, dtype=torch.bfloat16, device=dev)
    else:
        _ensure(out.dtype == torch.bfloat16 and out.device == dev and out.is_contiguous() and out.numel() == B * NH * D,
                'out: [B, 1, NH, 128] bf16 contiguous')
    n = lib.flashb_long_decode_ws_floats(cache._ref, NH, w, sinks, acc is not None)
    if n < 0:
        check(lib.flashb_long_decode(cache._ref, query.data_ptr(), 0, 0, NH, lengths.data_ptr(), None, w, sinks, 1.0,
                                     None, 0, 0, None, 0, 0, 1.0, 16, 0, out.data_ptr(), None))
    ws = torch.empty(n, dtype=torch.float32, device=dev)
    check(lib.flashb_long_decode(
        cache._ref, query.data_ptr(), query.stride(0) if B > 1 else 0, query.stride(1) if NH > 1 else 0, NH,
        _rows(lengths, 'lengths', B, dev), None if starts is None else _rows(starts, 'starts', B, dev), w, sinks,
        D ** -0.5 if scaling is None else scaling, *ap, *op, decay, ws.data_ptr(), n, out.data_ptr(), _stream(dev)))
    return out


def prefill(query, key, value, *, window=None, sinks=0, starts=None, q_start=None, scaling=None, out=None):
    """Attention of L tokens, those at slots q_start .. q_start + L - 1 (``q_start`` None: the last L slots of
    ``key``): ``query`` [B, NH, L, 128] over ``key`` / ``value`` [B, NKV, S, 128], bf16 with any strides that are
    multiples of 8 elements.  Returns out [B, L, NH, 128] bf16.  Slots from q_start + L on are not read."""
    dev = query.device
    for t, n in ((query, 'query'), (key, 'key'), (value, 'value')):
        _ensure(t.is_cuda and t.device == dev and t.dtype == torch.bfloat16 and t.dim() == 4 and t.shape[3] == D and
                t.stride(3) == 1 and t.shape[0] == query.shape[0], f'{n}: [B, heads, slots, 128] bf16 CUDA')
    B, NH, L = query.shape[:3]
    NKV, S = key.shape[1:3]
    _ensure(value.shape == key.shape, 'key and value differ in shape')
    _ensure(window is None or window >= 1, 'window: at least 1, or None')
    if out is None:
        out = torch.empty(B, L, NH, D, dtype=torch.bfloat16, device=dev)
    else:
        _ensure(out.dtype == torch.bfloat16 and out.device == dev and out.shape == (B, L, NH, D) and out.stride(3) == 1,
                'out: [B, L, NH, 128] bf16')
    if L == 0:
        return out
    o = out.stride()
    check(_native.lib().flashb_long_prefill(
        query.data_ptr(), *_strides(query), key.data_ptr(), *_strides(key), value.data_ptr(), *_strides(value), B, NH,
        NKV, L, S, S - L if q_start is None else int(q_start), None if starts is None else _rows(starts, 'starts', B, dev),
        0 if window is None else int(window), sinks, D ** -0.5 if scaling is None else scaling, out.data_ptr(), o[0],
        o[1], o[2], _stream(dev)))
    return out


def evict(cache, acc, lengths, keep, *, into, starts=None, sinks=0, recent=0, acc_into=None, lengths_into=None):
    """Moves at most ``keep`` of each row's slots, in slot order, to slots 0, 1, .. of ``into`` (a cache of the same
    kind with at least ``keep`` slots, sharing no memory): all if there are no more, else the first ``sinks``, the last
    ``recent`` and the others of largest ``acc`` [B, NKV, S] (equal weights: the lower slot).  KV heads choose each for
    themselves.

    Returns (kept [B, NKV, keep] int32: the slot each came from, -1 beyond; lengths [B] int64 of ``into``; the moved
    weights: ``acc_into`` [B, NKV, >= keep], all of it, or a new [B, NKV, keep]; 0 beyond).  ``into``'s rows start at
    slot 0."""
    dev, B = cache.device, cache.B
    a = _acc(acc, 'acc', cache, cache.S)
    _ensure(into.bits == cache.bits and into.device == dev, 'into: a cache of the same kind on the same device')
    kept = torch.empty(B, cache.NKV, keep, dtype=torch.int32, device=dev)
    n = torch.empty(B, dtype=torch.int64, device=dev) if lengths_into is None else lengths_into
    ao = torch.empty(B, cache.NKV, keep, dtype=torch.float32, device=dev) if acc_into is None else acc_into
    check(_native.lib().flashb_kv_evict(
        cache._ref, *a, _rows(lengths, 'lengths', B, dev), None if starts is None else _rows(starts, 'starts', B, dev),
        keep, sinks, recent, into._ref, *_acc(ao, 'acc_into', into, keep), ao.shape[2], kept.data_ptr(),
        _rows(n, 'lengths_into', B, dev), _stream(dev)))
    return kept, n, ao
