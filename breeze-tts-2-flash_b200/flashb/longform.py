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
scores, softmax statistics and sums.  The weights enter the product with V as two bf16 parts (``decode``, bf16 cache: the
error of fp32 weights), in fp16 (``decode``, 4 bits: 1 % more) or as one bf16 part (``prefill``: 1.3 times).  Outputs may not
share memory with inputs or themselves (``acc`` in place is the exception).  No reference counterpart: the reference's
cache holds the whole sequence in bf16 (``flash/backbone.py``).

Calls run on the current stream of the cache's device (``prefill``: of the query's), whichever device is current;
workspaces come from torch's allocator on that stream.
"""
import ctypes
import math

import torch

from . import _native
from ._native import FB_ERR_ARG, FbKVCache, FlashbError, check

D = 128
_INT = 2 ** 31 - 1
_BF16, _I64, _F32 = torch.bfloat16, torch.int64, torch.float32
_raw_stream = torch._C._cuda_getCurrentRawStream       # device index -> cudaStream_t (current_stream() builds an object)
# The library launches on the current device and sizes grids and workspaces by it; a default stream's handle does not name
# one.  So a call for another device's cache enters that device first.
_current, _on = torch._C._cuda_getDevice, torch.cuda.device
_lib = None


def _bind():
    """The library, looked up once (``_native.lib()`` takes a lock)."""
    global _lib
    _lib = _native.lib()
    return _lib


def _refuse(msg):
    raise FlashbError(FB_ERR_ARG, msg)


def _ensure(cond, msg):
    if not cond:
        _refuse(msg)


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
        self.device, self.index = k.device, k.get_device()
        self.B, self.NKV, self.S = k.shape[:3]
        self._ws = {}
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
        n = B * NKV * S
        t = torch.zeros(n * 2 * (D // 2 + D // 16), dtype=torch.uint8, device=device).split(
            [n * D // 2, n * D // 2, n * D // 16, n * D // 16])
        kq, vq, ks, vs = (x.view(B, NKV, S, w) for x, w in zip(t, (D // 2, D // 2, D // 16, D // 16)))
        return cls(kq, ks, vq, vs, k_scale=k_scale, v_scale=v_scale)

    def _slots(self, slots, L):
        """The row stride of a slot list of L entries."""
        shape, st = slots.shape, slots.stride()
        if slots.dtype != _I64 or slots.device != self.device or (shape != (L,) and shape != (self.B, L)) or (
                L > 1 and st[-1] != 1):
            _refuse('slots: [L] or [B, L] int64 on the cache\'s device')
        return st[0] if len(st) == 2 and self.B > 1 else 0

    def _heads(self, t, L):
        shape = t.shape
        return (t.dtype == _BF16 and t.device == self.device and shape == (self.B, self.NKV, L, D) and t.stride(3) == 1)

    def store(self, k, v, slots):
        """Stores bf16 heads ``k`` / ``v`` [B, NKV, L, 128] at ``slots`` ([L], or [B, L]: one list per row; distinct
        within a row, those outside the cache are skipped).  To nearest, ties to even, as in exact arithmetic."""
        if _current() != self.index:
            with _on(self.index):
                return self.store(k, v, slots)
        L = slots.shape[-1] if slots.dim() else -1
        if not self._heads(k, L) or not self._heads(v, L):
            _refuse('k, v: [B, NKV, L, 128] bf16 on the cache\'s device, L as in slots')
        sb = self._slots(slots, L)
        if L == 0:
            return
        rc = (_lib or _bind()).flashb_kv4_store(self._ref, k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v),
                                                slots.data_ptr(), sb, L, _raw_stream(self.index))
        if rc:
            check(rc)

    def read(self, slots):
        """The values at ``slots`` ([L] or [B, L]) as (k, v), each [B, NKV, L, 128] bf16 (0 outside the cache)."""
        if _current() != self.index:
            with _on(self.index):
                return self.read(slots)
        L = slots.shape[-1] if slots.dim() else -1
        sb = self._slots(slots, L)
        k = torch.empty(self.B, self.NKV, L, D, dtype=_BF16, device=self.device)
        v = torch.empty_like(k)
        if L:
            rc = (_lib or _bind()).flashb_kv4_read(self._ref, slots.data_ptr(), sb, L, k.data_ptr(), v.data_ptr(),
                                                   _raw_stream(self.index))
            if rc:
                check(rc)
        return k, v


def _strides(t):
    """(batch, head, position) strides in elements, 0 (the row for the position) where the axis has one entry."""
    sb, sh, sp, _ = t.stride()
    nb, nh, n, _ = t.shape
    return sb if nb > 1 else 0, sh if nh > 1 else 0, sp if n > 1 else D


def _rows(t, name, B, dev):
    if t.dtype != _I64 or t.device != dev or t.shape != (B,) or not t.is_contiguous():
        _refuse(name + ': [B] int64 on the cache\'s device')
    return t.data_ptr()


def _acc(t, name, cache, least):
    shape = t.shape
    if t.dtype != _F32 or t.device != cache.device or len(shape) != 3 or shape[0] != cache.B or shape[1] != cache.NKV or \
            shape[2] < least or t.stride(2) != 1:
        _refuse(f'{name}: [B, NKV, {least}] fp32 on the cache\'s device with unit stride per slot')
    return t.data_ptr(), t.stride(0), t.stride(1)


def _span(window, sinks):
    """window (0: none) and sinks as the library's ints."""
    if window is None:
        window = 0
    elif window < 1:
        _refuse('window: at least 1, or None')
    elif window > _INT:
        window = 0                                        # longer than any cache
    if sinks < 0:
        _refuse('sinks: at least 0')
    return window, sinks if sinks < _INT else _INT


def decode(query, cache, lengths, *, starts=None, window=None, sinks=0, scaling=None, acc=None, acc_out=None,
           decay=1.0, out=None):
    """Attention of one token per row, the one at slot ``lengths[b] - 1``: ``query`` [B, NH, 1, 128] bf16 over a
    ``KVCache`` or ``KV4Cache``.  Returns out [B, 1, NH, 128] bf16.

    ``window`` (None: all) and ``sinks`` choose the visible slots.  With ``acc`` [B, NKV, S] fp32 the weight of every
    slot, summed over the query heads of its group, is added: acc_out = decay acc + weight (``acc_out`` None: in place).
    The same inputs give the same bits."""
    if _current() != cache.index:
        with _on(cache.index):
            return decode(query, cache, lengths, starts=starts, window=window, sinks=sinks, scaling=scaling, acc=acc,
                          acc_out=acc_out, decay=decay, out=out)
    dev, B = cache.device, cache.B
    shape, st = query.shape, query.stride()
    if query.dtype != _BF16 or query.device != dev or len(shape) != 4 or shape[0] != B or shape[2] != 1 or \
            shape[3] != D or st[3] != 1:
        _refuse('query: [B, NH, 1, 128] bf16 on the cache\'s device')
    window, sinks = _span(window, sinks)
    NH = shape[1]
    scored = acc is not None
    if scored:
        ap = _acc(acc, 'acc', cache, cache.S)
        op = ap if acc_out is None else _acc(acc_out, 'acc_out', cache, cache.S)
    else:
        if acc_out is not None:
            _refuse('acc_out without acc')
        ap = op = _NO_ACC
    if out is None:
        out = torch.empty(B, 1, NH, D, dtype=_BF16, device=dev)
    elif out.dtype != _BF16 or out.device != dev or not out.is_contiguous() or out.numel() != B * NH * D:
        _refuse('out: [B, 1, NH, 128] bf16 contiguous')
    lib = _lib or _bind()
    key = (NH, window, sinks, scored)                     # the workspace's size follows from the shapes alone
    n = cache._ws.get(key)
    if n is None:
        n = lib.flashb_long_decode_ws_floats(cache._ref, NH, window, sinks, scored)
        if n >= 0:
            cache._ws[key] = n
    ws = torch.empty(n, dtype=_F32, device=dev) if n > 0 else None
    rc = lib.flashb_long_decode(
        cache._ref, query.data_ptr(), st[0] if B > 1 else 0, st[1] if NH > 1 else 0, NH,
        _rows(lengths, 'lengths', B, dev), None if starts is None else _rows(starts, 'starts', B, dev), window, sinks,
        _SCALING if scaling is None else scaling, *ap, *op, decay, None if ws is None else ws.data_ptr(), n,
        out.data_ptr(), _raw_stream(cache.index))
    if rc:
        check(rc)
    return out


_SCALING = D ** -0.5
_NO_ACC = (None, 0, 0)


def _bf16_heads(t, B, dev):
    shape = t.shape
    return t.dtype == _BF16 and t.device == dev and len(shape) == 4 and shape[0] == B and shape[3] == D and t.stride(3) == 1


def prefill(query, key, value, *, window=None, sinks=0, starts=None, q_start=None, scaling=None, out=None):
    """Attention of L tokens, those at slots q_start .. q_start + L - 1 (``q_start`` None: the last L slots of
    ``key``): ``query`` [B, NH, L, 128] over ``key`` / ``value`` [B, NKV, S, 128], bf16 with positive strides
    that are multiples of 8 elements; ``scaling`` > 0.  Returns out [B, L, NH, 128] bf16.  Slots from q_start + L on are not
    read."""
    if query.is_cuda and _current() != query.get_device():
        with _on(query.get_device()):
            return prefill(query, key, value, window=window, sinks=sinks, starts=starts, q_start=q_start,
                           scaling=scaling, out=out)
    dev = query.device
    B, NH, L = query.shape[:3] if query.dim() == 4 else (0, 0, 0)
    if not query.is_cuda or not (_bf16_heads(query, B, dev) and _bf16_heads(key, B, dev) and _bf16_heads(value, B, dev)):
        _refuse('query, key, value: [B, heads, slots, 128] bf16 on one CUDA device')
    NKV, S = key.shape[1], key.shape[2]
    if value.shape != key.shape:
        _refuse('key and value differ in shape')
    window, sinks = _span(window, sinks)
    if out is None:
        out = torch.empty(B, L, NH, D, dtype=_BF16, device=dev)
    elif not _bf16_heads(out, B, dev) or out.shape != (B, L, NH, D):
        _refuse('out: [B, L, NH, 128] bf16')
    q_start = S - L if q_start is None else q_start
    if q_start < 0 or q_start + L > S:
        _refuse(f'q_start: tokens at slots {q_start} .. {q_start + L - 1} of {S}')
    if L == 0:
        return out
    ob, ol, oh, _ = out.stride()
    rc = (_lib or _bind()).flashb_long_prefill(
        query.data_ptr(), *_strides(query), key.data_ptr(), *_strides(key), value.data_ptr(), *_strides(value), B, NH,
        NKV, L, S, q_start, None if starts is None else _rows(starts, 'starts', B, dev),
        window, sinks, _SCALING if scaling is None else scaling, out.data_ptr(), ob, ol, oh,
        _raw_stream(query.get_device()))
    if rc:
        check(rc)
    return out


def evict(cache, acc, lengths, keep, *, into, starts=None, sinks=0, recent=0, acc_into=None, lengths_into=None):
    """Moves at most ``keep`` of each row's slots, in slot order, to slots 0, 1, .. of ``into`` (a cache of the same
    kind with at least ``keep`` slots, sharing no memory): all if there are no more, else the first ``sinks``, the last
    ``recent`` and the others of largest ``acc`` [B, NKV, S] (equal weights: the lower slot).  KV heads choose each for
    themselves.

    Returns (kept [B, NKV, keep] int32: the slot each came from, -1 beyond; lengths [B] int64 of ``into``; the moved
    weights: ``acc_into`` [B, NKV, >= keep], all of it, or a new [B, NKV, keep]; 0 beyond).  ``into``'s rows start at
    slot 0.  Outputs may not be the inputs' tensors."""
    if _current() != cache.index:
        with _on(cache.index):
            return evict(cache, acc, lengths, keep, into=into, starts=starts, sinks=sinks, recent=recent,
                         acc_into=acc_into, lengths_into=lengths_into)
    dev, B = cache.device, cache.B
    a = _acc(acc, 'acc', cache, cache.S)
    if into.bits != cache.bits or into.device != dev:
        _refuse('into: a cache of the same kind on the same device')
    if not 1 <= keep <= into.S or sinks < 0 or recent < 0 or sinks + recent > keep:
        _refuse(f'keep: 1 to {into.S} slots, sinks and recent among them')
    kept = torch.empty(B, cache.NKV, keep, dtype=torch.int32, device=dev)
    n = torch.empty(B, dtype=_I64, device=dev) if lengths_into is None else lengths_into
    ao = torch.empty(B, cache.NKV, keep, dtype=_F32, device=dev) if acc_into is None else acc_into
    rc = (_lib or _bind()).flashb_kv_evict(
        cache._ref, *a, _rows(lengths, 'lengths', B, dev), None if starts is None else _rows(starts, 'starts', B, dev),
        keep, sinks, recent, into._ref, *_acc(ao, 'acc_into', into, keep), ao.shape[2], kept.data_ptr(),
        _rows(n, 'lengths_into', B, dev), _raw_stream(cache.index))
    if rc:
        check(rc)
    return kept, n, ao
