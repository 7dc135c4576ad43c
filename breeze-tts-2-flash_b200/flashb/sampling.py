"""The backbone sampler on the device, with the reference's Python surface (``flash/sampling.py``).

``sample_logits(logits, *, temperature, top_k, top_p, do_sample, present, repetition_penalty, suppress_idx, ok_true)``
returns ``(token, ok)`` like the reference's host-sync-free sampler (``flash/sampling.py:56-97``): the official op
order (repetition penalty on the ids in ``present``, suppression, greedy argmax or temperature / top-k / top-p /
softmax / multinomial) and the multinomial's validity predicate as a device flag instead of a device-side assert.
Here it is one ``flashb_cb0_sample`` launch (one CTA per row) instead of ~10 torch ops.  The multinomial draw is
``argmax(probs / q)`` with ``q`` Exp(1) draws (the identity ``torch.multinomial(p, 1) == argmax(p / Exp(1))``): pass
``q`` to control the randomness, else it is drawn on the device from torch's generator.

``token_scores`` says what logits say of given tokens: log probability, entropy, rank, the likeliest alternatives (the
reference has none).
"""
from typing import NamedTuple

import torch

from . import _native
from ._native import check

_INF = float('inf')
_F32, _BF16, _I64 = torch.float32, torch.bfloat16, torch.int64
_AS_F32, _AS_IS = dict(dtype=_F32), {}
_current, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_lib = None


def _bind():
    """The library, looked up once (``_native.lib()`` takes a lock)."""
    global _lib
    _lib = _native.lib()
    return _lib


def _refuse(msg):
    raise _native.FlashbError(_native.FB_ERR_ARG, msg)


class InvalidDistribution(RuntimeError):
    """The backbone sampling distribution is invalid (nan / inf / negative / all-zero probabilities); raised for the
    current request only (the reference's name, ``flash/sampling.py:25-29``)."""


def _rows(t, rows, dtype, device):
    t = torch.as_tensor(t, device=device).to(dtype)
    return (t.reshape(1).expand(rows) if t.numel() == 1 else t.reshape(rows)).contiguous()


def sample_rows(logits, temperature, top_k, top_p, do_sample, present=None, repetition_penalty=1.0,
                suppress_idx=None, q=None, tokens=None, pair_half=0, ok=None, mark_present=False):
    """Every row of ``logits`` [rows, V] fp32 at once (per-row parameters: scalars or [rows] tensors).  Returns
    (tokens, ok [rows] int64 0/1): tokens [rows], or with ``pair_half`` = h > 0 the [2 rows] backbone ids of CFG
    blocks [cond_0 .. cond_{h-1}, uncond_0 .. uncond_{h-1}] (row r's token in both rows of its pair).  ``present``
    [rows, V] uint8/bool presence masks (updated in place with the sampled tokens when ``mark_present``)."""
    def _ensure(cond, msg):
        if not cond:
            raise _native.FlashbError(_native.FB_ERR_ARG, msg)

    _ensure(logits.dtype == torch.float32 and logits.is_cuda and logits.dim() == 2 and logits.stride(1) == 1,
            'logits: [rows, V] fp32 CUDA with unit stride')
    rows, V = logits.shape
    dev = logits.device
    temp = _rows(temperature, rows, torch.float32, dev)
    topk = _rows(top_k, rows, torch.int64, dev)
    topp = _rows(top_p, rows, torch.float32, dev)
    ds = _rows(do_sample, rows, torch.int64, dev)
    if q is None:
        q = torch.empty(rows, V, dtype=torch.float32, device=dev).exponential_(1.0)
    _ensure(q.dtype == torch.float32 and q.shape == (rows, V) and q.stride(1) == 1, 'q: [rows, V] fp32')
    if present is not None:
        _ensure(present.dtype in (torch.uint8, torch.bool) and present.shape[-1] == V and present.stride(-1) == 1,
                'present: [rows, V] uint8/bool')
        present = present.view(torch.uint8) if present.dtype == torch.bool else present
        ldp = present.stride(0) if present.dim() == 2 and present.shape[0] == rows else 0
        _ensure(ldp >= V, 'present: one row per logits row')
    sup = None
    if suppress_idx is not None and suppress_idx.numel() > 0:
        sup = suppress_idx.to(device=dev, dtype=torch.int64).contiguous()
    if tokens is None:
        tokens = torch.empty(2 * rows if pair_half else rows, dtype=torch.int64, device=dev)
    _ensure(tokens.dtype == torch.int64 and tokens.is_contiguous() and tokens.numel() >= (2 if pair_half else 1) * rows,
            'tokens: int64, contiguous, one per row (two with pair_half)')
    ok = torch.empty(rows, dtype=torch.int64, device=dev) if ok is None else ok
    _p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    check(_native.lib().flashb_cb0_sample(
        logits.data_ptr(), logits.stride(0), rows, V, _p(present), ldp if present is not None else 0,
        float(repetition_penalty), _p(sup), 0 if sup is None else sup.numel(), temp.data_ptr(), topk.data_ptr(),
        topp.data_ptr(), ds.data_ptr(), q.data_ptr(), q.stride(0), tokens.data_ptr(), int(pair_half), ok.data_ptr(),
        int(bool(mark_present)), torch.cuda.current_stream(dev).cuda_stream))
    return tokens, ok


def sample_logits(logits, *, temperature, top_k, top_p, do_sample, present=None, repetition_penalty=1.0,
                  suppress_idx=None, ok_true=None, q=None):
    """Drop-in for the reference's ``sample_logits``: logits [..., V] (one row), returns (token of shape
    logits.shape[:-1], 0-dim bool ok) on the device, no host sync."""
    shape = logits.shape[:-1]
    x = logits.reshape(-1, logits.shape[-1]).float().contiguous()
    pres = None
    if present is not None:
        pres = present.reshape(-1, present.shape[-1]).to(torch.uint8)
        if pres.shape[0] == 1 and x.shape[0] > 1:
            pres = pres.expand(x.shape[0], -1).contiguous()
    tok, ok = sample_rows(x, temperature, top_k, top_p, do_sample, pres, repetition_penalty, suppress_idx,
                          q=None if q is None else q.reshape(x.shape).float().contiguous())
    return tok.view(shape), ok.bool().all()


class TokenScores(NamedTuple):
    """``token_scores``'s answer, a row of logits each."""
    logprob: torch.Tensor        # [rows] fp32: log probability of the given token
    entropy: torch.Tensor        # [rows] fp32: of the row's distribution, in nats
    rank: torch.Tensor           # [rows] int64: ids ahead of the given token (0: the greedy choice)
    top_ids: torch.Tensor        # [rows, top] int64: the likeliest ids, in order
    top_logprobs: torch.Tensor   # [rows, top] fp32: theirs


def token_scores(logits, tokens, *, top=0, temperature=1.0):
    """What ``logits`` [rows, V] (fp32 or bf16, unit inner stride, rows at least V apart; CFG logits, or the logits of a given
    reading) say of ``tokens`` [rows] int64 under softmax(logits / temperature): a ``TokenScores``, in one launch.

    Larger logits come first, equal ones by id, a NaN before all, as in the greedy sampler.  Suppressed ids (-inf) have
    probability 0; an id outside the vocabulary has log probability -inf and rank V.  A row with a NaN or +inf, or of -inf
    alone, has no distribution: NaN log probabilities and entropy."""
    kind = logits.dtype
    index = logits.get_device()
    if index < 0 or logits.dim() != 2 or (kind is not _F32 and kind is not _BF16):
        _refuse('logits: [rows, V] fp32 or bf16 on a CUDA device')
    rows, V = logits.shape
    ld, one = logits.stride()
    if V < 1 or (one != 1 and V > 1):
        _refuse('logits: [rows, V] with unit inner stride, V at least 1')
    if tokens.dtype is not _I64 or tokens.get_device() != index or tokens.shape != (rows,) or not tokens.is_contiguous():
        _refuse('tokens: [rows] int64 on the logits\' device')
    if not 0 <= top <= 32 or top > V:
        _refuse(f'top: 0 to {min(32, V)}')
    if _current() != index:
        with torch.cuda.device(index):
            return token_scores(logits, tokens, top=top, temperature=temperature)
    kw = _AS_F32 if kind is _BF16 else _AS_IS
    out = TokenScores(logits.new_empty(rows, **kw), logits.new_empty(rows, **kw), tokens.new_empty(rows),
                      tokens.new_empty((rows, top)), logits.new_empty((rows, top), **kw))
    if rows == 0:
        return out
    logprob, entropy, rank, ids, logprobs = out
    rc = (_lib or _bind()).flashb_token_scores(
        logits.data_ptr(), kind is _BF16, ld if rows > 1 else V, rows, V, tokens.data_ptr(), temperature, top,
        logprob.data_ptr(), entropy.data_ptr(), rank.data_ptr(), ids.data_ptr(), logprobs.data_ptr(), _raw_stream(index))
    if rc:
        check(rc)
    return out
