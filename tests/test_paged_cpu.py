"""CPU checks of the paged cache and the token scores: the C ABI refuses bad descriptors and sizes before it touches a GPU."""
import ctypes
import math

import pytest
import torch

import paged_ref as ref
from flashb import _native, paged
from flashb._native import FB_ERR_ARG, FB_ERR_UNSUPPORTED, FbPagedCache

P = 1 << 20


def desc(pages=8, NKV=2, page=16, **kw):
    d = FbPagedCache(pages=pages, NKV=NKV, page=page, k=1 << 30, v=1 << 31)
    d.k_sb = d.v_sb = NKV * page * 128
    d.k_sh = d.v_sh = page * 128
    d.k_sl = d.v_sl = 128
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def append(d, table=P, tsb=4, rows=2, width=4, lengths=P, offsets=P, T=10, qkv=1 << 24, ld=1024 + 512, NH=8, qn=None, kn=None,
           turns=P, rot=128, q=1 << 26, st=1024, sh=128):
    return _native.lib().flashb_paged_append(ctypes.byref(d), table, tsb, rows, width, lengths, offsets, T, qkv, ld, NH, qn, kn,
                                             1e-6, turns, rot, 0, 1.0, None, q, st, sh, None)


def attend(d, table=P, tsb=4, rows=2, width=4, lengths=P, offsets=P, T=10, q=1 << 24, st=1024, sh=128, NH=8, sinks=0,
           scaling=1.0, ws=1 << 28, n=1 << 40, out=1 << 26, ost=1024, osh=128):
    return _native.lib().flashb_paged_attend(ctypes.byref(d), table, tsb, rows, width, lengths, offsets, T, q, st, sh, NH, 0,
                                             sinks, scaling, ws, n, out, ost, osh, None)


def decode(d, table=P, rows=500, width=400, lengths=P, q=1 << 24, st=1024, NH=8, sinks=0, scaling=1.0, ws=1 << 28, n=1 << 40,
           out=1 << 26):
    return _native.lib().flashb_paged_decode(ctypes.byref(d), table, 4, rows, width, lengths, q, st, 128, NH, 0, sinks, scaling,
                                             ws, n, out, None)


@pytest.mark.parametrize('bad', [dict(pages=0), dict(NKV=0), dict(page=0), dict(page=8), dict(page=24), dict(page=1 << 21),
                                 dict(k=None), dict(v=None), dict(k=(1 << 30) + 8), dict(k_sl=64), dict(v_sb=4),
                                 dict(k_sh=-128)])
def test_bad_pools(bad):
    for f in (append, attend, decode):
        assert f(desc(**bad)) == FB_ERR_ARG and _native.last_error()


def test_bad_append_arguments():
    for kw in (dict(table=None), dict(lengths=None), dict(qkv=None), dict(q=None), dict(tsb=-1), dict(rows=0), dict(width=0),
               dict(T=0), dict(T=10, offsets=None), dict(NH=0), dict(ld=1024), dict(ld=1537), dict(qkv=(1 << 24) + 2),
               dict(q=(1 << 26) + 8), dict(st=0), dict(st=1020), dict(sh=-128), dict(rot=130), dict(rot=24), dict(rot=-16),
               dict(turns=None), dict(turns=P + 4), dict(qn=P), dict(kn=P), dict(qn=P + 2, kn=P), dict(width=1 << 27)):
        assert append(desc(), **kw) == FB_ERR_ARG, kw
    # what is written shares memory with what is read or written: q over the k heads, over half of itself, over the cache
    for kw in (dict(q=(1 << 24) + 256), dict(q=1 << 24, st=1536 * 2, T=2), dict(st=1024, sh=64), dict(st=512),
               dict(q=1 << 30), dict(q=(1 << 31) + 4096), dict(qkv=1 << 30)):
        assert append(desc(), **kw) == FB_ERR_ARG, kw
    assert append(desc(k_sh=0)) == FB_ERR_ARG and append(desc(v=(1 << 30) + 4096)) == FB_ERR_ARG


def test_bad_attend_arguments():
    for kw in (dict(table=None), dict(lengths=None), dict(offsets=None), dict(q=None), dict(out=None), dict(tsb=-1),
               dict(rows=0), dict(width=0), dict(T=0), dict(NH=7), dict(NH=1), dict(sinks=-1), dict(scaling=0.0),
               dict(scaling=-1.0), dict(scaling=float('nan')), dict(q=(1 << 24) + 8), dict(st=1028), dict(st=0),
               dict(out=(1 << 26) + 8), dict(ost=0), dict(osh=-128), dict(ost=512), dict(width=100, ws=None),
               dict(width=100, ws=(1 << 28) + 8), dict(width=100, n=100), dict(T=1 << 30)):
        assert attend(desc(), **kw) == FB_ERR_ARG, kw
    assert attend(desc(), NH=6) == FB_ERR_UNSUPPORTED and 'group 3' in _native.last_error()
    assert attend(desc(k_sb=0)) == FB_ERR_ARG


def test_bad_decode_arguments():
    for kw in (dict(table=None), dict(lengths=None), dict(q=None), dict(out=None), dict(rows=0), dict(width=0), dict(NH=7),
               dict(sinks=-1), dict(scaling=0.0), dict(q=(1 << 24) + 8), dict(st=1028), dict(out=(1 << 26) + 4), dict(ws=None),
               dict(n=10), dict(width=1 << 27)):
        assert decode(desc(), **kw) == FB_ERR_ARG, kw
    assert decode(desc(), NH=6) == FB_ERR_UNSUPPORTED


def test_bad_score_arguments():
    def scores(x=P, bf16=0, ld=100, rows=3, V=100, tokens=P, temperature=1.0, top=5, out=P, ids=P):
        return _native.lib().flashb_token_scores(x, bf16, ld, rows, V, tokens, temperature, top, out, out, out, ids, ids, None)
    for kw in (dict(x=None), dict(tokens=None), dict(out=None), dict(ids=None), dict(rows=0), dict(V=0), dict(ld=99),
               dict(top=-1), dict(top=33), dict(V=4, top=5), dict(temperature=0.0), dict(temperature=-1.0),
               dict(temperature=float('inf')), dict(temperature=float('nan')), dict(temperature=1e-39), dict(x=P + 2),
               dict(x=P + 1, bf16=1), dict(V=(1 << 24) + 1, ld=1 << 25)):
        assert scores(**kw) == FB_ERR_ARG, kw


def test_workspace_sizes():
    L = _native.lib()
    d = ctypes.byref(desc(page=64))
    attend_ws = lambda rows, width, T, NH=8, w=0, s=0: L.flashb_paged_attend_ws_floats(d, rows, width, T, NH, w, s)  # noqa: E731
    assert attend_ws(2, 4, 400) == 0 and attend_ws(2, 100, 400) > 0                     # few keys: nothing to cut
    assert attend_ws(1, 1000, 100) >= attend_ws(1, 1000, 100, w=64)                     # a short window needs no pieces
    assert attend_ws(0, 4, 10) == -1 and attend_ws(1, 4, 0) == -1 and attend_ws(1, 4, 10, NH=6) == -1
    assert L.flashb_paged_decode_ws_floats(d, 2, 4, 8, 0, 0) == 0
    assert L.flashb_paged_decode_ws_floats(d, 500, 400, 8, 0, 0) > 0
    assert L.flashb_paged_decode_ws_floats(d, 500, 0, 8, 0, 0) == -1


def test_python_refuses():
    k = torch.zeros(4, 1, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(_native.FlashbError):
        paged.PagedCache(k, k)                                                          # on the CPU
    from flashb.sampling import token_scores
    with pytest.raises(_native.FlashbError):
        token_scores(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    for kw in (dict(dim=0), dict(dim=136), dict(dim=24), dict(layout='other'), dict(base=1.0), dict(scaling=dict(kind='x')),
               dict(scaling=dict(kind='linear', factor=0.0)), dict(scaling=dict(kind='yarn', factor=2.0)),
               dict(scaling=dict(kind='linear', factor=2.0, original=4)), dict(freq=[1.0] * 3),
               dict(freq=[float('nan')] * 64), dict(freq=[1.0] * 64, scaling=dict(kind='linear', factor=2.0)),
               dict(amplitude=float('inf'))):
        with pytest.raises(_native.FlashbError):
            paged.Rotary(device='cpu', **kw)


def test_scaled_frequencies():
    """The interpolations by hand, at the pairs where they begin and end."""
    plain, amp = paged.Rotary._freq(128, 1e4, {})
    assert amp == 1.0 and plain[0] == 1.0 and math.isclose(plain[63], 1e4 ** (-126 / 128))
    lin, _ = paged.Rotary._freq(128, 1e4, dict(kind='linear', factor=4.0))
    assert torch.allclose(lin, plain / 4, rtol=1e-15)
    ntk, _ = paged.Rotary._freq(128, 1e4, dict(kind='ntk', factor=8.0))
    assert ntk[0] == 1.0 and math.isclose(ntk[63], plain[63] / 8, rel_tol=1e-12)
    yarn, amp = paged.Rotary._freq(128, 1e4, dict(kind='yarn', factor=16.0, original=4096))
    turns = 4096 * plain / (2 * math.pi)
    assert math.isclose(amp, 0.1 * math.log(16) + 1)
    keep, cut = turns > 35, turns < 0.9                    # a pair or two beside the ramp's rounded ends
    assert torch.equal(yarn[keep], plain[keep]) and torch.allclose(yarn[cut], plain[cut] / 16, rtol=1e-15)
    mid = ~keep & ~cut
    assert mid.any() and torch.all((yarn[mid] <= plain[mid]) & (yarn[mid] >= plain[mid] / 16))


def test_reference_angle_of_far_positions():
    assert ref.angle(1, 1.0) == 1.0
    assert math.isclose(ref.angle(7, 1.0), 7 - 2 * math.pi)
    assert math.isclose(ref.angle(10 ** 15, 0.5), float((10 ** 15 // 2) % ref.TURN))
