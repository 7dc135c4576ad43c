"""CPU checks of the long-speech entry points: the C ABI refuses bad descriptors and sizes before it touches a GPU."""
import ctypes

import pytest
import torch

import longform_ref as ref
from flashb import _native, longform
from flashb._native import FB_ERR_ARG, FB_ERR_UNSUPPORTED, FbKVCache


def desc(bits=16, B=2, NKV=2, S=64, **kw):
    row = 128 if bits == 16 else 64
    d = FbKVCache(bits=bits, B=B, NKV=NKV, S=S, k=1 << 20, v=1 << 21, k_scale=1.0, v_scale=1.0)
    d.k_sb = d.v_sb = NKV * S * row
    d.k_sh = d.v_sh = S * row
    d.k_sp = d.v_sp = row
    if bits == 4:
        d.ks, d.vs = 1 << 22, 1 << 23
        d.ks_sb = d.vs_sb = NKV * S * 8
        d.ks_sh = d.vs_sh = S * 8
        d.ks_sp = d.vs_sp = 8
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def decode(d, NH=8, q=1 << 24, lengths=1 << 25, window=0, sinks=0, ws=1 << 26, n=1 << 40, out=1 << 27, acc=None,
           acc_out=None, q_sb=1024):
    return _native.lib().flashb_long_decode(ctypes.byref(d), q, q_sb, 128, NH, lengths, None, window, sinks, 1.0, acc, 0,
                                            0, acc_out, 0, 0, 1.0, ws, n, out, None)


@pytest.mark.parametrize('bad', [dict(bits=8), dict(B=0), dict(NKV=0), dict(S=0), dict(k=None), dict(v=None),
                                 dict(k=(1 << 20) + 8), dict(k_sp=64), dict(k_sh=-128), dict(v_sb=4)])
def test_bad_bf16_descriptors(bad):
    assert decode(desc(**bad)) == FB_ERR_ARG and _native.last_error()


@pytest.mark.parametrize('bad', [dict(ks=None), dict(vs=(1 << 23) + 4), dict(ks_sp=4), dict(vs_sh=12), dict(k_sp=32),
                                 dict(k_scale=3.0), dict(v_scale=0.0), dict(v_scale=-1.0), dict(k_scale=float('nan')),
                                 dict(k_scale=float('inf')), dict(k_scale=2.0 ** 100)])
def test_bad_4bit_descriptors(bad):
    assert decode(desc(bits=4, **bad)) == FB_ERR_ARG and _native.last_error()


def test_bad_decode_arguments():
    d = desc()
    for kw in (dict(q=None), dict(lengths=None), dict(ws=None), dict(out=None), dict(q=(1 << 24) + 2), dict(q_sb=12),
               dict(acc=1 << 20), dict(acc_out=1 << 20), dict(NH=7), dict(NH=1), dict(sinks=-1)):
        assert decode(desc(B=500), **kw) == FB_ERR_ARG, kw
    assert decode(desc(B=500), n=10) == FB_ERR_ARG and 'workspace' in _native.last_error()
    assert decode(d, NH=6) == FB_ERR_UNSUPPORTED and 'group 3' in _native.last_error()
    assert decode(desc(B=1 << 29)) == FB_ERR_ARG                                       # more chunks than 32 bits hold


def test_workspace_sizes():
    L = _native.lib()
    ws = lambda d, NH, w, s, sc: L.flashb_long_decode_ws_floats(ctypes.byref(d), NH, w, s, sc)  # noqa: E731
    assert ws(desc(), 8, 0, 0, 0) == 0 and ws(desc(), 8, 0, 0, 1) == 0                 # few rows need none
    many = desc(B=500, S=4096)
    assert ws(many, 8, 0, 0, 0) > 0
    assert ws(many, 8, 0, 0, 1) - ws(many, 8, 0, 0, 0) == 500 * 2 * 4096 * 4           # the scores
    assert ws(many, 8, 100, 28, 1) - ws(many, 8, 100, 28, 0) == 500 * 2 * 128 * 4
    assert ws(desc(), 6, 0, 0, 0) == -1


def test_bad_prefill_store_and_evict_arguments():
    L = _native.lib()
    p = 1 << 20

    def prefill(NH=8, NKV=2, Lq=16, S=64, q_start=0, sinks=0, q=p, sl=128):
        return L.flashb_long_prefill(q, NH * Lq * 128, Lq * 128, sl, p, NKV * S * 128, S * 128, 128, p, NKV * S * 128,
                                     S * 128, 128, 2, NH, NKV, Lq, S, q_start, None, 8, sinks, 1.0, p, NH * Lq * 128,
                                     NH * 128, 128, None)
    for kw in (dict(q=None), dict(q=p + 2), dict(sl=4), dict(Lq=0), dict(q_start=49), dict(q_start=-1), dict(sinks=-1),
               dict(NH=7)):
        assert prefill(**kw) == FB_ERR_ARG, kw
    assert prefill(NH=6) == FB_ERR_UNSUPPORTED

    def store(d, k=p, slots=p, n=4, st=128):
        return L.flashb_kv4_store(ctypes.byref(d), k, 1024, st, 128, p, 1024, 512, 128, slots, 0, n, None)
    assert store(desc()) == FB_ERR_ARG and '16 bits' in _native.last_error()
    for kw in (dict(k=None), dict(k=p + 8), dict(slots=None), dict(n=0), dict(st=4)):
        assert store(desc(bits=4), **kw) == FB_ERR_ARG, kw
    assert L.flashb_kv4_read(ctypes.byref(desc(bits=4)), p, 0, 4, p + 8, p, None) == FB_ERR_ARG

    def evict(a, b, keep=8, sinks=0, recent=0, acc=p, acc_n=8, acc_out=2 * p, lengths_out=2 * p):
        return L.flashb_kv_evict(ctypes.byref(a), acc, 128, 64, p, None, keep, sinks, recent, ctypes.byref(b), acc_out, 128, 64,
                                 acc_n, p, lengths_out, None)
    other = dict(k=1 << 30, v=1 << 31)
    for a, b, kw in ((desc(), desc(), {}), (desc(), desc(bits=4, **other), {}), (desc(), desc(B=1, **other), {}),
                     (desc(), desc(**other), dict(keep=0)), (desc(), desc(**other), dict(keep=65)),
                     (desc(), desc(**other), dict(sinks=5, recent=4)), (desc(), desc(**other), dict(sinks=-1)),
                     (desc(), desc(**other), dict(acc=None)), (desc(), desc(**other), dict(acc_n=7)),
                     (desc(), desc(**other), dict(acc_out=p)), (desc(), desc(**other), dict(lengths_out=p)),
                     (desc(bits=4), desc(bits=4, k_scale=2.0, **other), {})):
        assert evict(a, b, **kw) == FB_ERR_ARG, kw


def test_python_refuses_cpu_tensors():
    k = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(_native.FlashbError):
        longform.KVCache(k, k)
    with pytest.raises(_native.FlashbError):
        longform.prefill(k, k, k)
    with pytest.raises(_native.FlashbError):
        longform.KV4Cache(*(torch.zeros(1, 1, 4, w, dtype=torch.uint8) for w in (64, 8, 64, 8)))


def test_reference_quantiser_by_hand():
    """The reference itself: ties, saturation and flushing of the 4-bit form."""
    x = torch.zeros(8, 16, dtype=torch.bfloat16)
    x[0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x[1] = -3 * x[0]
    x[2, 0] = 1e5
    x[3, 0] = 0.003                                             # / 6 is a quarter of the smallest scale: 0
    x[4, 0] = 2.0 ** -7                                         # / 6 rounds to the smallest scale, 2^-9
    x[5, 1] = float('nan')
    y = ref.quantise(x.repeat(1, 8))[:, :16]
    assert y[0, :8].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    assert torch.equal(y[1], -3 * y[0])
    assert y[2, 0] == 2688.0 and y[3].abs().sum() == 0 and y[4, 0] == 4 * 2.0 ** -9
    assert torch.isnan(y[5]).all()
