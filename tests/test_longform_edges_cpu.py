"""CPU checks of the long-speech entry points at their edges: refusals, the device of a call, the rotary table."""
import types

import pytest
import torch


def test_rotary_table_is_the_graphs_own():
    """From the graph's rotary module where it has one (an official graph), else from its configuration."""
    from flashb.engine import BackboneConfig, rope_table
    from flashb.long_speech import rotary_table
    cos, sin = rope_table(1e6, 128, 50, 'cpu')

    class Rotary:
        def __call__(self, x, pos):
            assert x.dtype == torch.bfloat16 and pos.tolist() == [list(range(50))]
            return cos.float()[None], sin.float()[None]
    official = types.SimpleNamespace(model=types.SimpleNamespace(rotary_emb=Rotary()))
    for g in (official, types.SimpleNamespace(cfg=BackboneConfig())):
        c, s = rotary_table(g, 50, 'cpu')
        assert torch.equal(c, cos) and torch.equal(s, sin) and c.dtype == torch.bfloat16 and c.is_contiguous()


class OnDevice1(torch.Tensor):
    """A CPU tensor that says it is on cuda:1."""
    is_cuda = True

    def get_device(self):
        return 1


@pytest.mark.parametrize('current', [0, 1])
def test_calls_run_on_the_device_of_their_tensors(monkeypatch, current):
    """Whichever device is current: the library is entered with the cache's, and the current one is as before after it."""
    from flashb import longform as lf
    at, calls = [current], []

    class on:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, at[0] = at[0], self.index

        def __exit__(self, *exc):
            at[0] = self.before

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, at[0], a[-1])) or 0
    monkeypatch.setattr(lf, '_current', lambda: at[0])
    monkeypatch.setattr(lf, '_on', on)
    monkeypatch.setattr(lf, '_lib', Lib())
    monkeypatch.setattr(lf, '_raw_stream', lambda index: f'stream of {index}')
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt).as_subclass(OnDevice1)  # noqa: E731
    q, k, n = z(2, 4, 1, 128), z(2, 2, 16, 128), z(2, dt=torch.int64)
    u8 = lambda w: z(2, 2, 16, w, dt=torch.uint8)  # noqa: E731
    cache, c4 = lf.KVCache(k, z(2, 2, 16, 128)), lf.KV4Cache(u8(64), u8(8), u8(64), u8(8))
    lf.decode(q, cache, n, acc=z(2, 2, 16, dt=torch.float32))
    lf.prefill(q, k, k)
    c4.store(k, k, z(16, dt=torch.int64))
    c4.read(z(16, dt=torch.int64))
    lf.evict(cache, z(2, 2, 16, dt=torch.float32), n, 4, into=lf.KVCache(z(2, 2, 4, 128), z(2, 2, 4, 128)))
    assert [c[0] for c in calls] == ['flashb_long_decode_ws_floats', 'flashb_long_decode', 'flashb_long_prefill',
                                     'flashb_kv4_store', 'flashb_kv4_read', 'flashb_kv_evict']
    assert all(c[1] == 1 for c in calls) and all(c[2] == 'stream of 1' for c in calls[1:])
    assert at[0] == current


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('B', [2, 500])                            # a cluster a row, the shared list
def test_decode_output_off_its_alignment_is_refused(bits, B):
    from flashb import _native
    from test_longform_cpu import decode, desc
    for off in (2, 4, 6):
        assert decode(desc(bits=bits, B=B), out=(1 << 27) + off) == _native.FB_ERR_ARG
        assert '8-byte' in _native.last_error()


@pytest.mark.parametrize('bad', [dict(keep=20, sinks=4, recent=17), dict(keep=20, sinks=4, recent=21), dict(keep=20, sinks=-1),
                                 dict(keep=20, recent=-1), dict(keep=3, sinks=4), dict(sinks=-1), dict(window=0),
                                 dict(keep=0), dict(keep=32)])
def test_long_speech_refuses_settings_that_cannot_be_kept(bad, monkeypatch):
    """When it is made, not when the cache is full for the first time; nothing is allocated before."""
    from flashb import long_speech
    from flashb._native import FB_ERR_ARG, FlashbError
    monkeypatch.setattr(long_speech.bb, '_prep', lambda g: dict(layers=None, B=2))
    with pytest.raises(FlashbError) as e:
        long_speech.LongSpeech(types.SimpleNamespace(), 32, **bad)
    assert e.value.rc == FB_ERR_ARG


def evict(a, b, keep=8, acc=1 << 20, acc_out=1 << 21, acc_n=8):
    import ctypes

    from flashb import _native
    return _native.lib().flashb_kv_evict(ctypes.byref(a), acc, 128, 64, 1 << 24, None, keep, 0, 0, ctypes.byref(b), acc_out, 128,
                                         64, acc_n, 1 << 25, 1 << 26, None)


def test_evict_refuses_memory_in_common():
    """Views of one buffer at any offset, not the same tensors alone: reads and writes would race."""
    from flashb import _native
    from test_longform_cpu import desc
    row = 2 * 128
    far = dict(k=1 << 30, v=1 << 31)
    src = desc()                                           # 2 rows, 2 heads, 64 slots: 64 KB at 1 MB and at 2 MB
    for k in ((1 << 20) + row, (1 << 20) + 200 * row, (1 << 20) + 255 * row, (1 << 20) - 255 * row, 1 << 21, (1 << 21) - row):
        for name in ('k', 'v'):
            assert evict(src, desc(**{**far, name: k})) == _native.FB_ERR_ARG and 'share memory' in _native.last_error()
    # other slots a head, so other strides: a slot of the one lies in the other
    assert evict(src, desc(S=48, **{**far, 'k': (1 << 20) + 100 * row})) == _native.FB_ERR_ARG
    # positions side by side: the halves of rows of 512 bytes share nothing, the same half does
    wide = dict(k_sb=65536, k_sh=32768, k_sp=256, v_sb=65536, v_sh=32768, v_sp=256)
    assert evict(desc(**wide), desc(**{**wide, **far, 'k': (1 << 20) + 512 * 9})) == _native.FB_ERR_ARG
    four = desc(bits=4)
    far4 = dict(k=1 << 30, v=1 << 31, ks=1 << 32, vs=1 << 33)
    for name, at in (('k', (1 << 20) + 64), ('ks', (1 << 22) + 8), ('vs', (1 << 22) + 8), ('ks', (1 << 20) + 64)):
        assert evict(four, desc(bits=4, **{**far4, name: at})) == _native.FB_ERR_ARG, name
    for at in ((1 << 20) + 4, (1 << 20) - 4, (1 << 20) + 4 * 255, 1 << 20):
        assert evict(src, desc(**far), acc_out=at) == _native.FB_ERR_ARG and 'acc' in _native.last_error()


@pytest.mark.parametrize('bits', [16, 4])
def test_decode_refuses_weights_that_overlap_their_sums(bits):
    """In place or apart; not shifted, and not in place with other strides."""
    import ctypes

    from flashb import _native
    from test_longform_cpu import desc
    d, acc = desc(bits=bits), 1 << 28                         # 2 rows, 2 heads, 64 slots

    def run(out, sb, sh):
        return _native.lib().flashb_long_decode(ctypes.byref(d), 1 << 24, 1024, 128, 8, 1 << 25, None, 0, 0, 1.0, acc, 128, 64,
                                                out, sb, sh, 1.0, None, 0, 1 << 27, None)
    for out, sb, sh in ((acc + 4, 128, 64), (acc - 4, 128, 64), (acc + 4 * 64, 128, 64), (acc, 256, 64), (acc, 64, 128),
                        (acc - 4 * 63, 64, 64)):
        assert run(out, sb, sh) == _native.FB_ERR_ARG and 'acc' in _native.last_error()


def test_outputs_that_overlap_themselves_are_refused():
    """Expanded tensors (a stride of 0) and keys that are the values: rows of such an output would race."""
    import ctypes

    from flashb import _native
    from test_longform_cpu import desc
    L, p = _native.lib(), 1 << 24
    far = dict(k=1 << 30, v=1 << 31)
    far4 = dict(bits=4, ks=1 << 32, vs=1 << 33, **far)

    def store(d):
        return L.flashb_kv4_store(ctypes.byref(d), p, 1024, 512, 128, p, 1024, 512, 128, p, 0, 4, None)
    for bad in (dict(k_sb=0), dict(v_sh=0), dict(ks_sb=0), dict(vs_sh=0), dict(k_sb=64 * 32), dict(v=1 << 30), dict(vs=1 << 32),
                dict(k_sp=128)):
        assert store(desc(**{**far4, **bad})) == _native.FB_ERR_ARG and 'share memory' in _native.last_error(), bad
        assert evict(desc(bits=4), desc(**{**far4, **bad})) == _native.FB_ERR_ARG, bad
    for bad in (dict(k_sb=0), dict(v_sh=0), dict(v=1 << 30), dict(k=(1 << 31) + 256 * 255), dict(k_sb=128 * 64)):
        assert evict(desc(), desc(**{**far, **bad})) == _native.FB_ERR_ARG and 'share memory' in _native.last_error(), bad
    acc = 1 << 28

    def sums(sb, sh, out=acc):
        return L.flashb_long_decode(ctypes.byref(desc()), p, 1024, 128, 8, p, None, 0, 0, 1.0, acc, sb, sh, out, sb, sh, 1.0,
                                    None, 0, 1 << 27, None)
    for sb, sh in ((0, 64), (128, 0), (64, 64), (128, 63)):
        for out in (acc, 1 << 29):
            assert sums(sb, sh, out) == _native.FB_ERR_ARG and 'acc_out' in _native.last_error()

    def prefill(sb, sl, sh):
        return L.flashb_long_prefill(p, 16 * 1024, 2048, 128, p, 16 * 256, 2048, 128, p, 16 * 256, 2048, 128, 2, 8, 2, 16, 16, 0,
                                     None, 0, 0, 1.0, 1 << 27, sb, sl, sh, None)
    for st in ((16 * 1024, 128, 128), (16 * 1024, 64, 2048), (8 * 1024, 1024, 128)):
        assert prefill(*st) == _native.FB_ERR_ARG and 'share memory' in _native.last_error()


def test_tensors_of_another_rank_are_refused(monkeypatch):
    """As bad shapes are, with FlashbError."""
    from flashb import longform as lf
    from flashb._native import FB_ERR_ARG, FlashbError
    monkeypatch.setattr(lf, '_current', lambda: 1)
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt).as_subclass(OnDevice1)  # noqa: E731
    u8 = lambda w: z(2, 2, 16, w, dt=torch.uint8)  # noqa: E731
    k, c4, n = z(2, 2, 16, 128), lf.KV4Cache(u8(64), u8(8), u8(64), u8(8)), z(2, dt=torch.int64)
    cache, acc = lf.KVCache(k, k), z(2, 2, 16, dt=torch.float32)
    none = z((), dt=torch.int64)
    for f in (lambda: lf.prefill(z(16, 128), k, k), lambda: lf.prefill(z(()), k, k), lambda: lf.prefill(z(1, 2, 2, 16, 128), k, k),
              lambda: lf.prefill(z(2, 4, 16, 128), z(16, 128), z(16, 128)), lambda: lf.decode(z(2, 512), cache, n),
              lambda: lf.decode(z(2, 4, 1, 128), cache, none), lambda: lf.decode(z(2, 4, 1, 128), cache, n, acc=none),
              lambda: c4.store(k, k, none), lambda: c4.read(none), lambda: c4.store(z(16, 128), z(16, 128), z(16, dt=torch.int64)),
              lambda: lf.evict(cache, none, n, 4, into=cache), lambda: lf.KVCache(z(16, 128), z(16, 128)),
              lambda: lf.KV4Cache(none, none, none, none)):
        with pytest.raises(FlashbError) as e:
            f()
        assert e.value.rc == FB_ERR_ARG
