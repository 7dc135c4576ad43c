"""The backbone over pages where steps are unusual: rows that have nothing this time, inputs that are refused."""
import pytest
import torch

from test_gpu_paged_speech import _graph, _speech, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('window', [None, 24])
def test_a_frame_beside_idle_rows(window):
    """Frames of some rows, others without a token: the bits of a step of those rows alone."""
    cfg, g = _graph(layers=2)
    wide = _speech(g, rows=5, max_slots=320, window=window)
    narrow = _speech(g, rows=2, max_slots=320, window=window)
    x = _x(cfg, 90, 3)
    assert torch.equal(wide.extend(x[:80], [0, 50, 0, 30, 0]), narrow.extend(x[:80], [50, 30]))
    for i in range(80, 88, 2):
        a, b = wide.extend(x[i:i + 2], [0, 1, 0, 1, 0]), narrow.extend(x[i:i + 2], [1, 1])
        assert torch.equal(a, b)
    assert wide.used == [0, 54, 0, 34, 0] and wide.lengths.tolist() == wide.used
    # all idle but one, and a row that begins
    a = wide.extend(x[88:90], [1, 0, 0, 1, 0])
    assert a.shape == (2, cfg.hidden) and wide.used == [1, 54, 0, 35, 0]
    assert torch.equal(wide.extend(x[:1], [0, 0, 0, 0, 1]), _speech(g, rows=1, max_slots=320, window=window).extend(x[:1], [1]))


def test_refused_inputs_change_nothing():
    from flashb._native import FB_ERR_ARG, FlashbError
    cfg, g = _graph(layers=1)
    s = _speech(g, max_slots=64)
    x = _x(cfg, 20, 1)
    s.extend(x[:5], [5, 0])
    before = list(s.free), list(s.used), s.lengths.clone(), s.table.clone()
    for bad in (x.float(), x.cpu(), x[:, :-8], x.half(), x[None]):
        with pytest.raises(FlashbError) as e:
            s.extend(bad, [18, 2])
        assert e.value.rc == FB_ERR_ARG
        assert (s.free, s.used) == before[:2] and torch.equal(s.lengths, before[2]) and torch.equal(s.table, before[3])
    assert s.extend(x[:18], [16, 2]).shape == (18, cfg.hidden) and s.used == [21, 2]


def test_refused_frames():
    from flashb._native import FB_ERR_ARG, FlashbError
    cfg, g = _graph(layers=1)
    s = _speech(g)
    ids = torch.randint(0, cfg.vocab, (3, cfg.codebooks)).cuda()
    for bad in (ids.cpu(), ids.int(), ids[:, :-1], ids[:, :1].expand(-1, cfg.codebooks + 1), ids[0], ids[None]):
        with pytest.raises(FlashbError) as e:
            s.embed(bad)
        assert e.value.rc == FB_ERR_ARG
    want = s.embed(ids)
    wide = torch.zeros(3, 2 * cfg.codebooks, dtype=torch.int64, device='cuda')
    wide[:, ::2] = ids
    assert want.shape == (3, cfg.hidden) and torch.equal(s.embed(wide[:, ::2]), want)
    assert s.embed(ids[:0]).shape == (0, cfg.hidden)


def test_rows_end_at_their_last_slot():
    """``max_slots`` that is no whole number of pages is the limit all the same."""
    from flashb._native import FB_ERR_ARG, FB_ERR_STATE, FlashbError
    from flashb.paged_speech import PagedSpeech
    cfg, g = _graph(layers=1)
    s = _speech(g, max_slots=40)
    x = _x(cfg, 50, 1)
    s.extend(x[:39], [39, 0])
    for counts in ([2, 0], [0, 41]):
        with pytest.raises(FlashbError) as e:
            s.extend(x[:sum(counts)], counts)
        assert e.value.rc == FB_ERR_STATE and s.used == [39, 0] and s.lengths.tolist() == [39, 0]
    s.extend(x[:41], [1, 40])
    assert s.used == [40, 40]
    for n in (0, -16):
        with pytest.raises(FlashbError) as e:
            PagedSpeech(g, 2, 40, max_slots=n)
        assert e.value.rc == FB_ERR_ARG
