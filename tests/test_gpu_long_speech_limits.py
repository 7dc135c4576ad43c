"""GPU tests of the long-speech path at its limits: the end of the rotary table, prompts and settings that do not fit."""
import pytest
import torch

from test_gpu_long_speech import _ids, _pair

pytestmark = pytest.mark.gpu


def _prompt(cfg, B, L, seed=11):
    return torch.randn(B, L, cfg.hidden, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


@pytest.mark.parametrize('starts', [None, [3, 5], [4, 0]])
def test_reading_ends_with_the_rotary_table(starts):
    """Evictions keep a reading going; the last position of the table is its last frame, and the next one raises."""
    from flashb._native import FB_ERR_STATE, FlashbError
    cfg, _, g, s = _pair(2, 60, slots=32, keep=20, sinks=2)
    s.prefill(_prompt(cfg, 2, 20), None if starts is None else torch.tensor(starts, device='cuda'))
    left = 61 - 20 + (0 if starts is None else min(starts))       # positions 20 (less the padding) .. 60
    for ids in _ids(cfg, 2, left):
        g.input_ids_buf.copy_(ids)
        s.step()
    assert int(g.position_ids.max()) == 61
    lengths, logits = s.lengths.clone(), g.cfg_logits_buf.clone()
    for _ in range(2):
        with pytest.raises(FlashbError) as e:
            s.step()
        assert e.value.rc == FB_ERR_STATE
    assert torch.equal(s.lengths, lengths) and torch.equal(g.cfg_logits_buf, logits)


def test_prompt_past_the_rotary_table_raises():
    from flashb._native import FB_ERR_STATE, FlashbError
    cfg, _, g, s = _pair(2, 30, slots=64)
    with pytest.raises(FlashbError) as e:
        s.prefill(_prompt(cfg, 2, 40))
    assert e.value.rc == FB_ERR_STATE
    # 31 positions: a padded prompt of 34 fits where no row has more tokens than that
    assert torch.isfinite(s.prefill(_prompt(cfg, 2, 34), torch.tensor([3, 4], device='cuda'))).all()
    assert int(g.position_ids.max()) == 31


def test_a_table_of_its_own_instead_of_a_long_graph():
    """A graph of one slot and ``positions``: the same bits as on a graph whose own cache covers the whole reading."""
    from flashb._native import FlashbError
    from flashb.engine import BackboneConfig, SyntheticBackboneGraph
    from flashb.long_speech import LongSpeech
    cfg = BackboneConfig(layers=2)
    long = SyntheticBackboneGraph(cfg, batch_size=2, max_seq_len=119, seed=5)
    short = SyntheticBackboneGraph(cfg, batch_size=2, max_seq_len=1, weights_from=long)
    kw = dict(slots=48, keep=30, sinks=2, window=25, four_bits=True)
    a, b = LongSpeech(long, **kw), LongSpeech(short, positions=120, **kw)
    assert torch.equal(a.cos_tab, b.cos_tab) and torch.equal(a.sin_tab, b.sin_tab)
    x = _prompt(cfg, 2, 20)
    assert torch.equal(a.prefill(x), b.prefill(x))
    for ids in _ids(cfg, 2, 100):
        for g, s in ((long, a), (short, b)):
            g.input_ids_buf.copy_(ids)
            s.step()
        assert torch.equal(long.hidden_buf, short.hidden_buf)
    for s in (a, b):
        with pytest.raises(FlashbError):
            s.step()
    with pytest.raises(FlashbError):
        LongSpeech(short, positions=0, **kw)


def test_command_holds_no_cache_of_the_whole_reading(capsys):
    """What the command allocates does not grow with the frames, but for the rotary table; its logits are finite."""
    from flashb import long_speech
    args = ['--layers', '2', '--prompt', '20', '--slots', '32', '--keep', '24', '--window', '16']

    def peak(frames):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        long_speech.main(args + ['--frames', str(frames)])
        assert 'logits finite: True' in capsys.readouterr().out
        return torch.cuda.max_memory_allocated() - before
    peak(8)                                                        # what the first use of the libraries takes
    a, b = peak(8), peak(300)
    # the ids of the frames (2 rows of 16 int64) and cos and sin of 128 bf16; 4096 for the allocator's rounding
    assert b - a <= 292 * (2 * 16 * 8 + 2 * 128 * 2) + 4096


def test_starts_outside_the_prompt_are_clamped():
    """As the operators clamp them: positions neither begin past 0 nor lie below it."""
    cfg, g, g2, a = _pair(2, 40, slots=32)
    from flashb.long_speech import LongSpeech
    b = LongSpeech(g, 32)
    x = _prompt(cfg, 2, 20)
    assert torch.equal(a.prefill(x, torch.tensor([-3, 99], device='cuda')), b.prefill(x, torch.tensor([0, 20], device='cuda')))
    assert g.position_ids.tolist() == [[20], [0]]
    for ids in _ids(cfg, 2, 3):
        for h, s in ((g2, a), (g, b)):
            h.input_ids_buf.copy_(ids)
            s.step()
        assert torch.equal(g2.hidden_buf, g.hidden_buf) and torch.equal(g2.position_ids, g.position_ids)


@pytest.mark.parametrize('four_bits', [False, True])
def test_a_second_reading_is_like_a_first(four_bits):
    """After ``reset``, the same bits as from caches made anew, evictions among them."""
    from flashb._native import FlashbError
    from flashb.long_speech import LongSpeech
    kw = dict(slots=40, keep=24, sinks=2, window=30, four_bits=four_bits)
    cfg, g, g2, used = _pair(2, 70, **kw)
    used.prefill(_prompt(cfg, 2, 30, seed=12), torch.tensor([7, 0], device='cuda'))
    for ids in _ids(cfg, 2, 35):
        g2.input_ids_buf.copy_(ids)
        used.step()
    with pytest.raises(FlashbError):
        used.prefill(_prompt(cfg, 2, 20))
    used.reset()
    new = LongSpeech(g, **kw)
    x = _prompt(cfg, 2, 20)
    assert torch.equal(used.prefill(x), new.prefill(x))
    for ids in _ids(cfg, 2, 51):
        for h, s in ((g2, used), (g, new)):
            h.input_ids_buf.copy_(ids)
            s.step()
        assert torch.equal(g2.hidden_buf, g.hidden_buf) and torch.equal(g2.cfg_logits_buf, g.cfg_logits_buf)
    for s in (used, new):                                          # the table's end counts from the new beginning
        with pytest.raises(FlashbError):
            s.step()
