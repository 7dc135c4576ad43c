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
