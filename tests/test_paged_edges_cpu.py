"""CPU checks of the paged cache's arguments where they can be taken for something else."""
import pytest
import torch

from flashb import paged
from flashb._native import FB_ERR_ARG, FlashbError


def test_a_scaling_without_its_kind_is_refused():
    """A factor that names no kind of scaling would leave the positions as they are."""
    for how in (dict(factor=4.0), dict(kind=None, factor=4.0), dict(original=4096), dict(type='yarn', factor=2.0)):
        with pytest.raises(FlashbError) as e:
            paged.Rotary._freq(128, 1e4, how)
        assert e.value.rc == FB_ERR_ARG
    plain, amp = paged.Rotary._freq(128, 1e4, {})
    same, amp2 = paged.Rotary._freq(128, 1e4, dict(kind=None))
    assert torch.equal(plain, same) and amp == amp2 == 1.0
