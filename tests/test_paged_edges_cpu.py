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


def test_scalings_that_leave_fp32_are_refused():
    """scaling x log2(e) is what the kernels multiply by: infinite, it would make NaN of a score of 0."""
    from test_paged_cpu import attend, decode, desc
    for scaling in (2.4e38, 3.3e38, 3.4028234e38):
        assert attend(desc(), scaling=scaling) == FB_ERR_ARG and decode(desc(), scaling=scaling) == FB_ERR_ARG
