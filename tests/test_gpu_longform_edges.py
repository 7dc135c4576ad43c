"""GPU tests of the long-speech operators at their edges: padding beside odd values, scores and values at the ends of
their range, long rows, many rows, captured calls."""
import pytest
import torch

import longform_ref as ref
from test_gpu_longform import HEADS, SC, dev, four, lf, randn, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('heads', HEADS)
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_prefill_padding_is_zero_beside_a_visible_odd_value(heads, bad):
    """Tokens before their row's start see nothing and give 0, also where later tokens of the same tile see such a V."""
    NH, NKV = heads
    L, past, starts = 40, 6, [11, 0, 30]                # tokens at slots 6 .. 45; rows with 5, 0 and 24 padded ones
    q, k, v = randn((3, NH, L, 128), 1), randn((3, NKV, past + L, 128), 2), randn((3, NKV, past + L, 128), 3)
    for j in (12, 31, past + L - 1):
        vv = v.clone()
        vv[:, :, j] = bad
        got = lf().prefill(q.cuda(), k.cuda(), vv.cuda(), starts=torch.tensor(starts, device='cuda')).cpu()
        for b, st in enumerate(starts):
            pad = max(0, st - past)
            assert (got[b, :pad] == 0).all()
            sees = torch.arange(past, past + L) >= max(j, st) if j >= st else torch.zeros(L, dtype=torch.bool)
            assert torch.isfinite(got[b, ~sees]).all() and not torch.isfinite(got[b, sees]).any()
