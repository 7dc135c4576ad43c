"""The two places that cut a step's rows into pieces -- every CTA for up to 32 rows, a plan kernel for more -- cut alike."""
import pytest
import torch

from test_gpu_paged import cuda, make, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('NH,NKV', [(8, 2), (16, 4), (4, 4), (16, 2)])
@pytest.mark.parametrize('window,sinks', [(None, 0), (1200, 20)])
def test_an_idle_row_more_changes_no_bit(NH, NKV, window, sinks):
    """32 rows, then the same and an empty one: the same pieces, joined in the same order, give the same bits."""
    m = paged()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        counts = torch.randint(0, 4, (32,), generator=g).tolist()
        pasts = torch.randint(0, 100, (32,), generator=g).tolist()
        for b in range(seed, 32, (5, 9, 13, 31)[seed]):
            counts[b], pasts[b] = 1 + b % 7, 1300 + 97 * (b % 11)
        s = make(counts, pasts, NH, NKV, page=32, seed=seed)
        c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
        q, table, lengths, off = (cuda(s[k]) for k in ('q', 'table', 'lengths', 'offsets'))
        few = m.attend(q, c, table, lengths, offsets=off, window=window, sinks=sinks)
        more = m.attend(q, c, torch.cat((table, table[:1])), torch.cat((lengths, lengths[:1] * 0)),
                        offsets=torch.cat((off, off[-1:])), window=window, sinks=sinks)
        assert torch.equal(few, more)
