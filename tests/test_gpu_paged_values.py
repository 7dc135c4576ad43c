"""Infinities in the visible slots of a paged cache: what the definition says of each dim, from every form of the attention."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BF, cuda, make, paged

pytestmark = pytest.mark.gpu
INF = float('inf')


def check_infinities(s, edits, window=None, sinks=0):
    """edits: (row, slot, KV head, dim, value) of V."""
    m = paged()
    page = s['keys'].shape[2]
    for b, slot, h, d, val in edits:
        s['values'][int(s['table'][b, slot // page]), h, slot % page, d] = val
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    got = m.attend(s['q'].cuda(), c, cuda(s['table']), cuda(s['lengths']), offsets=cuda(s['offsets']), window=window,
                   sinks=sinks).cpu().double()
    want, size = ref.attend(s['q'], s['keys'], s['values'], s['table'], s['lengths'], s['offsets'], window, sinks)
    assert (want == INF).any() and (want == -INF).any() and want.isnan().any()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got == INF, want == INF) and torch.equal(got == -INF, want == -INF)
    fin = torch.isfinite(want)
    # as for finite values: a weight rounded to bf16, scores in fp32, the output's own rounding
    assert torch.all((got - want).abs()[fin] <= ((BF + 2.0 ** -11) * size + BF * want.abs())[fin])


def edits(rows):
    """An infinity each way in dims of their own, both in a third, in the first and in later slots."""
    out = []
    for b, slots in rows:
        for i, j in enumerate(slots):
            out += [(b, j, i % 2, 3 + i, INF), (b, j, 1, 40 + i, -INF), (b, j, 0, 127, INF if i else -INF)]
    return out


@pytest.mark.parametrize('NH,NKV', [(16, 4), (8, 8), (16, 2), (4, 2)])
@pytest.mark.parametrize('page', [16, 64])
def test_single_tokens_of_few_rows(NH, NKV, page):
    s = make([1, 1, 1], [4, 100, 300], NH, NKV, page, single=True)
    check_infinities(s, edits([(0, (0, 3)), (1, (50, 100)), (2, (0, 299))]))


@pytest.mark.parametrize('NH,NKV', [(16, 4), (16, 2)])
def test_single_tokens_of_few_rows_over_a_window(NH, NKV):
    s = make([1, 1, 1], [40, 100, 300], NH, NKV, 32, single=True)
    check_infinities(s, edits([(0, (0, 37)), (1, (2, 100)), (2, (1, 290))]), 33, 3)


@pytest.mark.parametrize('NH,NKV', [(16, 4), (2, 2)])
def test_single_tokens_of_many_rows(NH, NKV):
    g = torch.Generator().manual_seed(NH)
    pasts = torch.randint(5, 900, (130,), generator=g).tolist()
    s = make([1] * 130, pasts, NH, NKV, 64, single=True)
    check_infinities(s, edits([(0, (0, 3)), (64, (1, pasts[64])), (129, (2, pasts[129] - 1))]))


def test_single_tokens_of_long_rows():
    s = make([1, 1, 1], [9000, 5000, 7000], 8, 2, 64, single=True)
    check_infinities(s, edits([(0, (0, 8999)), (2, (17, 5001))]))


def test_runs():
    s = make([20, 3, 1], [100, 64, 30], 8, 2, 16)
    check_infinities(s, edits([(0, (0, 99)), (1, (50, 64)), (2, (0, 29))]))
    s = make([20, 3], [2000, 1500], 8, 2, 16)
    check_infinities(s, edits([(0, (0, 1999)), (1, (700, 1499))]))


@pytest.mark.parametrize('single', [True, False])
def test_a_row_gone_bad_does_not_hold_up_the_step(single):
    """A long row of NaN among others: NaN for itself, and the step's time (a key at a time it was 30 times and more)."""
    m = paged()
    rows, page, n = 16, 64, 4096
    g = torch.Generator(device='cuda').manual_seed(1)
    k, v = (torch.randn(rows * n // page, 4, page, 128, generator=g, device='cuda').bfloat16() for _ in range(2))
    table = torch.arange(rows * n // page, device='cuda', dtype=torch.int32).view(rows, -1)
    lengths = torch.full((rows,), n, device='cuda')
    offsets = None if single else torch.arange(rows + 1, device='cuda')
    q = torch.randn(rows, 16, 128, generator=g, device='cuda').bfloat16()
    c = m.PagedCache(k, v)

    def took():
        best = float('inf')
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                out = m.attend(q, c, table, lengths, offsets=offsets)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return out, best
    good, before = took()
    k[table[3].long()] = float('nan')
    bad, after = took()
    others = [r for r in range(rows) if r != 3]
    assert torch.equal(bad[others], good[others]) and bad[3].isnan().all()
    assert after < 8 * before, (before, after)
