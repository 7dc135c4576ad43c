"""The paged cache on the GPU where it can go wrong: many rows, large pages, every launch of a step captured, two calls at
once, values that are not finite beside rotated dims, calls that are refused."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BF, D, check_append, check_attend, cuda, make, paged

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    from flashb import _native
    assert _native.device_error() == 0


def test_more_rows_than_the_plan_keeps():
    """1300 rows, runs of 0 to 3 tokens; a plan with more than a row a thread and rows past its table."""
    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, 4, (1300,), generator=g).tolist()
    pasts = torch.randint(0, 40, (1300,), generator=g).tolist()
    check_attend(make(counts, pasts, NH=4, NKV=2, page=16))
    pasts[7], pasts[1111] = 700, 900                            # long enough to cut
    check_attend(make(counts, pasts, NH=4, NKV=2, page=16, seed=2))
    check_append(counts, pasts, NH=2, NKV=1, page=16, rotary=dict())


def test_many_rows_without_a_plan():
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(14, 22, (70,), generator=g).tolist()
    check_attend(make(counts, [0] * 70, NH=4, NKV=4, page=16))


@pytest.mark.parametrize('rows', [33, 128, 131])
def test_runs_of_very_different_lengths_without_a_plan(rows):
    """Query tiles of one row up to seven, empty rows before, between and behind, two to five rows a lane of the search."""
    g = torch.Generator().manual_seed(rows)
    counts = [0] * rows
    for b in torch.randperm(rows, generator=g)[:12].tolist():
        counts[b] = int(torch.randint(1, 200, (1,), generator=g))
    check_attend(make(counts, torch.randint(0, 200, (rows,), generator=g).tolist(), page=16))


@pytest.mark.parametrize('rows,NH,NKV', [(32, 8, 2), (33, 8, 2), (60, 4, 4), (300, 2, 1)])
def test_cut_rows_among_many(rows, NH, NKV):
    """Lists that every CTA works out and lists of the plan, of one row a thread and more."""
    g = torch.Generator().manual_seed(rows)
    counts = torch.randint(0, 4, (rows,), generator=g).tolist()
    pasts = torch.randint(0, 100, (rows,), generator=g).tolist()
    for b in (0, 5, rows // 2, rows - 1):
        counts[b], pasts[b] = 1 + b % 3, 1500 + 100 * (b % 7)
    check_attend(make(counts, pasts, NH, NKV, page=32))
    check_attend(make(counts, pasts, NH, NKV, page=32), 900, 3)


def test_more_query_tiles_than_a_round():
    """Few rows of many tokens: the plan again, most query tiles whole."""
    check_attend(make([2, 1500, 1], [700, 40, 600], NH=8, NKV=8, page=64))


def test_many_query_tiles_joined():
    """More rows to join than warps that join them, most of a query tile's rows without a token."""
    g = torch.Generator().manual_seed(9)
    pasts = torch.randint(900, 2400, (24,), generator=g).tolist()
    check_attend(make([1] * 20 + [3, 2, 20, 1], pasts, NH=8, NKV=2, page=64))


@pytest.mark.parametrize('page', [256, 1024])
def test_large_pages(page):
    check_attend(make([3, 40, 1], [300, 0, 1500], page=page))
    check_attend(make([1, 1], [300, 1500], page=page, single=True))
    check_append([3, 40, 1], [300, 0, 1500], page=page, rotary=dict(layout='interleaved', dim=64))


@pytest.mark.parametrize('NH,NKV', [(16, 4), (8, 8), (16, 2)])
def test_cut_rows(NH, NKV):
    """Long rows of few tokens: query tiles in pieces, of several rows, beside single tokens and short rows."""
    check_attend(make([2, 1, 5, 0, 1, 9], [2500, 1800, 10, 700, 3000, 1100], NH, NKV, page=64))
    check_attend(make([17, 40], [1500, 2100], NH, NKV, page=16))
    check_attend(make([30, 3, 1], [1900, 2500, 2000], NH, NKV, page=32), 700, 40)


def test_cut_rows_with_holes_and_values_that_are_not_finite():
    s = make([20, 3], [2000, 1500], page=16, seed=4)
    s['table'][0, 20:90] = -1
    s['table'][1, 94:] = -1                                     # the last tokens' own pages
    check_attend(s)
    s = make([20, 3], [2000, 1500], page=16, seed=5, nan=False)
    s['values'][int(s['table'][0, 40]), 2, 5] = float('inf')
    s['keys'][int(s['table'][1, 93]), 1, 15] = float('nan')
    m = paged()
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    got = m.attend(s['q'].cuda(), c, cuda(s['table']), cuda(s['lengths']), offsets=cuda(s['offsets'])).cpu()
    want, _ = ref.attend(s['q'], s['keys'], s['values'], s['table'], s['lengths'], s['offsets'])
    odd = ~torch.isfinite(want)
    assert odd.any() and torch.equal(~torch.isfinite(got), odd)
    assert torch.allclose(got.double()[~odd], want[~odd], atol=0.05)


def test_scores_that_grow_and_shrink_along_a_row():
    """The reference of the weights has to move up in later tiles, and stays when scores fall; scores past 2^16."""
    for f in (1.0, 30.0, 3000.0):
        s = make([40, 2], [700, 1200], NH=4, NKV=2, page=64, seed=6)
        for b in range(2):
            n = int(s['lengths'][b])
            for j in range(n):
                e, o = int(s['table'][b, j // 64]), j % 64
                w = (j / n) if b == 0 else (1 - j / n)
                s['keys'][e, :, o] = (s['keys'][e, :, o].float() * w * f).bfloat16()
        check_attend(s, scaling=0.1)


def test_a_whole_step_captured():
    """Plan, single tokens, runs and joins in one graph, replayed on other lengths and runs of the same sizes."""
    m = paged()
    s = make([1, 60, 1, 2], [1500, 1400, 900, 20], page=16, nan=False, width=120)
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    q, table, lengths, off = (cuda(s[k]) for k in ('q', 'table', 'lengths', 'offsets'))
    rot = m.Rotary()
    qkv = torch.randn(64, 24 * D, generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    out, qr = torch.zeros_like(q), torch.zeros_like(q)

    def step():
        m.attend(q, c, table, lengths, offsets=off, out=out)
        m.append(qkv, c, table, lengths, offsets=off, rotary=rot, out=qr)
        m.attend(q, c, table, lengths, offsets=off, out=out)
    step()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    out.zero_()
    for _ in range(3):
        graph.replay()
    assert torch.equal(out, first)
    off.copy_(torch.tensor([0, 30, 31, 63, 64]))
    lengths.copy_(torch.tensor([1200, 1100, 32, 1]))
    graph.replay()
    want, size = ref.attend(s['q'], c.keys.cpu(), c.values.cpu(), s['table'], lengths.cpu(), off.cpu())
    assert torch.all((out.cpu().double() - want).abs() <= (BF + 2.0 ** -11) * size + BF * want.abs())


def test_two_calls_at_once():
    m = paged()
    a, b = make([40, 3], [900, 1500], page=16, seed=8), make([1, 70, 1], [800, 600, 50], page=16, seed=9)
    args = []
    for s in (a, b):
        c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
        args.append((cuda(s['q']), c, cuda(s['table']), cuda(s['lengths']), cuda(s['offsets'])))
    want = [m.attend(*x[:4], offsets=x[4]) for x in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(10):
        for i, (st, x) in enumerate(zip(streams, args)):
            with torch.cuda.stream(st):
                got[i].append(m.attend(*x[:4], offsets=x[4]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_steps_without_dependent_launch():
    from flashb import _native
    s = make([1, 60, 1, 2], [1500, 1400, 900, 20], page=16)
    _native.lib().flashb_set_pdl(0)
    try:
        check_attend(s)
    finally:
        _native.lib().flashb_set_pdl(1)
    check_attend(s)


@pytest.mark.parametrize('norm', [False, True])
@pytest.mark.parametrize('T,NH,NKV', [(9473, 1, 1), (17001, 2, 1), (20011, 7, 3), (33333, 1, 2), (40001, 11, 1)])
def test_append_in_rounds(T, NH, NKV, norm):
    """More tokens than the CTAs that an SM holds take at once: each token's bits are those of a call of its row's part alone."""
    m = paged()
    g = torch.Generator().manual_seed(T)
    cut = [0, 37, 37, T // 3, T - 5000, T]                      # runs, one of them empty
    offsets = torch.tensor(cut)
    lengths = offsets.diff() + torch.tensor([3, 5, 100, 0, 71])
    width = int((lengths.max() + 63) // 64)
    table = torch.randperm(5 * width, generator=g).view(5, width).int()
    qkv = torch.randn(T, (NH + 2 * NKV) * D, generator=g).bfloat16().cuda()
    w = [torch.randn(D, generator=g).bfloat16().cuda() for _ in range(2)] if norm else [None, None]
    rot = m.Rotary(96, layout='interleaved')
    got = []
    for parts in (1, 5):
        keys, values = (torch.zeros(5 * width, NKV, 64, D, dtype=torch.bfloat16, device='cuda') for _ in range(2))
        c = m.PagedCache(keys, values)
        if parts == 1:
            q = m.append(qkv, c, table.cuda(), lengths.cuda(), offsets=offsets.cuda(), rotary=rot, q_norm=w[0], k_norm=w[1])
        else:
            q = torch.zeros_like(got[0][0])
            for b in range(5):
                for lo in range(cut[b], cut[b + 1], 3000):      # pieces of the row's run
                    hi = min(lo + 3000, cut[b + 1])
                    q[lo:hi] = m.append(qkv[lo:hi], c, table[b:b + 1].cuda(), (lengths[b:b + 1] - (cut[b + 1] - hi)).cuda(),
                                        offsets=torch.tensor([0, hi - lo]).cuda(), rotary=rot, q_norm=w[0], k_norm=w[1])
        got.append((q, keys, values))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert int((got[0][2] != 0).any(-1).sum()) == T * NKV       # every token's values are somewhere


def test_infinities_beside_rotated_dims():
    """What is not rotated is copied: an infinity there stays alone, whatever stands beside it."""
    m = paged()
    for layout in ('half', 'interleaved'):
        for dim in (0, 64):
            c = m.PagedCache.empty(2, 1, 16)
            qkv = torch.randn(2, 3 * D, generator=torch.Generator().manual_seed(1)).bfloat16()
            qkv[:, 100] = float('inf')
            qkv[:, D + 127] = float('nan')
            q = m.append(qkv.cuda(), c, torch.tensor([[0], [1]], dtype=torch.int32).cuda(), torch.tensor([3, 9]).cuda(),
                         rotary=m.Rotary(dim, layout=layout) if dim else None)
            odd = torch.zeros(2, D, dtype=torch.bool)
            odd[:, 100] = True
            assert torch.equal(~torch.isfinite(q.cpu()[:, 0]), odd)
            assert torch.equal(q.cpu()[:, 0, dim:], qkv[:, dim:D])
            k = torch.stack((c.keys[0, 0, 2], c.keys[1, 0, 8])).cpu()
            assert torch.isfinite(k[:, :127]).all() and torch.isnan(k[:, 127]).all()


def test_calls_that_are_refused():
    from flashb._native import FB_ERR_ARG, FB_ERR_UNSUPPORTED, FlashbError
    m = paged()
    s = make([5, 9], [10, 30], NH=8, NKV=2, page=16)
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    q, t, n, o = (cuda(s[k]) for k in ('q', 'table', 'lengths', 'offsets'))
    qkv = torch.zeros(14, 12 * D, dtype=torch.bfloat16, device='cuda')
    w = torch.ones(D, dtype=torch.bfloat16, device='cuda')

    def refused(f, *a, rc=FB_ERR_ARG, **kw):
        with pytest.raises(FlashbError) as e:
            f(*a, **kw)
        assert e.value.rc == rc
    for a in ((q.float(), c, t, n), (q.cpu(), c, t, n), (q[:, :, :64], c, t, n), (q, c, t.long(), n), (q, c, t.cpu(), n),
              (q, c, t[0], n), (q, c, t[:, ::2], n), (q, c, t[:0], n), (q, c, t, n.int()), (q, c, t, n[:1]),
              (q, c, t, n.cpu()), (q[:, :7], c, t, n)):
        refused(m.attend, *a, offsets=o)
    refused(m.attend, q[:, :6], c, t, n, offsets=o, rc=FB_ERR_UNSUPPORTED)
    for kw in (dict(offsets=None), dict(offsets=o[:2]), dict(offsets=o.int()), dict(offsets=o, window=0),
               dict(offsets=o, sinks=-1), dict(offsets=o, scaling=0.0), dict(offsets=o, scaling=float('inf')),
               dict(offsets=o, out=q), dict(offsets=o, out=q[:1].expand(14, -1, -1)), dict(offsets=o, out=q.float()),
               dict(offsets=o, out=torch.empty_like(q)[:5])):
        refused(m.attend, q, c, t, n, **kw)
    pool = c.keys.flatten()[:2 * 8 * D].view(2, 8, D)
    refused(m.attend, q[:2], c, t, n, out=pool)
    refused(m.attend, q[:2], c, t, n, out=q[:2])
    for a in ((qkv.float(), c, t, n), (qkv[:, :500], c, t, n), (qkv[:, :512], c, t, n), (qkv.t(), c, t, n), (qkv.cpu(), c, t, n)):
        refused(m.append, *a, offsets=o)
    for kw in (dict(q_norm=w), dict(k_norm=w), dict(q_norm=w.float(), k_norm=w), dict(q_norm=w[:64], k_norm=w),
               dict(positions=n), dict(positions=torch.zeros(14, device='cuda')), dict(out=qkv[:, D:9 * D].view(14, 8, D)),
               dict(out=qkv[:, :8 * D].view(14, 8, D).transpose(0, 1))):
        refused(m.append, qkv, c, t, n, offsets=o, **kw)
    for k, v in ((c.keys, c.keys[:1]), (c.keys[:, :, :8], c.values[:, :, :8]), (c.keys.float(), c.values.float())):
        refused(m.PagedCache, k, v)
    refused(m.append, qkv, m.PagedCache(c.keys, c.keys), t, n, offsets=o)


def test_empty_steps():
    m = paged()
    c = m.PagedCache.empty(2, 2, 16)
    t, n, o = torch.zeros(3, 1, dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int64).cuda(), torch.zeros(
        4, dtype=torch.int64).cuda()
    e = torch.zeros(0, 4, D, dtype=torch.bfloat16).cuda()
    assert m.attend(e, c, t, n, offsets=o).shape == (0, 4, D)
    assert m.append(torch.zeros(0, 8 * D, dtype=torch.bfloat16).cuda(), c, t, n, offsets=o).shape == (0, 4, D)
    q = torch.ones(2, 4, D, dtype=torch.bfloat16).cuda()
    out = torch.full_like(q, 7.0)
    assert torch.equal(m.attend(q, c, t, n, offsets=o, out=out), torch.full_like(q, 7.0))     # tokens of no run


def test_scores_of_nothing_and_refusals():
    from flashb._native import FlashbError
    from flashb.sampling import token_scores
    x, t = torch.zeros(0, 5).cuda(), torch.zeros(0, dtype=torch.int64).cuda()
    assert token_scores(x, t, top=3).top_ids.shape == (0, 3)
    x, t = torch.zeros(2, 5).cuda(), torch.zeros(2, dtype=torch.int64).cuda()
    for a, kw in (((x.half(), t), {}), ((x, t.int()), {}), ((x, t[:1]), {}), ((x, t.cpu()), {}), ((x[0], t), {}),
                  ((x.t(), torch.zeros(5, dtype=torch.int64).cuda()), {}), ((x[:1].expand(2, 5), t), {}),
                  ((x, t), dict(top=6)), ((x, t), dict(top=-1)), ((x, t), dict(temperature=0.0))):
        with pytest.raises(FlashbError):
            token_scores(*a, **kw)
