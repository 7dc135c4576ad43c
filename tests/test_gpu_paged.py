"""The paged cache on the GPU against its definitions in 64 bits: rows of every length, pages anywhere, runs of any size."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
D = 128
BF = 2.0 ** -8                                             # a bf16 rounding, relative


def paged():
    from flashb import paged as m
    return m


def make(counts, pasts, NH=16, NKV=4, page=16, seed=0, spare=3, single=False, nan=True, layout='hnd', width=None):
    """A step of rows with those new tokens over those slots: pages in random order, the pool's other slots NaN."""
    g = torch.Generator().manual_seed(seed)
    lengths = torch.tensor([p + n for p, n in zip(pasts, counts)], dtype=torch.int64)
    need = [-(-max(int(n), 0) // page) for n in lengths]
    W = max(max(need), 1) + 1 if width is None else width
    P = sum(need) + spare
    order = torch.randperm(P, generator=g).int()
    table = torch.full((len(counts), W), -1, dtype=torch.int32)
    shape = (P, NKV, page, D) if layout == 'hnd' else (P, page, NKV, D)
    keys, values = (torch.full(shape, float('nan') if nan else 0.0, dtype=torch.bfloat16) for _ in range(2))
    if layout != 'hnd':
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        for i in range(n):
            m = min(page, int(lengths[b]) - i * page)
            for t in (keys, values):
                t[int(table[b, i]), :, :m] = torch.randn(NKV, m, D, generator=g).bfloat16()
    T = sum(counts)
    q = torch.randn(T, NH, D, generator=g).bfloat16()
    offsets = None if single else torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int64)
    return dict(q=q, keys=keys, values=values, table=table, lengths=lengths, offsets=offsets)


def cuda(x):
    """To the GPU, strides kept."""
    if x is None:
        return None
    if x.dim() == 4 and not x.is_contiguous():
        return x.transpose(1, 2).cuda().transpose(1, 2)
    return x.cuda()


def check_attend(s, window=None, sinks=0, scaling=None, part=None):
    m = paged()
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    out = torch.full(s['q'].shape, 7.0, dtype=torch.bfloat16, device='cuda')
    got = m.attend(cuda(s['q']), c, cuda(s['table']), cuda(s['lengths']), offsets=cuda(s['offsets']), window=window,
                   sinks=sinks, scaling=scaling, out=out)
    assert got is out
    want, size = ref.attend(s['q'], s['keys'], s['values'], s['table'], s['lengths'], s['offsets'], window, sinks,
                            **({} if scaling is None else dict(scaling=scaling)))
    live = ~torch.isnan(size).all(-1).all(-1)
    got = got.cpu().double()
    assert torch.all(got[~live] == 7.0)
    # weights: rounded to one bf16 part (runs) or two (one token a row); scores: sums of 128 products in fp32, up to 2^-11
    # of a weight and its sum; the output's own rounding
    part = part or (BF if s['offsets'] is not None else 2.0 ** -15)
    tol = (part + 2.0 ** -11) * size + BF * want.abs()
    bad = ~((got - want).abs() <= tol) & live[:, None, None]
    assert not bad.any(), (bad.sum(), bad.nonzero()[:4].tolist(), (got - want)[bad][:4], want[bad][:4])
    again = m.attend(cuda(s['q']), c, cuda(s['table']), cuda(s['lengths']), offsets=cuda(s['offsets']), window=window,
                     sinks=sinks, scaling=scaling)
    assert torch.equal(again.cpu()[live], out.cpu()[live])


HEADS = [(16, 4), (8, 2), (4, 4), (16, 8), (16, 2)]


@pytest.mark.parametrize('NH,NKV', HEADS)
@pytest.mark.parametrize('page', [16, 64])
def test_single_tokens(NH, NKV, page):
    check_attend(make([1] * 7, [0, 1, 14, 15, 16, 17, 300], NH, NKV, page, single=True))


@pytest.mark.parametrize('window,sinks', [(1, 0), (5, 0), (16, 1), (33, 4), (64, 17), (100, 64), (1000, 3), (40, 1000)])
def test_single_tokens_window(window, sinks):
    check_attend(make([1] * 6, [0, 31, 63, 99, 257, 511], page=32, single=True), window, sinks)


@pytest.mark.parametrize('rows,past', [(40, 900), (130, 200), (3, 5000)])
def test_single_tokens_many(rows, past):
    g = torch.Generator().manual_seed(rows)
    pasts = torch.randint(0, past, (rows,), generator=g).tolist()
    check_attend(make([1] * rows, pasts, page=64, single=True))
    check_attend(make([1] * rows, pasts, page=16, single=True), 130, 5)


@pytest.mark.parametrize('NH,NKV', HEADS)
@pytest.mark.parametrize('page', [16, 32, 64, 128])
def test_runs(NH, NKV, page):
    check_attend(make([1, 0, 37, 5, 130, 1], [0, 9, 0, 63, 40, 200], NH, NKV, page))


@pytest.mark.parametrize('window,sinks', [(1, 0), (7, 2), (32, 4), (33, 33), (100, 64), (500, 1), (20, 1000)])
def test_runs_window(window, sinks):
    check_attend(make([70, 1, 33, 0, 128], [130, 300, 0, 5, 257], page=16), window, sinks)
    check_attend(make([70, 1, 33, 0, 128], [130, 300, 0, 5, 257], page=128, seed=1), window, sinks)


def test_runs_long_rows():
    check_attend(make([3, 40], [3000, 2500], page=64))
    check_attend(make([20], [4000], NH=8, NKV=2, page=256))


def test_one_run_of_one_token():
    check_attend(make([1], [0]))
    check_attend(make([1], [0], single=True))


def test_tokens_last_layout():
    check_attend(make([5, 60], [100, 3], page=32, layout='nhd'))
    check_attend(make([1, 1], [100, 3], page=32, layout='nhd', single=True))


def test_strided_query_and_output():
    m = paged()
    s = make([5, 60], [100, 3], page=32)
    T = s['q'].shape[0]
    wide = torch.zeros(T, 24, D, dtype=torch.bfloat16, device='cuda')
    wide[:, :16] = s['q'].cuda()
    out = torch.zeros(16, T, D, dtype=torch.bfloat16, device='cuda').transpose(0, 1)
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    args = cuda(s['table']), cuda(s['lengths'])
    m.attend(wide[:, :16], c, *args, offsets=cuda(s['offsets']), out=out)
    assert torch.equal(out, m.attend(s['q'].cuda(), c, *args, offsets=cuda(s['offsets'])))


@pytest.mark.parametrize('single', [False, True])
def test_pages_that_are_not_there(single):
    """Entries of -1 and past the pool: their slots are not visible; a row of them alone gives 0."""
    s = make([1] * 3 if single else [40, 9, 3], [150, 90, 47], page=16, single=single)
    s['table'][0, 2] = -1
    s['table'][0, 5] = 10 ** 9
    s['table'][1, :] = -7
    s['table'][2, 0] = s['keys'].shape[0]
    check_attend(s)
    check_attend(s, 40, 20)


@pytest.mark.parametrize('single', [False, True])
def test_rows_that_see_nothing(single):
    """Lengths of zero, below the run's size, below zero, past the table."""
    s = make([1] * 5 if single else [3, 5, 2, 4, 6], [20, 20, 20, 20, 20], page=16, single=single, width=2)
    s['lengths'][1] = 0
    s['lengths'][2] = -10 ** 12
    s['lengths'][0] = 2
    s['lengths'][3] = 10 ** 12
    s['keys'].nan_to_num_(0.5)
    s['values'].nan_to_num_(0.25)
    check_attend(s)
    check_attend(s, 4, 1)


def test_tokens_outside_the_runs_are_left_alone():
    s = make([4, 8], [10, 30])
    s['offsets'] = torch.tensor([2, 4, 9])
    check_attend(s)


@pytest.mark.parametrize('single', [False, True])
def test_values_that_are_not_finite(single):
    """NaN and infinities in a visible slot show in the rows that see it and in no other."""
    m = paged()
    s = make([1, 1] if single else [20, 30], [100, 64], page=16, single=single, nan=False)
    for t, val in (('values', float('inf')), ('keys', float('nan'))):
        x = {k: (v.clone() if v is not None else None) for k, v in s.items()}
        slot = 110 if not single else 100
        x[t][int(x['table'][0, slot // 16]), 1, slot % 16, 3] = val
        c = m.PagedCache(cuda(x['keys']), cuda(x['values']))
        got = m.attend(x['q'].cuda(), c, cuda(x['table']), cuda(x['lengths']), offsets=cuda(x['offsets'])).cpu()
        want, _ = ref.attend(x['q'], x['keys'], x['values'], x['table'], x['lengths'], x['offsets'])
        odd = ~torch.isfinite(want)
        assert odd.any() and torch.equal(~torch.isfinite(got), odd)
        assert torch.allclose(got.double()[~odd], want[~odd], atol=0.05)


def test_scores_of_minus_infinity_alone():
    m = paged()
    for single in (False, True):
        s = make([1], [40], NH=4, NKV=1, single=single)
        s['q'].fill_(1.0)
        s['keys'].fill_(float('-inf'))
        s['values'].fill_(1.0)
        c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
        got = m.attend(s['q'].cuda(), c, cuda(s['table']), cuda(s['lengths']), offsets=cuda(s['offsets']))
        assert torch.isnan(got).all()


def test_large_scores():
    s = make([9, 33], [120, 64], seed=5)
    s['q'] *= 40
    check_attend(s, scaling=0.25)
    s = make([1, 1], [120, 64], seed=5, single=True)
    s['q'] *= 40
    check_attend(s, scaling=0.25)


# ------------------------------------------------------------------------------------------------------------- append
def check_append(counts, pasts, NH=16, NKV=4, page=16, norm=True, rotary=None, positions=None, single=False, seed=0,
                 in_place=False, layout='hnd', edit=None):
    m = paged()
    s = make(counts, pasts, NH, NKV, page, seed, single=single, nan=False, layout=layout)
    if edit:
        edit(s)
    g = torch.Generator().manual_seed(seed + 1)
    T = sum(counts)
    qkv = torch.randn(T, (NH + 2 * NKV) * D, generator=g).bfloat16()
    w = [(1 + 0.2 * torch.randn(D, generator=g)).bfloat16() for _ in range(2)] if norm else [None, None]
    rot = m.Rotary(**rotary) if rotary is not None else None
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    dq = qkv.cuda()
    out = dq[:, :NH * D].view(T, NH, D) if in_place else torch.full((T, NH, D), 7.0, dtype=torch.bfloat16, device='cuda')
    m.append(dq, c, cuda(s['table']), cuda(s['lengths']), offsets=cuda(s['offsets']), rotary=rot,
             q_norm=cuda(w[0]), k_norm=cuda(w[1]), positions=cuda(positions), out=out, eps=1e-5)
    freq = rot.freq if rot else torch.zeros(0)
    lay, amp = (rot.layout, rot.amplitude) if rot else ('half', 1.0)
    q, K, V = ref.append(qkv, s['keys'], s['values'], s['table'], s['lengths'], s['offsets'], freq, lay, amp, w[0], w[1],
                         1e-5, positions)
    live = ~torch.isnan(q).all(-1).all(-1)
    got = out.cpu().double()
    if not in_place:
        assert torch.all(got[~live] == 7.0)
    # one rounding; the norm's sum and root, the sine and the angle in fp32: 2^-19 of the head's largest value.  The turns
    # per position are freq / 2 pi in 64 bits: 2 pi, the quotient and its product with the position are each off by 2^-53
    # at most, so the angle by 3 x 2^-53 of position x freq radians (freq <= 1), and so much of the head's largest value.
    far = int(positions.abs().max()) if positions is not None else 10 ** 4
    big = (2.0 ** -19 + 3 * 2.0 ** -53 * far) * max(1.0, abs(amp))
    for a, b in ((got[live], q[live]), (c.keys.cpu().double(), K)):
        assert torch.all((a - b).abs() <= BF * b.abs() + big * b.abs().amax(-1, keepdim=True))
    assert torch.equal(c.values.cpu(), V.bfloat16())
    return s


@pytest.mark.parametrize('NH,NKV', HEADS)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_append_heads(NH, NKV, layout):
    check_append([3, 0, 21, 1], [0, 5, 40, 90], NH, NKV, rotary=dict(base=1e4, layout=layout))


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('dim', [16, 32, 48, 64, 96, 112, 128])
def test_append_part_of_the_head(dim, layout):
    check_append([5, 2], [30, 1], rotary=dict(dim=dim, base=500.0, layout=layout), page=32, norm=dim % 32 == 0)


@pytest.mark.parametrize('scaling', [dict(kind='linear', factor=4.0), dict(kind='ntk', factor=8.0),
                                     dict(kind='yarn', factor=16.0, original=2048),
                                     dict(kind='yarn', factor=2.0, original=64, fast=4.0, slow=0.5)])
def test_append_scaled(scaling):
    check_append([5, 2], [300, 1], rotary=dict(base=1e4, scaling=scaling), norm=False)


def test_append_no_rotation_no_norm_in_place_single():
    check_append([5, 2], [30, 1], norm=False)
    check_append([5, 2], [30, 1], rotary=dict(), in_place=True)
    check_append([1] * 9, list(range(9)), rotary=dict(), single=True, page=64)
    check_append([5, 2], [30, 1], rotary=dict(), layout='nhd')
    check_append([1], [0], rotary=dict())


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_append_far_positions(layout):
    pos = torch.tensor([0, 1, 131071, 10 ** 6 + 1, 2 ** 31 + 5, -7, 2 ** 40 + 1])
    check_append([4, 3], [30, 1], rotary=dict(base=1e6, layout=layout), positions=pos)


def test_append_many_tokens_and_rows():
    check_append([3] * 70, list(range(70)), NH=4, NKV=2, rotary=dict())
    check_append([301], [17], NH=4, NKV=2, rotary=dict(), page=128)


def test_append_slots_without_a_page():
    def edit(s):
        s['table'][0, 1] = -1
        s['table'][1, 0] = 10 ** 9
        s['lengths'][2] = 10 ** 10
        s['lengths'][3] = -4
    check_append([20, 3, 5, 2], [10, 4, 7, 9], rotary=dict(), edit=edit, positions=torch.arange(30))


def test_append_then_attend():
    """The two together, a step after a step, against one attention over everything in 64 bits."""
    m = paged()
    NH, NKV, page = 8, 2, 16
    g = torch.Generator().manual_seed(3)
    c = m.PagedCache.empty(20, NKV, page)
    table = torch.randperm(20, generator=g).int()[:18].view(3, 6)
    rot = m.Rotary(base=1e4)
    total = torch.zeros(3, dtype=torch.int64)
    K, V = c.keys.cpu().double(), c.values.cpu().double()
    for counts in ([40, 0, 7], [1, 1, 1], [3, 33, 0], [1, 1, 1]):
        T = sum(counts)
        total += torch.tensor(counts)
        single = counts == [1, 1, 1]
        off = None if single else torch.tensor([0] + list(torch.tensor(counts).cumsum(0)))
        qkv = torch.randn(T, (NH + 2 * NKV) * D, generator=g).bfloat16()
        q = m.append(qkv.cuda(), c, table.cuda(), total.cuda(), offsets=cuda(off), rotary=rot)
        got = m.attend(q, c, table.cuda(), total.cuda(), offsets=cuda(off)).cpu().double()
        rq, K, V = ref.append(qkv, K, V, table, total, off, rot.freq, 'half', 1.0, None, None, 0, None)
        want, size = ref.attend(q.cpu(), c.keys.cpu(), c.values.cpu(), table, total, off)
        assert torch.all((got - want).abs() <= (BF + 2.0 ** -11) * size + BF * want.abs())
        assert torch.all((c.keys.cpu().double() - K).abs() <= BF * K.abs() + 2.0 ** -16)


def test_captured_and_replayed():
    """One graph for steps of any rows up to its size: tokens behind the last run stay as they are."""
    m = paged()
    s = make([40, 9, 3], [150, 90, 47], page=16, nan=False)
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    q, table, lengths, off = (cuda(s[k]) for k in ('q', 'table', 'lengths', 'offsets'))
    out = torch.zeros_like(q)
    m.attend(q, c, table, lengths, offsets=off, out=out)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.attend(q, c, table, lengths, offsets=off, out=out)
    out.zero_()
    graph.replay()
    assert torch.equal(out, first)
    off.copy_(torch.tensor([0, 5, 5, 8]))
    lengths.copy_(torch.tensor([20, 0, 50]))
    out.fill_(7.0)
    graph.replay()
    want, size = ref.attend(s['q'], s['keys'], s['values'], s['table'], lengths.cpu(), off.cpu())
    got = out.cpu().double()
    assert torch.all(got[8:] == 7.0)
    assert torch.all((got - want).abs()[:8] <= ((BF + 2.0 ** -11) * size + BF * want.abs())[:8])


def test_other_stream():
    m = paged()
    s = make([40, 9, 3], [150, 90, 47], page=16, nan=False)
    c = m.PagedCache(cuda(s['keys']), cuda(s['values']))
    args = cuda(s['q']), c, cuda(s['table']), cuda(s['lengths'])
    want = m.attend(*args, offsets=cuda(s['offsets']))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = m.attend(*args, offsets=cuda(s['offsets']))
    st.synchronize()
    assert torch.equal(got, want)
