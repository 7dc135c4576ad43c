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


@pytest.mark.parametrize('bits', [16, 4])
def test_evict_between_views_that_share_no_memory(bits):
    """Two layers of a buffer [B, layers, NKV, S, .], its heads beside its slots, and the two ends of each row's slots."""
    L = lf()
    B, NKV, S, keep = 2, 2, 60, 20
    k, v = randn((B, NKV, S, 128), 34), randn((B, NKV, S, 128), 35)
    acc = torch.rand(B, NKV, S, generator=torch.Generator().manual_seed(36))
    lengths = rows([60, 41])
    want, n_want = ref.evict(acc, lengths, None, keep, 1, 2)
    widths = (128, 128) if bits == 16 else (64, 8, 64, 8)
    dt = torch.bfloat16 if bits == 16 else torch.uint8
    every = lambda f: [f(torch.zeros, w) for w in widths]  # noqa: E731
    layers = every(lambda z, w: z(B, 2, NKV, S, w, dtype=dt, device='cuda'))
    sides = every(lambda z, w: z(B, S, NKV, 2, w, dtype=dt, device='cuda'))
    ends = every(lambda z, w: z(B, NKV, 2 * S, w, dtype=dt, device='cuda'))
    kind = L.KVCache if bits == 16 else L.KV4Cache
    for src, dst in ((kind(*(t[:, 0] for t in layers)), kind(*(t[:, 1] for t in layers))),
                     (kind(*(t[..., 0, :].transpose(1, 2) for t in sides)), kind(*(t[..., 1, :].transpose(1, 2) for t in sides))),
                     (kind(*(t[:, :, :S] for t in ends)), kind(*(t[:, :, S:] for t in ends)))):
        if bits == 16:
            src.keys.copy_(k)
            src.values.copy_(v)
        else:
            src.store(k.cuda(), v.cuda(), torch.arange(S, device='cuda'))
        both = torch.zeros(B, 2, NKV, S, device='cuda')
        both[:, 0].copy_(acc)
        kept, n, moved = L.evict(src, both[:, 0], lengths.cuda(), keep, into=dst, sinks=1, recent=2, acc_into=both[:, 1])
        assert torch.equal(kept.cpu(), want) and torch.equal(n.cpu(), n_want)
        gk, gv = (dst.keys, dst.values) if bits == 16 else dst.read(torch.arange(keep, device='cuda'))
        at = want.clamp(min=0).long()
        for got, x in ((gk, k), (gv, v)):
            x = x.double() if bits == 16 else ref.quantise(x)
            assert torch.equal(got[:, :, :keep].cpu().double(), torch.gather(x, 2, at[..., None].expand(-1, -1, -1, 128)))
        assert torch.equal(moved[..., :keep].cpu(), torch.gather(acc, 2, at)) and (moved[..., keep:] == 0).all()


@pytest.mark.parametrize('std', [2.0 ** -40, 2.0 ** -100])
@pytest.mark.parametrize('scaling', [0.0, 1e-30, -1e-30])
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('B', [1, 70])
def test_decode_scores_too_small_for_fp32(std, scaling, bits, B):
    """A scale that underflows gives every visible slot the same weight, and those past the length none."""
    NH, NKV, S = 8, 2, 150
    q, k, v = randn((B, NH, 1, 128), 4, std), randn((B, NKV, S, 128), 5), randn((B, NKV, S, 128), 6)
    lengths = rows([S - 1 - b % 9 for b in range(B)])
    if bits == 4:
        cache, k, v = four(k, v)
    else:
        cache = lf().KVCache(k.cuda(), v.cuda())
    acc = torch.zeros(B, NKV, S, device='cuda')
    out, wt, tol = ref.decode(q, k, v, lengths, None, None, 0, scaling)
    ref.assert_within(lf().decode(q.cuda(), cache, lengths.cuda(), scaling=scaling, acc=acc), out, tol)
    ref.assert_within(acc, wt, 2.0 ** -18 * wt)


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('B', [1, 70])
def test_decode_shows_a_nan_scaling(bits, B):
    q, k, v = randn((B, 8, 1, 128), 4), randn((B, 2, 150, 128), 5), randn((B, 2, 150, 128), 6)
    cache = four(k, v)[0] if bits == 4 else lf().KVCache(k.cuda(), v.cuda())
    lengths = rows([149 if b else 0 for b in range(B)][::-1])
    got = lf().decode(q.cuda(), cache, lengths.cuda(), scaling=float('nan')).cpu()
    assert torch.isnan(got[:B - 1]).all() and (got[B - 1] == 0).all()


def large(shape, seed):
    """Values of one sign up to bf16's largest: their plain sum passes fp32's range, their mean does not."""
    g = torch.Generator().manual_seed(seed)
    return ((0.5 + 0.5 * torch.rand(shape, generator=g)) * 3.3e38).to(torch.bfloat16)


@pytest.mark.parametrize('B,S', [(1, 300), (1, 9000), (64, 300), (40, 1100)])
@pytest.mark.parametrize('heads', [(8, 2), (8, 8), (16, 2)])
def test_decode_values_up_to_the_largest(B, S, heads):
    NH, NKV = heads
    q, k, v = randn((B, NH, 1, 128), 7), randn((B, NKV, S, 128), 8), large((B, NKV, S, 128), 9)
    lengths = rows([S - b % 5 for b in range(B)])
    out, wt, tol = ref.decode(q, k, v, lengths, None, None, 0, SC)
    acc = torch.zeros(B, NKV, S, device='cuda')
    ref.assert_within(lf().decode(q.cuda(), lf().KVCache(k.cuda(), v.cuda()), lengths.cuda(), acc=acc), out, tol)
    ref.assert_within(acc, wt, 2.0 ** -18 * wt)


@pytest.mark.parametrize('odd', [False, True])
def test_prefill_values_up_to_the_largest(odd):
    """odd: a later slot's NaN has the rows before it computed again."""
    NH, NKV, L = 8, 2, 200
    q, k, v = randn((1, NH, L, 128), 10), randn((1, NKV, L, 128), 11), large((1, NKV, L, 128), 12)
    out, tol = ref.prefill(q, k, v, 0, None, None, 0, SC)
    n = L
    if odd:
        n = L - 1
        v[:, :, n] = float('nan')
    got = lf().prefill(q.cuda(), k.cuda(), v.cuda()).cpu()
    ref.assert_within(got[:, :n], out[:, :n], tol[:, :n])
    assert torch.isnan(got[:, n:]).all()


@pytest.mark.parametrize('e', [-60, -100])
def test_values_far_below_one(e):
    """Down to 2^-100 values keep their relative precision: the bounds without their absolute part."""
    NH, NKV, S = 8, 2, 150
    q, k, v = randn((1, NH, S, 128), 13), randn((1, NKV, S, 128), 14), randn((1, NKV, S, 128), 15) * 2.0 ** e
    out, tol = ref.prefill(q, k, v, 0, None, None, 0, SC)
    ref.assert_within(lf().prefill(q.cuda(), k.cuda(), v.cuda()), out, tol - 1e-30 + 2.0 ** -125)
    out, _, tol = ref.decode(q[:, :, -1:], k, v, rows([S]), None, None, 0, SC)
    got = lf().decode(q[:, :, -1:].cuda(), lf().KVCache(k.cuda(), v.cuda()), rows([S]).cuda())
    ref.assert_within(got, out, tol - 1e-30 + 2.0 ** -125)


@pytest.mark.parametrize('std', [30.0, 300.0])
@pytest.mark.parametrize('window', [None, 150])
def test_prefill_scores_of_any_size(std, window):
    """Nearly one-hot rows whose maximum rises from tile to tile: the sums so far are scaled down again and again."""
    NH, NKV, L = 8, 2, 400
    q, k, v = randn((1, NH, L, 128), 16, std), randn((1, NKV, L, 128), 17), randn((1, NKV, L, 128), 18)
    k = (k.float() * torch.linspace(0.02, 1.0, L)[None, None, :, None]).to(torch.bfloat16)
    out, tol = ref.prefill(q, k, v, 0, None, window, 3, SC)
    # a score is off by at most 2^-21 sum |q k| scaling < 2^-21 x 2^11 at std 300
    got = lf().prefill(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=3)
    ref.assert_within(got, out, tol + 2.0 ** -9 * std / 300 * v.double().abs().max())


@pytest.mark.parametrize('heads,L,window,sinks', [((16, 4), 1500, None, 0), ((16, 4), 1500, 700, 70), ((8, 8), 1300, 1024, 4),
                                                  ((16, 2), 900, 333, 33)])
def test_prefill_of_many_tiles(heads, L, window, sinks):
    NH, NKV = heads
    q, k, v = randn((1, NH, L, 128), 19), randn((1, NKV, L, 128), 20), randn((1, NKV, L, 128), 21)
    out, tol = ref.prefill(q, k, v, 0, rows([5]), window, sinks, SC)
    got = lf().prefill(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=sinks, starts=torch.tensor([5], device='cuda'))
    ref.assert_within(got, out, tol)


@pytest.mark.parametrize('B,NKV,S,keep,sinks,recent', [(1, 2, 13000, 5000, 4, 100), (2, 1, 12000, 64, 0, 0),
                                                       (40, 8, 700, 333, 4, 50), (300, 2, 260, 100, 1, 0)])
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('ties', [False, True])
def test_evict_long_rows_and_many(B, NKV, S, keep, sinks, recent, bits, ties):
    """Rows whose keys do not fit the shared memory, and more rows than CTAs fit the GPU."""
    L = lf()
    g = torch.Generator().manual_seed(22)
    acc = torch.rand(B, NKV, S, generator=g).pow(4)
    if ties:
        acc = (acc * 6).floor() / 4
    lengths = torch.randint(S // 2, S + 1, (B,), generator=g)
    lengths[0] = S
    starts = torch.randint(0, 5, (B,), generator=g)
    k, v = randn((B, NKV, S, 128), 23).cuda(), randn((B, NKV, S, 128), 24).cuda()
    if bits == 4:
        src, dst = L.KV4Cache.empty(B, NKV, S), L.KV4Cache.empty(B, NKV, keep)
        src.store(k, v, torch.arange(S, device='cuda'))
        k, v = src.read(torch.arange(S, device='cuda'))
    else:
        src = L.KVCache(k, v)
        dst = L.KVCache(*(torch.zeros(B, NKV, keep, 128, dtype=torch.bfloat16, device='cuda') for _ in range(2)))
    kept, n, moved = L.evict(src, acc.cuda(), lengths.cuda(), keep, into=dst, starts=starts.cuda(), sinks=sinks,
                             recent=recent)
    want, n_want = ref.evict(acc, lengths, starts, keep, sinks, recent)
    assert torch.equal(kept.cpu(), want) and torch.equal(n.cpu(), n_want)
    gk, gv = dst.read(torch.arange(keep, device='cuda')) if bits == 4 else (dst.keys, dst.values)
    ok, idx = (want >= 0).cuda(), want.clamp(min=0).long().cuda()
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got, torch.gather(x, 2, idx[..., None].expand(-1, -1, -1, 128)) * ok[..., None])
    assert torch.equal(moved, torch.gather(acc.cuda(), 2, idx) * ok)


def test_every_call_in_a_graph_follows_the_device():
    """Prefill, store, read, decode over 4 bits and eviction captured once; the inputs change between replays."""
    L = lf()
    B, NH, NKV, S, n = 2, 8, 2, 160, 50
    q, k, v = randn((B, NH, n, 128), 25).cuda(), randn((B, NKV, n, 128), 26).cuda(), randn((B, NKV, n, 128), 27).cuda()
    starts, lengths = torch.zeros(B, dtype=torch.int64, device='cuda'), torch.tensor([n, n], device='cuda')
    slots = torch.arange(n, device='cuda')
    src, dst = L.KV4Cache.empty(B, NKV, S), L.KV4Cache.empty(B, NKV, S)
    acc = torch.zeros(B, NKV, S, device='cuda')

    def run():
        src.store(k, v, slots)
        kk, vv = src.read(slots)
        a = L.prefill(q, kk, vv, window=20, sinks=2, starts=starts)
        o = L.decode(q[:, :, -1:], src, lengths, starts=starts, window=20, sinks=2, acc=acc)
        return a, o, L.evict(src, acc, lengths, 30, into=dst, starts=starts, sinks=2, recent=4)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, o, (kept, m, _) = run()
    for seed, st, off in ((28, [0, 9], 0), (29, [30, 2], 7)):
        for x, y in ((q, randn(q.shape, seed)), (k, randn(k.shape, seed + 10)), (v, randn(v.shape, seed + 20))):
            x.copy_(y)
        slots.copy_(torch.arange(n) + off)
        starts.copy_(torch.tensor(st) + off)
        lengths.fill_(n + off)
        acc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        k4, v4 = ref.quantise(k.cpu()), ref.quantise(v.cpu())
        # the prefill has the read keys at slots 0 .., its rows begin off slots later there
        want, tol = ref.prefill(q.cpu(), k4, v4, 0, torch.tensor(st) + off, 20, 2, SC)
        ref.assert_within(a, want, tol)
        want, wt, tol = ref.decode(q[:, :, -1:].cpu(), k4, v4, rows([n, n]), torch.tensor(st), 20, 2, SC)
        ref.assert_within(o, want, tol)
        ref.assert_within(acc[:, :, off:n + off], wt, 2.0 ** -18 * wt + 1e-30)
        want, n_want = ref.evict(acc.cpu(), [n + off] * B, [s + off for s in st], 30, 2, 4)
        assert torch.equal(kept.cpu(), want) and torch.equal(m.cpu(), n_want)


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('B,S', [(1, 3000), (64, 900)])
def test_the_same_inputs_give_the_same_bits(B, S, bits):
    L = lf()
    NH, NKV = 16, 4
    q, k, v = randn((B, NH, 40, 128), 30).cuda(), randn((B, NKV, S, 128), 31).cuda(), randn((B, NKV, S, 128), 32).cuda()
    lengths = torch.randint(1, S + 1, (B,), generator=torch.Generator().manual_seed(33)).cuda()
    cache = four(k.cpu(), v.cpu())[0] if bits == 4 else L.KVCache(k, v)
    first = None
    for _ in range(5):
        acc = torch.zeros(B, NKV, S, device='cuda')
        got = [L.decode(q[:, :, :1], cache, lengths, window=700, sinks=3), L.decode(q[:, :, :1], cache, lengths, acc=acc), acc]
        if bits == 16:
            got.append(L.prefill(q, k, v, window=500, sinks=3))
        first = got if first is None else first
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize('scale', [1.0, 2.0 ** 7])
def test_kv4_every_scale_against_every_value_that_matters(scale):
    """Every block maximum's scale, and for each scale every bf16 from its block's maximum down to where codes are 0."""
    bits = torch.arange(0x0001, 0x7f80, dtype=torch.int32).to(torch.int16)
    every = bits.view(torch.bfloat16)                       # the positive finite values, in order
    s = ref.e4m3(every.double() / scale / 6)
    last = torch.nonzero(torch.cat((s[1:] != s[:-1], torch.tensor([True])))).view(-1)
    first = torch.cat((torch.zeros(1, dtype=torch.int64), last[:-1] + 1))
    blocks = []
    for at in torch.cat((first, last, last[-2:-1] + 500)).tolist():
        if s[at] == 0:
            continue
        below = every[max(0, at - 5 * 128):at + 1]           # five binades: codes 0.25 and less are 1 / 24 of the maximum
        below = torch.nn.functional.pad(below, (0, -len(below) % 15)).view(-1, 15)
        blocks.append(torch.cat((every[at].expand(len(below), 1), below), 1))
    x = torch.cat(blocks)
    x = torch.cat((x, torch.cat((every, every.new_zeros(-len(every) % 16))).view(-1, 16)))
    x = torch.where(torch.rand(x.shape, generator=torch.Generator().manual_seed(37)) < 0.5, x, -x)
    x = torch.nn.functional.pad(x.view(-1), (0, -x.numel() % 128)).view(1, 1, -1, 128)
    n = x.shape[2]
    c = lf().KV4Cache.empty(1, 1, n, k_scale=scale, v_scale=1.0)
    c.store(x.cuda(), x.cuda(), torch.arange(n, device='cuda'))
    k, v = c.read(torch.arange(n, device='cuda'))
    assert torch.equal(k.cpu().double(), ref.quantise(x, scale)) and torch.equal(v.cpu().double(), ref.quantise(x))
