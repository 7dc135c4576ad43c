"""GPU tests of the long-speech operators against their definitions in 64 bits (``longform_ref``)."""
import pytest
import torch

import longform_ref as ref

pytestmark = pytest.mark.gpu
HEADS = [(16, 4), (8, 8), (4, 2), (16, 2)]
SC = 128 ** -0.5


def lf():
    from flashb import longform
    return longform


def randn(shape, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def four(k, v, k_scale=1.0, v_scale=1.0):
    """A 4-bit cache holding k / v (CPU bf16), and the values it stands for."""
    B, NKV, S, _ = k.shape
    c = lf().KV4Cache.empty(B, NKV, S, k_scale=k_scale, v_scale=v_scale)
    c.store(k.cuda(), v.cuda(), torch.arange(S, device='cuda'))
    return c, ref.quantise(k, k_scale), ref.quantise(v, v_scale)


def rows(x):
    return None if x is None else torch.tensor(x, dtype=torch.int64)


def dev(t):
    return None if t is None else t.cuda()


DECODE = [
    # S, lengths, starts, window, sinks
    (1, [1, 0], None, None, 0),
    (17, [17, 16, 1, 0], [0, 3, 0, 0], None, 0),
    (64, [64, 33], [0, 40], 8, 2),                    # a row that begins after its length: nothing visible
    (130, [130, 129, 128, 65, 64, 63], None, 1, 0),
    (130, [130, 100, 5], [1, 99, 4], 16, 33),         # sinks beyond and inside the window
    (777, [777, 500], [0, 13], 300, 4),
    (2000, [2000], None, None, 0),
    (5, [9, -3], [-2, 0], None, 0),                   # clamped to the cache
]


@pytest.mark.parametrize('heads', HEADS)
@pytest.mark.parametrize('S,lengths,starts,window,sinks', DECODE)
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('scored', [False, True])
def test_decode(heads, S, lengths, starts, window, sinks, bits, scored):
    NH, NKV = heads
    B = len(lengths)
    q, k, v = randn((B, NH, 1, 128), 1, 1.5), randn((B, NKV, S, 128), 2), randn((B, NKV, S, 128), 3)
    if bits == 4:
        cache, k, v = four(k, v)
    else:
        cache = lf().KVCache(k.cuda(), v.cuda())
    lengths, starts = rows(lengths), rows(starts)
    out, wt, tol = ref.decode(q, k, v, lengths, starts, window, sinks, SC)
    acc0 = torch.rand(B, NKV, S, generator=torch.Generator().manual_seed(4))
    acc = acc0.cuda() if scored else None
    got = lf().decode(q.cuda(), cache, lengths.cuda(), starts=dev(starts), window=window, sinks=sinks, acc=acc,
                      decay=0.75)
    ref.assert_within(got, out, tol)
    if scored:
        want = 0.75 * acc0.double() + wt
        # fp32 scores below 2^5 in log2 units, off by 2^-19 at most; the exponential and the sum by 2^-21
        ref.assert_within(acc, want, 2.0 ** -18 * wt + 2.0 ** -23 * want + 1e-30)


@pytest.mark.parametrize('bits', [16, 4])
def test_decode_many_ragged_rows_share_the_grid(bits):
    """Far more chunks than CTAs, rows of every length, and more rows than one scan step of the plan."""
    B, NH, NKV, S = 300, 4, 2, 700
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, S + 1, (B,), generator=g)
    q, k, v = randn((B, NH, 1, 128), 6), randn((B, NKV, S, 128), 7), randn((B, NKV, S, 128), 8)
    if bits == 4:
        cache, k, v = four(k, v)
    else:
        cache = lf().KVCache(k.cuda(), v.cuda())
    out, _, tol = ref.decode(q, k, v, lengths, None, None, 0, SC)
    ref.assert_within(lf().decode(q.cuda(), cache, lengths.cuda()), out, tol)


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_decode_ignores_what_invisible_slots_hold(bits, bad):
    B, NH, NKV, S = 2, 8, 2, 333
    q, k, v = randn((B, NH, 1, 128), 9), randn((B, NKV, S, 128), 10), randn((B, NKV, S, 128), 11)
    lengths, starts, window, sinks = rows([300, 77]), rows([5, 70]), 20, 3
    outs = []
    for poison in (False, True):
        kk, vv = k.clone(), v.clone()
        if poison:
            for b in range(B):
                m = ~ref.visible(int(lengths[b]) - 1, int(starts[b]), S, window, sinks)
                kk[b, :, m], vv[b, :, m] = bad, bad
        cache = four(kk, vv)[0] if bits == 4 else lf().KVCache(kk.cuda(), vv.cuda())
        acc = torch.zeros(B, NKV, S, device='cuda')
        outs.append((lf().decode(q.cuda(), cache, lengths.cuda(), starts=starts.cuda(), window=window, sinks=sinks,
                                 acc=acc), acc))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_decode_shows_a_visible_nan():
    q, k, v = randn((1, 4, 1, 128), 12), randn((1, 2, 40, 128), 13), randn((1, 2, 40, 128), 14)
    v[0, 1, 20, 5] = float('nan')
    out = lf().decode(q.cuda(), lf().KVCache(k.cuda(), v.cuda()), torch.tensor([40], device='cuda')).cpu()
    nan = torch.isnan(out)
    assert nan[0, 0, 2:, 5].all() and nan.sum() == 2


@pytest.mark.parametrize('std', [1e-3, 30.0, 300.0])
def test_decode_scores_of_any_size(std):
    """Nearly flat and nearly one-hot rows; the score errors grow with the scores, so the bound does."""
    q, k, v = randn((2, 8, 1, 128), 15, std), randn((2, 2, 257, 128), 16), randn((2, 2, 257, 128), 17)
    n = rows([257, 100])
    for bits in (16, 4):
        kk, vv = k, v
        if bits == 4:
            cache, kk, vv = four(k, v)
        else:
            cache = lf().KVCache(k.cuda(), v.cuda())
        out, _, tol = ref.decode(q, kk, vv, n, None, None, 0, SC)
        # a score is off by at most 2^-21 sum |q k| scaling < 2^-21 x 2^11 at std 300
        got = lf().decode(q.cuda(), cache, n.cuda())
        ref.assert_within(got, out, tol + 2.0 ** -9 * std / 300 * vv.double().abs().max())


def test_decode_tensor_scales_strides_streams_and_repeats():
    L = lf()
    B, NH, NKV, S = 3, 16, 4, 210
    qkv = randn((B, (NH + 2 * NKV) * 128), 18).cuda()
    q = qkv.as_strided((B, NH, 1, 128), (qkv.stride(0), 128, qkv.stride(0), 1))
    k, v = randn((B, NKV, S, 128), 19, 2.0 ** -9), randn((B, NKV, S, 128), 20, 2.0 ** 13)
    n = rows([210, 1, 64])
    c4, k4, v4 = four(k, v, k_scale=2.0 ** -9, v_scale=2.0 ** 11)
    out, _, tol = ref.decode(q.cpu(), k4, v4, n, None, None, 0, 40.0)
    ref.assert_within(L.decode(q, c4, n.cuda(), scaling=40.0), out, tol)
    # positions, heads and rows at odd distances: [S, B, NKV, 136]
    big = torch.full((2, S, B, NKV, 136), float('nan'), dtype=torch.bfloat16, device='cuda')
    kk, vv = (big[i, ..., :128].permute(1, 2, 0, 3) for i in range(2))
    kk.copy_(k)
    vv.copy_(v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    dn = n.cuda()
    with torch.cuda.stream(side):
        a = L.decode(q, L.KVCache(kk, vv), dn, scaling=40.0, window=50, sinks=1)
        b = L.decode(q, L.KVCache(kk, vv), dn, scaling=40.0, window=50, sinks=1)
    side.synchronize()
    assert torch.equal(a, b)
    out, _, tol = ref.decode(q.cpu(), k, v, n, None, 50, 1, 40.0)
    ref.assert_within(a, out, tol)


def test_decode_in_a_graph_follows_device_lengths():
    L = lf()
    q, k, v = randn((2, 8, 1, 128), 21).cuda(), randn((2, 2, 300, 128), 22), randn((2, 2, 300, 128), 23)
    cache = L.KVCache(k.cuda(), v.cuda())
    n = torch.tensor([10, 300], device='cuda')
    acc = torch.zeros(2, 2, 300, device='cuda')
    out = torch.empty(2, 1, 8, 128, dtype=torch.bfloat16, device='cuda')
    L.decode(q, cache, n, window=64, sinks=4, acc=acc, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.decode(q, cache, n, window=64, sinks=4, acc=acc, out=out)
    for a in ([1, 2], [150, 299], [0, 77]):
        n.copy_(torch.tensor(a))
        acc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want, wt, tol = ref.decode(q.cpu(), k, v, rows(a), None, 64, 4, SC)
        ref.assert_within(out, want, tol)
        ref.assert_within(acc, wt, 2.0 ** -18 * wt + 1e-30)


def test_decode_slots_past_two_gigabytes():
    """Byte offsets beyond 32 bits: one head of 2^23 + 5 slots is over 2 GB of keys."""
    S = 2 ** 23 + 5
    k = torch.zeros(1, 1, S, 128, dtype=torch.bfloat16, device='cuda')
    v = torch.zeros(1, 1, S, 128, dtype=torch.bfloat16, device='cuda')
    tk, tv, q = randn((70, 128), 24), randn((70, 128), 25), randn((1, 2, 1, 128), 26)
    at = torch.cat((torch.arange(6), torch.arange(S - 64, S)))
    k[0, 0, at.cuda()], v[0, 0, at.cuda()] = tk.cuda(), tv.cuda()
    got = lf().decode(q.cuda(), lf().KVCache(k, v), torch.tensor([S], device='cuda'), window=64, sinks=6)
    out, _, tol = ref.decode(q, tk[None, None], tv[None, None], rows([70]), None, None, 0, SC)
    ref.assert_within(got, out, tol)


PREFILL = [
    # L, past, starts, window, sinks
    (1, 0, [0, 0], None, 0),
    (1, 40, [0, 41], 7, 1),                           # the second row begins after its only token
    (33, 0, [0, 20], None, 0),
    (130, 0, [5, 0], 1, 0),
    (127, 3, [0, 64], 31, 40),
    (300, 0, [0, 17], 64, 4),
    (200, 171, [0, 190], 128, 1),
    (260, 0, None, 5000, 3),
]


@pytest.mark.parametrize('heads', HEADS)
@pytest.mark.parametrize('L,past,starts,window,sinks', PREFILL)
def test_prefill(heads, L, past, starts, window, sinks):
    NH, NKV = heads
    q, k, v = randn((2, NH, L, 128), 31, 1.5), randn((2, NKV, past + L, 128), 32), randn((2, NKV, past + L, 128), 33)
    out, tol = ref.prefill(q, k, v, past, rows(starts), window, sinks, SC)
    got = lf().prefill(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=sinks, starts=dev(rows(starts)))
    ref.assert_within(got, out, tol)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_prefill_ignores_what_invisible_slots_hold(bad):
    """Left padding, slots past the tokens, slots behind the window, and for each token the slots after it."""
    NH, NKV, L, past, S = 8, 2, 150, 90, 300
    starts, window, sinks = rows([7, 100]), 25, 5
    q, k, v = randn((2, NH, L, 128), 34), randn((2, NKV, S, 128), 35), randn((2, NKV, S, 128), 36)
    run = lambda kk, vv: lf().prefill(q.cuda(), kk.cuda(), vv.cuda(), window=window, sinks=sinks,  # noqa: E731
                                      starts=starts.cuda(), q_start=past)
    clean, tol = ref.prefill(q, k, v, past, starts, window, sinks, SC)
    m = torch.stack([torch.stack([ref.visible(past + i, int(s), S, window, sinks) for i in range(L)]) for s in starts])
    kk, vv = k.clone(), v.clone()
    for b in range(2):
        kk[b, :, ~m[b].any(0)], vv[b, :, ~m[b].any(0)] = bad, bad
    ref.assert_within(run(kk, vv), clean, tol)
    # one poisoned slot that some tokens see: the others' outputs stay
    j = past + 70
    kk, vv = k.clone(), v.clone()
    kk[:, :, j], vv[:, :, j] = bad, bad
    got = run(kk, vv).cpu().double()
    for b in range(2):
        free = ~m[b, :, j]
        ref.assert_within(got[b, free], clean[b, free], tol[b, free])
        assert torch.isnan(got[b, ~free]).all()


def test_prefill_strides_and_out():
    NH, NKV, L = 8, 4, 75
    qkv = randn((2 * L, (NH + 2 * NKV) * 128 + 8), 37).cuda()
    st = qkv.stride(0)
    view = lambda h0, n: qkv[:, h0 * 128:].as_strided((2, n, L, 128), (L * st, 128, st, 1),  # noqa: E731
                                                       qkv.storage_offset() + h0 * 128)
    q, k, v = view(0, NH), view(NH, NKV), view(NH + NKV, NKV)
    big = torch.zeros(2, NH, L, 128, dtype=torch.bfloat16, device='cuda')
    got = lf().prefill(q, k, v, window=20, sinks=2, scaling=0.2, out=big.transpose(1, 2))
    out, tol = ref.prefill(q.cpu(), k.cpu(), v.cpu(), 0, None, 20, 2, 0.2)
    ref.assert_within(got, out, tol)


def test_decode_continues_a_prefill():
    """The last token of a prefill is the token a decode step computes."""
    q, k, v = randn((2, 16, 90, 128), 38).cuda(), randn((2, 4, 90, 128), 39).cuda(), randn((2, 4, 90, 128), 40).cuda()
    st = torch.tensor([0, 11], device='cuda')
    a = lf().prefill(q, k, v, window=33, sinks=4, starts=st)[:, -1:]
    b = lf().decode(q[:, :, -1:], lf().KVCache(k, v), torch.tensor([90, 90], device='cuda'), starts=st, window=33, sinks=4)
    out, _, tol = ref.decode(q[:, :, -1:].cpu(), k.cpu(), v.cpu(), rows([90, 90]), rows([0, 11]), 33, 4, SC)
    ref.assert_within(a, out, tol)
    ref.assert_within(b, out, tol)


def awkward():
    """Heads that reach every code, tie, scale and special case of the 4-bit form."""
    g = torch.Generator().manual_seed(41)
    x = torch.randn(64, 128, generator=g)
    x[1] = 0
    x[2] *= 2.0 ** -20                                           # the scale rounds to 0
    x[3] *= 2.0 ** -7                                            # subnormal scales
    x[4] *= 1e5                                                  # saturated
    x[5] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] * 16)      # ties at scale 1
    x[6] = -3 * x[5]                                             # ties at scale 3
    x[7] = torch.linspace(-1, 1, 128)
    x[8, 17], x[9, 40], x[10, 0] = float('nan'), float('inf'), -float('inf')
    # block maxima on and around ties of the e4m3 scale
    x[11:43] = 0.001 * x[11:43]
    x[11:43, ::16] = (6 * (1 + torch.arange(256) / 16).view(32, 8)) * 2.0 ** (torch.arange(32) - 20).view(32, 1)
    x[43] = 1e-40
    x[44] = -0.0
    x[45] = 3e38
    return x.to(torch.bfloat16)


@pytest.mark.parametrize('scale', [1.0, 2.0 ** -10, 64.0])
def test_kv4_is_exact_arithmetic(scale):
    x = awkward().view(1, 1, 64, 128)
    y = x.flip(2).contiguous()
    c = lf().KV4Cache.empty(1, 1, 80, k_scale=scale, v_scale=1.0)
    slots = torch.randperm(80, generator=torch.Generator().manual_seed(42))[:64].cuda()
    c.store(x.cuda(), y.cuda(), slots)
    k, v = c.read(slots)
    for got, want in ((k, ref.quantise(x, scale)), (v, ref.quantise(y))):
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=-7e77), torch.nan_to_num(want, nan=-7e77))


@pytest.mark.parametrize('L', [1, 2, 3, 16, 17, 100])
def test_kv4_slots_per_row_strides_and_edges(L):
    B, NKV, S = 3, 2, 100
    qkv = randn((B * L, 5 * 128), 43).cuda()
    k = qkv.as_strided((B, NKV, L, 128), (L * 640, 128, 640, 1), 128)
    v = qkv.as_strided((B, NKV, L, 128), (L * 640, 128, 640, 1), 384)
    slots = torch.stack([torch.arange(L) + o for o in (0, -1, S - L + 1)]).cuda()     # two rows leave the cache
    c = lf().KV4Cache.empty(B, NKV, S)
    c.store(k, v, slots)
    gk, gv = c.read(slots)
    ok = ((slots >= 0) & (slots < S)).cpu()[:, None, :, None]
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got.cpu().double(), ref.quantise(x.cpu()) * ok)
    # nothing else was written
    every = c.read(torch.arange(S, device='cuda'))[0].cpu()
    held = torch.zeros(B, S, dtype=torch.bool)
    for b in range(B):
        held[b, slots[b][(slots[b] >= 0) & (slots[b] < S)].cpu()] = True
    assert (every.abs().sum((1, 3)) > 0).equal(held)


def test_kv4_codes_are_e2m1_and_e4m3():
    x = awkward()[11:43].view(1, 1, 32, 128).cuda()
    c = lf().KV4Cache.empty(1, 1, 32)
    c.store(x, x, torch.arange(32, device='cuda'))
    code = torch.stack((c.kq & 15, c.kq >> 4), -1).flatten(-2).cpu()
    val = torch.cat((ref.GRID, -ref.GRID))[code.int()].view(32, 8, 16)
    s = c.ks.cpu().view(torch.float8_e4m3fn).double().view(32, 8, 1)
    assert torch.equal((val * s).view(1, 1, 32, 128), ref.quantise(x.cpu()))


EVICT = [
    # S, lengths, starts, keep, sinks, recent
    (1, [1, 0], None, 1, 0, 0),
    (40, [40, 13, 12, 0], [0, 0, 5, 0], 12, 2, 3),
    (1500, [1500, 1025, 700], [0, 1, 650], 333, 4, 100),
    (1500, [1500, 1500], None, 64, 64, 0),            # nothing to choose
    (1500, [1500, 1499], None, 64, 0, 64),
    (5000, [5000], [4], 4096, 0, 0),
    (90, [200, -5], [-3, 0], 50, 1, 1),
]


@pytest.mark.parametrize('S,lengths,starts,keep,sinks,recent', EVICT)
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('kind', ['spread', 'ties', 'special'])
def test_evict(S, lengths, starts, keep, sinks, recent, bits, kind):
    L = lf()
    B, NKV = len(lengths), 2
    g = torch.Generator().manual_seed(50)
    acc = torch.rand(B, NKV, S, generator=g).pow(4)
    if kind == 'ties':
        acc = (acc * 6).floor() / 4
    if kind == 'special':
        acc[..., ::3] = 0.0
        acc[..., 1::7] = -0.0
        acc[..., 2::11] = float('nan')
        acc[..., 3::13] = float('inf')
        acc[..., 4::17] = -1.5
    k, v = randn((B, NKV, S, 128), 51), randn((B, NKV, S, 128), 52)
    room = keep + 9
    if bits == 4:
        src, k, v = four(k, v)
        dst = L.KV4Cache.empty(B, NKV, room)
    else:
        src = L.KVCache(k.cuda(), v.cuda())
        dst = L.KVCache(*(torch.zeros(B, NKV, room, 128, dtype=torch.bfloat16, device='cuda') for _ in range(2)))
    acc_into = torch.full((B, NKV, room), 7.0, device='cuda')
    kept, n, moved = L.evict(src, acc.cuda(), rows(lengths).cuda(), keep, into=dst, starts=dev(rows(starts)), sinks=sinks,
                             recent=recent, acc_into=acc_into)
    want, n_want = ref.evict(acc, lengths, starts, keep, sinks, recent)
    assert torch.equal(kept.cpu(), want) and torch.equal(n.cpu(), n_want) and moved is acc_into
    at = torch.arange(room, device='cuda')
    gk, gv = dst.read(at) if bits == 4 else (dst.keys, dst.values)
    slot = torch.full((B, NKV, room), -1)
    slot[..., :keep] = want
    ok = slot >= 0
    idx = slot.clamp(min=0).long()
    for got, x in ((gk, k), (gv, v)):
        rows_ = torch.gather(x.double(), 2, idx[..., None].expand(-1, -1, -1, 128)) * ok[..., None]
        assert torch.equal(got.cpu().double(), rows_)
    a = torch.where(ok, torch.gather(acc, 2, idx), torch.zeros(()))
    assert torch.equal(torch.nan_to_num(moved.cpu(), nan=-9.0), torch.nan_to_num(a, nan=-9.0))


def test_bounded_cache_end_to_end():
    """Decode with accumulation, evict into a smaller cache, go on decoding there: the second decode sees exactly the
    kept slots."""
    L = lf()
    B, NH, NKV, S = 2, 8, 2, 400
    q, k, v = randn((B, NH, 1, 128), 60), randn((B, NKV, S, 128), 61), randn((B, NKV, S, 128), 62)
    src = L.KVCache(k.cuda(), v.cuda())
    acc = torch.zeros(B, NKV, S, device='cuda')
    n = torch.tensor([400, 250], device='cuda')
    L.decode(q.cuda(), src, n, acc=acc)
    dst = L.KVCache(*(torch.zeros(B, NKV, 128, 128, dtype=torch.bfloat16, device='cuda') for _ in range(2)))
    kept, n2, _ = L.evict(src, acc, n, 100, into=dst, sinks=4, recent=32)
    got = L.decode(q.cuda(), dst, n2)
    kept = kept.cpu().long()
    for h in range(NKV):
        kk = torch.stack([k[b, h, kept[b, h]] for b in range(B)])[:, None]
        vv = torch.stack([v[b, h, kept[b, h]] for b in range(B)])[:, None]
        out, _, tol = ref.decode(q[:, 4 * h:4 * h + 4], kk, vv, rows([100, 100]), None, None, 0, SC)
        ref.assert_within(got[:, :, 4 * h:4 * h + 4], out, tol)


def test_refusals():
    from flashb._native import FlashbError
    L = lf()
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device='cuda')  # noqa: E731
    q, k = z(2, 8, 1, 128), z(2, 2, 16, 128)
    c, n = L.KVCache(k, k.clone()), torch.tensor([3, 4], device='cuda')
    bad = [
        lambda: L.KVCache(k.float(), k.float()),
        lambda: L.KVCache(k[..., :64], k[..., :64]),
        lambda: L.KVCache(k, z(2, 2, 17, 128)),
        lambda: L.KVCache(k.cpu(), k.cpu()),
        lambda: L.decode(q.float(), c, n),
        lambda: L.decode(z(2, 8, 2, 128), c, n),
        lambda: L.decode(z(3, 8, 1, 128), c, n),
        lambda: L.decode(z(2, 6, 1, 128), c, n),                     # a group of 3
        lambda: L.decode(z(2, 7, 1, 128), c, n),
        lambda: L.decode(z(2, 64, 1, 128), c, n),                    # a group of 32
        lambda: L.decode(q, c, n.int()),
        lambda: L.decode(q, c, n.cpu()),
        lambda: L.decode(q, c, n[:1]),
        lambda: L.decode(q, c, n, window=0),
        lambda: L.decode(q, c, n, window=4, sinks=-1),
        lambda: L.decode(q, c, n, acc_out=z(2, 2, 16, dt=torch.float32)),
        lambda: L.decode(q, c, n, acc=z(2, 2, 15, dt=torch.float32)),
        lambda: L.decode(q, c, n, acc=z(2, 2, 16)),
        lambda: L.decode(q, c, n, out=z(2, 1, 4, 128)),
        lambda: L.decode(z(2, 8, 1, 132)[..., 4:], c, n),            # rows 8 bytes off a 16-byte boundary
        lambda: L.decode(q, L.KVCache(z(2, 2, 16, 132)[..., 4:], k), n),
        lambda: L.prefill(z(2, 8, 5, 128), k, k, q_start=12),
        lambda: L.prefill(z(2, 8, 5, 128), k, k, q_start=-1),
        lambda: L.prefill(z(2, 8, 17, 128), k, k),
        lambda: L.prefill(z(2, 6, 5, 128), k, k),
        lambda: L.prefill(z(2, 8, 5, 128), k, k, out=z(2, 8, 5, 128)),
        lambda: L.prefill(z(2, 8, 5, 128), k, k, window=-1),
        lambda: L.KV4Cache.empty(2, 2, 16, k_scale=3.0),
        lambda: L.evict(c, z(2, 2, 16, dt=torch.float32), n, 4, into=c),
        lambda: L.evict(c, z(2, 2, 16, dt=torch.float32), n, 17, into=L.KVCache(z(2, 2, 16, 128), z(2, 2, 16, 128))),
        lambda: L.evict(c, z(2, 2, 16, dt=torch.float32), n, 4, into=L.KVCache(z(2, 2, 16, 128), z(2, 2, 16, 128)),
                        sinks=3, recent=2),
        lambda: L.evict(c, z(2, 2, 16, dt=torch.float32), n, 4, into=L.KV4Cache.empty(2, 2, 16)),
        lambda: L.evict(c, z(2, 2, 16, dt=torch.float32), n, 0, into=L.KVCache(z(2, 2, 16, 128), z(2, 2, 16, 128))),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(FlashbError):
            f()
            pytest.fail(f'case {i} was accepted')
    c4 = L.KV4Cache.empty(2, 2, 16)
    for f in (lambda: c4.store(k.float(), k, torch.arange(16, device='cuda')),
              lambda: c4.store(k, k[:, :, :5], torch.arange(16, device='cuda')),
              lambda: c4.store(k, k, torch.arange(15, device='cuda')),
              lambda: c4.store(k, k, torch.arange(16, device='cuda').int()),
              lambda: c4.read(torch.zeros(3, 16, dtype=torch.int64, device='cuda'))):
        with pytest.raises(FlashbError):
            f()
    assert torch.cuda.is_available() and float(z(1).sum()) == 0.0      # the context is fine


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('B,S', [(1, 9000), (2, 8192), (8, 4500), (24, 640), (40, 300)])
def test_decode_on_either_side_of_the_cluster_rule(B, S, bits):
    """Few rows of many keys and more rows of fewer: one cluster a row, or the shared list (with many pieces a row)."""
    NH, NKV = 16, 4
    g = torch.Generator().manual_seed(70)
    lengths = torch.randint(S // 2, S + 1, (B,), generator=g)
    lengths[0] = S
    q, k, v = randn((B, NH, 1, 128), 71), randn((B, NKV, S, 128), 72), randn((B, NKV, S, 128), 73)
    if bits == 4:
        cache, k, v = four(k, v)
    else:
        cache = lf().KVCache(k.cuda(), v.cuda())
    out, wt, tol = ref.decode(q, k, v, lengths, None, None, 0, SC)
    acc = torch.zeros(B, NKV, S, device='cuda')
    ref.assert_within(lf().decode(q.cuda(), cache, lengths.cuda()), out, tol)
    ref.assert_within(lf().decode(q.cuda(), cache, lengths.cuda(), acc=acc), out, tol)
    ref.assert_within(acc, wt, 2.0 ** -18 * wt + 1e-30)


def test_decode_scored_with_eight_heads_a_group_in_full_clusters():
    """The most shared memory a cluster's CTA can want: 8 chunks of scores of 8 heads."""
    B, NH, NKV, S = 1, 16, 2, 16384
    q, k, v = randn((B, NH, 1, 128), 74), randn((B, NKV, S, 128), 75), randn((B, NKV, S, 128), 76)
    cache, k, v = four(k, v)
    n = rows([S])
    out, wt, tol = ref.decode(q, k, v, n, None, None, 0, SC)
    acc = torch.zeros(B, NKV, S, device='cuda')
    ref.assert_within(lf().decode(q.cuda(), cache, n.cuda(), acc=acc), out, tol)
    ref.assert_within(acc, wt, 2.0 ** -18 * wt + 1e-30)


# slots (of the cache's last 300) that hold the odd key: the last one, alone in its tile; one among others; a tile's all
ODD = [[299], [150], list(range(256, 288))]


def at_the_end(B, S, n, at):
    """A cache of B rows whose last n slots are visible, and the slots ``at`` of those."""
    return [S - n + j for j in at], rows([S] * B)


@pytest.mark.parametrize('at', ODD)
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('B,S', [(1, 300), (1, 9000), (64, 300), (40, 1100)])
@pytest.mark.parametrize('scored', [False, True])
def test_decode_shows_a_visible_nan_key_wherever_it_lies(at, bits, B, S, scored):
    """One NaN score makes its head's softmax NaN, in whichever part of the row it is; other heads and rows stay."""
    NH, NKV = 8, 2
    q, k, v = randn((B, NH, 1, 128), 70), randn((B, NKV, S, 128), 71), randn((B, NKV, S, 128), 72)
    slots, lengths = at_the_end(B, S, 300, at)
    starts = torch.full((B,), S - 300, dtype=torch.int64).cuda()
    def run(kk):
        cache = four(kk, v)[0] if bits == 4 else lf().KVCache(kk.cuda(), v.cuda())
        acc = torch.zeros(B, NKV, S, device='cuda') if scored else None
        return lf().decode(q.cuda(), cache, lengths.cuda(), starts=starts, acc=acc), acc
    clean, w0 = run(k)
    kk = k.clone()
    kk[B // 2, 1, slots] = float('nan')
    got, w1 = run(kk)
    assert torch.isnan(got[B // 2, 0, 4:]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[B // 2, 0, 4:] = False
    assert torch.equal(got[keep], clean[keep])
    if scored:
        assert torch.isnan(w1[B // 2, 1, S - 300:]).all()
        keep = torch.ones_like(w1, dtype=torch.bool)
        keep[B // 2, 1, S - 300:] = False
        assert torch.equal(w1[keep], w0[keep])


@pytest.mark.parametrize('B,S', [(1, 300), (64, 300), (40, 1100)])
@pytest.mark.parametrize('scored', [False, True])
def test_decode_scores_of_minus_infinity(B, S, scored):
    """A key with a score of -inf weighs nothing; where all are, softmax has 0 / 0."""
    NH, NKV = 4, 2
    q, k, v = randn((B, NH, 1, 128), 73), randn((B, NKV, S, 128), 74), randn((B, NKV, S, 128), 75)
    q[..., 0] = 1.0
    k[0, :, ::3, 0] = float('-inf')
    k[0, 0, S - 64:, 0] = float('-inf')                    # the last tiles whole
    lengths = rows([S] * B)
    acc = torch.zeros(B, NKV, S, device='cuda') if scored else None
    out, wt, tol = ref.decode(q, k, v, lengths, None, None, 0, SC)
    ref.assert_within(lf().decode(q.cuda(), lf().KVCache(k.cuda(), v.cuda()), lengths.cuda(), acc=acc), out, tol)
    if scored:
        assert (acc[0, :, ::3] == 0).all() and torch.isfinite(acc).all()
    k[0, 1, :, 0] = float('-inf')
    got = lf().decode(q.cuda(), lf().KVCache(k.cuda(), v.cuda()), lengths.cuda(), acc=acc)
    assert torch.isnan(got[0, 0, 2:]).all() and torch.isfinite(got[0, 0, :2]).all() and torch.isfinite(got[1:]).all()
    if scored:
        assert torch.isnan(acc[0, 1]).all() and torch.isfinite(acc[0, 0]).all()


def test_prefill_scores_of_minus_infinity():
    NH, NKV, L, pad = 4, 2, 200, 3
    q, k, v = randn((1, NH, L, 128), 76), randn((1, NKV, L, 128), 77), randn((1, NKV, L, 128), 78)
    q[..., 0] = 1.0
    k[0, :, 100:110, 0] = float('-inf')
    starts = rows([pad])
    for window in (None, 8):                                # 8: tokens 107 to 109 see such keys alone
        out, tol = ref.prefill(q, k, v, 0, starts, window, 0, SC)
        got = lf().prefill(q.cuda(), k.cuda(), v.cuda(), window=window, starts=starts.cuda()).cpu()
        nan = torch.isnan(out)
        assert torch.equal(torch.isnan(got), nan) and bool(nan.any()) == (window == 8)
        ref.assert_within(got[~nan], out[~nan], tol[~nan])
        assert (got[0, :pad] == 0).all()


@pytest.mark.parametrize('big', [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 62])
def test_windows_and_sinks_of_any_size(big):
    """More than the cache holds, past 32 bits too: no window, or every slot a sink."""
    NH, NKV, S, L = 8, 2, 200, 70
    q, k, v = randn((1, NH, L, 128), 79).cuda(), randn((1, NKV, S, 128), 80).cuda(), randn((1, NKV, S, 128), 81).cuda()
    starts, n = torch.tensor([9], device='cuda'), torch.tensor([S], device='cuda')
    cache = lf().KVCache(k, v)
    whole, step = lf().prefill(q, k, v, starts=starts), lf().decode(q[:, :, -1:], cache, n, starts=starts)
    for kw in (dict(window=big), dict(window=16, sinks=big), dict(window=big, sinks=big)):
        # the same sums over other tiles: equal up to the rounding of the weights
        torch.testing.assert_close(lf().prefill(q, k, v, starts=starts, **kw), whole, atol=2.0 ** -6, rtol=2.0 ** -6)
        torch.testing.assert_close(lf().decode(q[:, :, -1:], cache, n, starts=starts, **kw), step, atol=2.0 ** -6, rtol=2.0 ** -6)
    from flashb._native import FlashbError
    into = lf().KVCache(torch.zeros_like(k), torch.zeros_like(v))
    acc = torch.zeros(1, NKV, S, device='cuda')
    for f in (lambda: lf().evict(cache, acc, n, big, into=into), lambda: lf().evict(cache, acc, n, 8, into=into, sinks=big),
              lambda: lf().evict(cache, acc, n, 8, into=into, recent=big), lambda: lf().prefill(q, k, v, q_start=big),
              lambda: lf().decode(q[:, :, -1:], cache, n, window=4, sinks=-big),
              lambda: lf().evict(cache, acc, n, 8, into=into, starts=starts, lengths_into=starts)):
        with pytest.raises(FlashbError):
            f()


@pytest.mark.parametrize('scaling', [-0.1, 0.0, 0.05])
@pytest.mark.parametrize('heads', HEADS)
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('B', [1, 70])
def test_decode_scalings_of_any_sign(scaling, heads, bits, B):
    NH, NKV = heads
    S = 150
    q, k, v = randn((B, NH, 1, 128), 82), randn((B, NKV, S, 128), 83), randn((B, NKV, S, 128), 84)
    lengths = rows([S - b % 9 for b in range(B)])
    if bits == 4:
        cache, k, v = four(k, v)
    else:
        cache = lf().KVCache(k.cuda(), v.cuda())
    acc = torch.zeros(B, NKV, S, device='cuda')
    out, wt, tol = ref.decode(q, k, v, lengths, None, None, 0, scaling)
    ref.assert_within(lf().decode(q.cuda(), cache, lengths.cuda(), scaling=scaling, acc=acc), out, tol)
    assert (acc.cpu().double() - wt).abs().max() <= 2.0 ** -12 * wt.max()
