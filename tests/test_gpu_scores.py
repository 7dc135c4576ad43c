"""Token scores on the GPU against their definition in 64 bits."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu


def check(x, tokens, top, temperature=1.0, times=1):
    from flashb.sampling import token_scores
    got = token_scores(x.cuda().repeat(times, 1), tokens.cuda().repeat(times), top=top, temperature=temperature)
    lp, h, rank, ids, tl = (a.repeat(times, *[1] * (a.dim() - 1)) for a in ref.scores(x, tokens, top, temperature))
    assert torch.equal(got.rank.cpu(), rank)
    assert torch.equal(got.top_ids.cpu(), ids)
    # differences from the maximum and their scaling in fp32 (2^-22 of them), the sum and its logarithm (2^-18)
    for a, b in ((got.logprob.cpu().double(), lp), (got.top_logprobs.cpu().double(), tl)):
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        fin = torch.isfinite(b)
        assert torch.all((a - b).abs()[fin] <= (2.0 ** -22 * b.abs() + 2.0 ** -18)[fin])
    a = got.entropy.cpu().double()
    assert torch.equal(torch.isnan(a), torch.isnan(h))
    fin = torch.isfinite(h)
    assert torch.all((a - h).abs()[fin] <= (2.0 ** -18 * (1 + h))[fin])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [1, 2, 31, 33, 255, 257, 1000, 2049])
def test_sizes(V, dtype):
    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(5, V, generator=g)).to(dtype)
    check(x, torch.randint(0, V, (5,), generator=g), min(V, 7))
    check(x, torch.randint(0, V, (5,), generator=g), 0, 0.7)
    check(x, torch.randint(0, V, (5,), generator=g), min(V, 32), 2.5)


@pytest.mark.parametrize('V', [4095, 4097, 9001, 40000])
def test_large_vocabularies(V):
    g = torch.Generator().manual_seed(V)
    x = 3 * torch.randn(3, V, generator=g)
    check(x, torch.randint(0, V, (3,), generator=g), 20)
    check(x.bfloat16(), torch.randint(0, V, (3,), generator=g), 20)


def test_many_rows():
    g = torch.Generator().manual_seed(4)
    check(torch.randn(700, 65, generator=g), torch.randint(0, 65, (700,), generator=g), 3)


@pytest.mark.parametrize('V,top,dtype', [(590, 20, torch.float32), (1056, 5, torch.bfloat16), (1056, 32, torch.bfloat16),
                                         (2149, 32, torch.float32), (2149, 3, torch.bfloat16), (2149, 32, torch.bfloat16)])
def test_more_rows_than_the_device_holds(V, top, dtype):
    """Fewer threads a row, more units each."""
    g = torch.Generator().manual_seed(V + top)
    x = 2 * torch.randn(167, V, generator=g)
    x[::7, ::3] = float('-inf')
    t = x.argmax(1)
    t[::2] = torch.randint(0, V, (84,), generator=g)
    t[7::14] -= t[7::14] % 3                                 # ids that are masked themselves
    check(x.to(dtype), t, top, times=30)


@pytest.mark.parametrize('V', [16, 40, 513, 5000])
def test_ranks_among_zeros_and_the_smallest_numbers(V):
    """-0 equals 0; the numbers next to it, on both sides, do not."""
    g = torch.Generator().manual_seed(V)
    for dtype, tiny in ((torch.bfloat16, 2.0 ** -133), (torch.float32, 2.0 ** -149)):
        some = torch.tensor([0.0, -0.0, tiny, -tiny, 2 * tiny], dtype=dtype)
        x = some[torch.randint(0, 5, (20, V), generator=g)]
        assert ((x == 0).sum() > 0) and ((x.abs() == tiny).sum() > 0)
        t = torch.randint(0, V, (20,), generator=g)
        x[0] = 0.0
        x[1, 1:] = tiny
        t[1] = 0                                             # after all of them
        check(x, t, min(V, 9))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_the_rank_of_a_masked_id(dtype):
    """Ids that are masked as well come before it by their number alone, wherever the row's ends lie."""
    g = torch.Generator().manual_seed(11)
    for V in (3, 20, 45, 333):
        x = torch.randn(40, V, generator=g)
        x[:, ::2] = float('-inf')
        check(x.to(dtype), torch.arange(40) * 2 % V // 2 * 2, min(V // 2, 4))


def test_ties_go_to_the_lowest_id():
    x = torch.randint(-3, 3, (6, 500), generator=torch.Generator().manual_seed(1)).float()
    x[1] = 2.0
    x[2, ::2] = -0.0
    x[2, 1::2] = 0.0
    t = torch.tensor([3, 499, 77, 0, 250, 499])
    check(x, t, 32)
    check(x.bfloat16(), t, 32)


def test_rows_whose_largest_logits_crowd():
    """Equal, rising and falling rows; the largest in one thread's vectors; few ids that are not suppressed."""
    V = 20000
    x = torch.zeros(7, V)
    x[1] = torch.arange(V) / 1000
    x[2] = -x[1]
    x[3, ::2048] = torch.arange(10, dtype=torch.float32)
    x[4] = torch.randn(V, generator=torch.Generator().manual_seed(1))
    x[4, 5000:7000] = 9.0
    x[5] = float('-inf')
    x[5, [7, 19999, 4000]] = torch.tensor([1.0, 2.0, 1.0])
    x[6, -3:] = 30.0
    t = torch.tensor([3, 19999, 0, 2048, 6000, 4000, 19998])
    check(x, t, 32)
    check(x, t, 1)
    check(x[:, 1:], t - 1, 20)
    check(x.bfloat16(), t, 20)
    check(x.bfloat16()[:, 3:], t - 3, 5, 0.5)


@pytest.mark.parametrize('V,top', [(100, 32), (276, 32), (300, 9), (511, 20), (600, 31)])
def test_small_vocabularies_many_alternatives(V, top):
    """More logits at the threshold than two a thread, with ties among the last that count."""
    g = torch.Generator().manual_seed(V)
    x = 2 * torch.randn(40, V, generator=g)
    x[:10] = x[:10].round()
    x[10] = 1.0
    x[11, :V // 2] = 5.0
    t = torch.randint(0, V, (40,), generator=g)
    check(x, t, top)
    check(x.bfloat16(), t, top, 0.7)


def test_large_logits():
    x = 100 * torch.randn(4, 2500, generator=torch.Generator().manual_seed(9))
    x[1] *= 1e4
    x[2] *= 1e18
    x[3] *= 1e30
    t = torch.tensor([1, 2, 3, 4])
    check(x, t, 6)
    check(x, t, 6, 0.01)


def test_suppressed_ids_and_rows_without_a_distribution():
    inf, nan = float('inf'), float('nan')
    x = torch.randn(8, 300, generator=torch.Generator().manual_seed(2))
    x[0, 5:] = -inf
    x[1] = -inf
    x[2, 7] = inf
    x[3, 9] = nan
    x[4, 1:] = -inf
    x[5] = 1e30
    x[5, ::2] = -1e30
    x[6] = -3e38
    t = torch.tensor([3, 0, 7, 9, 200, 1, 299, 4])
    check(x, t, 8)
    check(x, torch.tensor([9, -1, 300, 10 ** 12, 0, 0, -10 ** 12, 2 ** 32 + 4]), 8)


def test_strided_rows_and_unaligned_starts():
    g = torch.Generator().manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16):
        wide = (2 * torch.randn(9, 777, generator=g)).to(dtype)
        from flashb.sampling import token_scores
        for lo, hi in ((0, 777), (1, 700), (3, 501), (5, 38)):
            x, t = wide.cuda()[:, lo:hi], torch.arange(9).cuda()
            a, b = token_scores(x, t, top=5), token_scores(x.contiguous(), t, top=5)
            for p, q in zip(a, b):
                assert torch.allclose(p.double(), q.double(), rtol=1e-5, atol=1e-5)
            check(wide[:, lo:hi], torch.arange(9), 5)


def test_sharp_rows_keep_small_numbers():
    """An almost certain token: its log probability and the entropy are small, not zero."""
    x = torch.zeros(3, 2049)
    x[:, 100] = torch.tensor([20.0, 25.0, 30.0])
    from flashb.sampling import token_scores
    got = token_scores(x.cuda(), torch.full((3,), 100).cuda())
    lp, h, *_ = ref.scores(x, torch.full((3,), 100), 0, 1.0)
    assert torch.allclose(got.logprob.cpu().double(), lp, rtol=1e-4, atol=0)
    assert torch.allclose(got.entropy.cpu().double(), h, rtol=1e-4, atol=0)


def test_captured():
    from flashb.sampling import token_scores
    x, t = torch.randn(4, 100, device='cuda'), torch.arange(4, device='cuda')
    token_scores(x, t, top=3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_scores(x, t, top=3)
    x.copy_(torch.randn(4, 100))
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(out, token_scores(x, t, top=3)))
