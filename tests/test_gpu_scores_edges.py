"""Token scores on the GPU where it can go wrong: what few warps work out for a row, masks at every temperature."""
import pytest
import torch

import paged_ref as ref
from test_gpu_scores import check

pytestmark = pytest.mark.gpu
MAX = torch.finfo(torch.float32).max


def check_far(x, tokens, top, temperature):
    """``check`` for values that may be past fp32's range, in which the outputs are: past its ends they are infinite."""
    from flashb.sampling import token_scores
    got = token_scores(x.cuda(), tokens.cuda(), top=top, temperature=temperature)
    lp, h, rank, ids, tl = ref.scores(x, tokens, top, temperature)
    assert torch.equal(got.rank.cpu(), rank) and torch.equal(got.top_ids.cpu(), ids)
    for a, b in ((got.logprob.cpu().double(), lp), (got.top_logprobs.cpu().double(), tl)):
        b = torch.where(b < -MAX, torch.full_like(b, -float('inf')), b)
        fin = torch.isfinite(b)
        assert torch.equal(torch.isfinite(a), fin) and torch.equal(a[~fin], b[~fin])
        # differences from the maximum, the temperature's inverse, their product and the logarithm taken from it: four
        # roundings of 2^-24 each; the sum and its logarithm 2^-18
        assert torch.all((a - b).abs()[fin] <= (2.0 ** -22 * b.abs() + 2.0 ** -18)[fin])
    a = got.entropy.cpu().double()
    assert torch.all((a - h).abs() <= 2.0 ** -18 * (1 + h)) and not h.isnan().any()


@pytest.mark.parametrize('V,dtype', [(1100, torch.float32), (2049, torch.float32), (2200, torch.bfloat16), (4099, torch.bfloat16)])
def test_rows_thinned_by_one_of_several_warps(V, dtype):
    """130 to 512 logits at the threshold in CTAs of two and four warps: the branch that one warp works out alone."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(6, V, generator=g).clamp(max=3.0)
    for r, n in enumerate((130, 257, 300, 400, 511, 512)):
        at = torch.randperm(V, generator=g)[:n]
        x[r, at] = 9.0 if r % 2 else torch.randint(8, 20, (n,), generator=g).float()
    check(x.to(dtype), x.argmax(1), 32, times=60)
    check(x.to(dtype), torch.randint(0, V, (6,), generator=g), 5, times=60)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('temperature', [1e-9, 1e-6, 0.01, 0.5, 1.5, 2.0, 2.5, 100.0, 1e9, 1e15, 1e29, 1e35])
def test_masked_rows_at_any_temperature(temperature, dtype):
    """A masked id has probability 0 at each, by -inf or by the type's lowest value; the entropy is a number."""
    g = torch.Generator().manual_seed(int(1e3 * temperature) % 1000)
    for V in (20, 333, 2049):
        x = 2 * torch.randn(6, V, generator=g).to(dtype)
        t = x.argmax(1)
        t[1::2] = torch.randint(0, V, (3,), generator=g)
        if temperature < 1e30:                               # (the lowest value itself counts at temperatures near it)
            x[3:, V // 3:V // 2] = torch.finfo(dtype).min
        x[:, :V // 4] = float('-inf')
        x[:, -1] = float('-inf')
        x[2, ::2] = float('-inf')
        check_far(x, t, 0, temperature)
        check_far(x, t, 5, temperature)


@pytest.mark.parametrize('V,dtype', [(333, torch.float32), (2049, torch.float32), (4099, torch.bfloat16)])
@pytest.mark.parametrize('temperature', [0.01, 0.7, 1.0, 1.5, 2.0, 2.5, 50.0])
def test_masked_ids_leave_the_bits_of_any_far_logit(temperature, V, dtype):
    """-inf and a logit of -10^4 and less add exactly 0 to every sum, so that the rows' bits are equal: all of them in one
    pass, or a last bit would differ here and there."""
    from flashb.sampling import token_scores
    g = torch.Generator().manual_seed(V)
    x = 2 * torch.randn(64, V, generator=g).to(dtype)
    t = torch.randint(V // 4, V - 1, (64,), generator=g).cuda()
    got = []
    for mask in (-1e4, float('-inf'), -1e6, -1e10, -1e15, -1e25, torch.finfo(dtype).min):
        x[:, :V // 5] = mask
        x[:, -1] = mask
        x[::3, V // 2] = mask
        got.append(token_scores(x.cuda(), t, top=5, temperature=temperature))
    some = (t != V // 2)
    for other in got[1:]:
        for name, a, b in zip(other._fields, got[0], other):
            assert torch.equal(a[some], b[some]), name


@pytest.mark.parametrize('temperature', [1.0, 2.0, 4.0, 1e20, 1e38])
def test_differences_past_the_largest_number(temperature):
    """Logits of both ends of fp32: their difference is past its range, divided by the temperature it need not be."""
    x = torch.tensor([[3e38, -3e38, 1e38, 0.0, 2.9e38, 3e38], [-3e38, -3.2e38, -3.1e38, -3e38, 3.4e38, 0.0]])
    if temperature < 2:
        x = x / 2
    for t in ([1, 1], [3, 0], [0, 4]):
        check_far(x, torch.tensor(t), 6, temperature)


def test_the_lowest_number_below_a_large_logit():
    """... on the fast path: its limit is on the largest logit's exponent alone."""
    x = torch.randn(3, 700, generator=torch.Generator().manual_seed(1)) * 1e35
    x[:, 5] = -MAX
    x[:, 600] = 2e36
    check_far(x, torch.tensor([5, 600, 7]), 9, 2e28)
    check_far(x.bfloat16(), torch.tensor([5, 600, 7]), 9, 2e28)
