"""Token scores on the GPU where it can go wrong: what few warps work out for a row, masks at every temperature."""
import pytest
import torch

from test_gpu_scores import check

pytestmark = pytest.mark.gpu


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
