"""The long-speech operators from their definitions, in 64 bits on the CPU (plain loops over rows and heads)."""
import torch

D = 128
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def visible(p, start, S, window, sinks):
    """[S] bool: the slots the token at slot p sees."""
    j = torch.arange(S)
    m = (j >= start) & (j <= p)
    if window is not None:
        m &= (j > p - window) | (j < start + sinks)
    return m


def attend(q, k, v, m, scaling):
    """q [g, D], k / v [S, D], m [S] -> (out [g, D], weights [g, S], sum of p |v| [g, D]); only visible rows are read."""
    at = torch.nonzero(m).view(-1)
    w = torch.zeros(q.shape[0], m.numel(), dtype=torch.float64)
    if at.numel() == 0:
        z = torch.zeros(q.shape[0], D, dtype=torch.float64)
        return z, w, z.clone()
    s = q.double() @ k[at].double().T * scaling
    p = torch.softmax(s, -1)
    w[:, at] = p
    return p @ v[at].double(), w, p @ v[at].double().abs()


def decode(q, k, v, lengths, starts, window, sinks, scaling):
    """q [B, NH, 1, D], k / v [B, NKV, S, D] -> (out [B, 1, NH, D], weights [B, NKV, S], bound [B, 1, NH, D])."""
    B, NH = q.shape[:2]
    NKV, S = k.shape[1:3]
    g = NH // NKV
    out = torch.zeros(B, 1, NH, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    wt = torch.zeros(B, NKV, S, dtype=torch.float64)
    for b in range(B):
        n = max(0, min(int(lengths[b]), S))
        m = visible(n - 1, 0 if starts is None else max(0, int(starts[b])), S, window, sinks)
        for h in range(NKV):
            o, w, a = attend(q[b, h * g:h * g + g, 0], k[b, h], v[b, h], m, scaling)
            out[b, 0, h * g:h * g + g], mag[b, 0, h * g:h * g + g] = o, a
            wt[b, h] = w.sum(0)
    return out, wt, bound(out, mag)


def prefill(q, k, v, q_start, starts, window, sinks, scaling):
    B, NH, L = q.shape[:3]
    NKV, S = k.shape[1:3]
    g = NH // NKV
    out = torch.zeros(B, L, NH, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        for i in range(L):
            m = visible(q_start + i, 0 if starts is None else int(starts[b]), S, window, sinks)
            for h in range(NKV):
                o, _, a = attend(q[b, h * g:h * g + g, i], k[b, h], v[b, h], m, scaling)
                out[b, i, h * g:h * g + g], mag[b, i, h * g:h * g + g] = o, a
    # the weights are rounded to bf16 on the way: 2^-8 of sum p |v| at most
    return out, 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -12) * mag + 1e-30


def bound(out, mag):
    """How far a decode's bf16 output may be: half an ulp, 2^-8 of the output at most, here half as 2^-9 of the output
    and half as 2^-9 of sum p |v|, which is no less; and 2^-12 of sum p |v| for weights of 11 bits and more and for
    fp32 scores, exponentials and sums (ample for scores below 2^8)."""
    return 2.0 ** -9 * out.abs() + (2.0 ** -9 + 2.0 ** -12) * mag + 1e-30


def assert_within(got, ref, tol):
    off = (got.double().cpu() - ref).abs()
    assert torch.isfinite(off).all()
    worst = (off - tol).max().item()
    assert worst <= 0, f'off by up to {off.max().item():.3e}, {worst:.3e} over the bound'


def e4m3(x):
    """Nearest e4m3 value of x >= 0 (ties to even, saturated)."""
    x = x.clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(max=448.0)


def quantise(x, scale=1.0):
    """x [..., D] bf16 -> the values its 4-bit form stands for, in 64 bits."""
    b = (x.double() / scale).reshape(-1, 16)
    odd = ~torch.isfinite(b).all(1)
    b = torch.where(odd[:, None], torch.zeros_like(b), b)
    s = e4m3(b.abs().amax(1) / 6)
    a = torch.where(s[:, None] > 0, b.abs() / s.clamp(min=1e-30)[:, None], torch.zeros_like(b))
    d = (a.clamp(max=8.0)[..., None] - GRID).abs()              # far beyond 6 all distances would round alike
    best = d.argmin(-1)                                         # the lower neighbour at a tie
    up = (best + 1).clamp(max=7)
    tie = d.gather(-1, up[..., None]) == d.gather(-1, best[..., None])
    best = torch.where(tie[..., 0] & (best % 2 == 1), up, best)
    y = torch.copysign(GRID[best] * s[:, None], b) * scale
    y[odd] = float('nan')
    return y.reshape(x.shape)


def evict(acc, lengths, starts, keep, sinks, recent):
    """kept [B, NKV, keep] (-1 beyond), lengths [B]."""
    B, NKV, S = acc.shape
    kept = torch.full((B, NKV, keep), -1, dtype=torch.int32)
    n_out = torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        hi = max(0, min(int(lengths[b]), S))
        lo = min(hi, 0 if starts is None else max(0, int(starts[b])))
        n = hi - lo
        n_out[b] = min(n, keep)
        for h in range(NKV):
            rows = list(range(lo, hi))
            if n > keep:
                mid = rows[sinks:n - recent]
                key = lambda j: float('inf') if acc[b, h, j] != acc[b, h, j] else float(acc[b, h, j])  # noqa: E731
                nan = lambda j: not (acc[b, h, j] != acc[b, h, j])  # noqa: E731
                best = sorted(mid, key=lambda j: (nan(j), -key(j), j))[:keep - sinks - recent]
                rows = sorted(rows[:sinks] + best + (rows[n - recent:] if recent else []))
            kept[b, h, :len(rows)] = torch.tensor(rows, dtype=torch.int32)
    return kept, n_out
