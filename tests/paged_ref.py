"""The paged operators and the token scores from their definitions, in 64 bits on the CPU, a token at a time."""
import math
from fractions import Fraction

import torch

D = 128


def runs(lengths, offsets):
    """[(row, token, slot)] of a step."""
    out = []
    for b, n in enumerate(lengths.tolist()):
        lo, hi = (b, b + 1) if offsets is None else (int(offsets[b]), int(offsets[b + 1]))
        out += [(b, t, n - (hi - t)) for t in range(lo, hi)]
    return out


def page_of(table, b, slot, page, pages):
    """The page of a row's slot, None where there is none."""
    if slot < 0 or slot >= table.shape[1] * page:
        return None
    e = int(table[b, slot // page])
    return e if 0 <= e < pages else None


TURN = Fraction('6.28318530717958647692528676655900576839433879875021')


def angle(pos, freq):
    """pos x freq radians less its whole turns: an exact product, so that far positions keep their angle."""
    return float(Fraction(pos) * Fraction(float(freq)) % TURN)


def rotate(x, pos, freq, layout, amplitude):
    """x [heads, 128] (64 bits) at one position."""
    half = len(freq)
    y = x.clone()
    for i in range(half):
        p, m = (i, i + half) if layout == 'half' else (2 * i, 2 * i + 1)
        t = angle(pos, freq[i])
        y[:, p] = amplitude * (x[:, p] * math.cos(t) - x[:, m] * math.sin(t))
        y[:, m] = amplitude * (x[:, m] * math.cos(t) + x[:, p] * math.sin(t))
    return y


def norm(x, w, eps):
    return x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def append(qkv, keys, values, table, lengths, offsets, freq, layout, amplitude, q_norm, k_norm, eps, positions):
    """(q [T, NH, 128] with NaN where no token is, keys, values) in 64 bits."""
    pages, NKV, page, _ = keys.shape
    T = qkv.shape[0]
    x = qkv.double().view(T, -1, D)
    NH = x.shape[1] - 2 * NKV
    q = torch.full((T, NH, D), float('nan'), dtype=torch.float64)
    K, V = keys.double(), values.double()
    for b, t, slot in runs(lengths, offsets):
        pos = slot if positions is None else int(positions[t])
        q[t] = rotate(norm(x[t, :NH], q_norm, eps), pos, freq, layout, amplitude)
        e = page_of(table, b, slot, page, pages)
        if e is not None:
            K[e, :, slot % page] = rotate(norm(x[t, NH:NH + NKV], k_norm, eps), pos, freq, layout, amplitude)
            V[e, :, slot % page] = x[t, NH + NKV:]
    return q, K, V


def attend(q, keys, values, table, lengths, offsets, window=None, sinks=0, scaling=D ** -0.5):
    """(out [T, NH, 128], sum_j p_j |v_j| of each) in 64 bits; NaN where no token is."""
    pages, NKV, page, _ = keys.shape
    T, NH, _ = q.shape
    G = NH // NKV
    out = torch.full((T, NH, D), float('nan'), dtype=torch.float64)
    size = out.clone()
    S = table.shape[1] * page
    lengths = lengths.clamp(0, S)
    entries = {}
    for b, t, p in runs(lengths, offsets):
        if b not in entries:
            e = table[b].long().repeat_interleave(page)
            slot = torch.arange(S)
            there = (e >= 0) & (e < pages)
            entries[b] = (e, slot, there)
        e, slot, there = entries[b]
        see = there & (slot <= p)
        if window is not None:
            see &= (slot > p - window) | (slot < sinks)
        j = slot[see]
        if j.numel() == 0:
            out[t] = size[t] = 0
            continue
        k = keys[e[j], :, j % page].double().repeat_interleave(G, 1)         # [n, NH, D]
        v = values[e[j], :, j % page].double().repeat_interleave(G, 1)
        z = torch.einsum('hd,nhd->hn', q[t].double(), k) * scaling
        w = torch.softmax(z, -1)
        out[t], size[t] = torch.einsum('hn,nhd->hd', w, v), torch.einsum('hn,nhd->hd', w, v.abs())
    return out, size


def scores(logits, tokens, top, temperature):
    """(logprob, entropy, rank, ids, logprobs) of each row."""
    got = []
    for x, tok in zip(logits.double(), tokens.tolist()):
        V = x.numel()
        order = sorted(range(V), key=lambda i: (0, 0.0, i) if math.isnan(x[i]) else (1, -float(x[i]), i))
        bad = bool(torch.isnan(x).any()) or float(x.max()) in (math.inf, -math.inf)
        nan = float('nan')
        # the temperature as the library takes it: fp32
        z = x / float(torch.tensor(temperature, dtype=torch.float32))
        if bad:
            lp = torch.full((V,), nan, dtype=torch.float64)
        else:
            # from the largest, its own 1 apart: max + log(sum) would round an almost certain token's away
            lp = z - z[order[0]]
            lp = lp - torch.log1p(lp.exp()[order[1:]].sum())
        p = lp.exp()
        h = nan if bad else float(-torch.where(p > 0, p * lp, torch.zeros_like(p)).sum())
        inside = 0 <= tok < V
        got.append((float(lp[tok]) if inside else (nan if bad else -math.inf), h, order.index(tok) if inside else V,
                    order[:top], [float(lp[i]) for i in order[:top]]))
    lp, h, rank, ids, tl = zip(*got)
    return (torch.tensor(lp, dtype=torch.float64), torch.tensor(h, dtype=torch.float64), torch.tensor(rank),
            torch.tensor(ids).view(len(got), top), torch.tensor(tl, dtype=torch.float64).view(len(got), top))
