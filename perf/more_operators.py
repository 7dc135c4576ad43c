"""Measured cases of the paged operators (``flashb.paged``) and of the token scores (``flashb.sampling``): rotary positions
with the write into a paged cache, attention of a chunk of new tokens over it, log probabilities of given tokens.

``run`` computes each operator in plain torch operations (``own`` false) or calls the library (``own`` true); ``exact``
gives the same outputs from the definitions in 64 bits.

A cache is a pool of pages of ``page`` slots; slot j of row b lies in page table[b, j // page].  ``offsets`` [rows + 1]
cuts the step's tokens into one run per row (None: one token a row), and row b's run ends at slot lengths[b] - 1.  The
token at slot p sees slot j when j <= p and (j > p - window or j < sinks).
"""
import math
import os
import sys

import torch

own = False

D = 128
HEADS = ((16, 4), (8, 2), (8, 8), (16, 8), (16, 2))  # (query heads, key/value heads): the backbone's, the depth model's, others
EPS = 1e-6


def _lib(name):
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'breeze-tts-2-flash_b200')
    if root not in sys.path:
        sys.path.insert(0, root)
    import importlib
    return importlib.import_module('flashb.' + name)


# ------------------------------------------------------------------------------------------------------------- cases
# mix: how a step's n tokens fall on its rows.  single: one each; even: n / rows each; one: the first row takes all but one
# token a row (its prompt's chunk beside the others' next tokens); ragged: cut at random, rows without a token among them.
# ctx: slots that a row holds before the step; rows differ (uniform up to ctx) where there are more than two.
def listed():
    return [
        # the new token of one stream (a conditional / unconditional pair): pure latency
        dict(name='append_one', op='append', b=2, n=2, mix='single', nh=16, nkv=4, page=64, ctx=700, rot=128,
             layout='half', scale='none', norm=1),
        # the new tokens of 64 streams, far positions of a long reading, interpolated frequencies
        dict(name='append_many', op='append', b=128, n=128, mix='single', nh=16, nkv=4, page=16, ctx=200000, rot=128,
             layout='half', scale='yarn', norm=1),
        # eight prompts of odd lengths at once, half of each head rotated, interleaved pairs, no norm
        dict(name='append_prompts', op='append', b=8, n=16391, mix='ragged', nh=16, nkv=4, page=64, ctx=0, rot=64,
             layout='interleaved', scale='linear', norm=0),
        # one stream's next token over its pages
        dict(name='decode_one', op='attend', b=2, n=2, mix='single', nh=16, nkv=4, page=16, ctx=2048, window=0, sinks=0),
        # 64 streams of different ages
        dict(name='decode_many', op='attend', b=128, n=128, mix='single', nh=16, nkv=4, page=64, ctx=8191, window=0,
             sinks=0),
        # a short prompt of one stream
        dict(name='chunk_short', op='attend', b=2, n=394, mix='even', nh=16, nkv=4, page=64, ctx=0, window=0, sinks=0),
        # a chunk of a prompt beside the next tokens of 31 streams
        dict(name='chunk_mixed', op='attend', b=64, n=575, mix='one', nh=16, nkv=4, page=64, ctx=8000, window=0, sinks=0),
        # a few tokens each, on a sliding window with first tokens that stay
        dict(name='chunk_window', op='attend', b=32, n=801, mix='ragged', nh=16, nkv=4, page=16, ctx=12000, window=2048,
             sinks=4),
        # a long chunk of a long text
        dict(name='chunk_long', op='attend', b=1, n=2048, mix='even', nh=16, nkv=4, page=128, ctx=32768, window=0, sinks=0),
        # one frame of one stream: the backbone's and the depth model's codebooks
        dict(name='scores_frame', op='scores', rows=17, v=2049, dtype='float32', top=4, temperature=1.0, masked=1),
        # a frame of 64 streams, every codebook
        dict(name='scores_many', op='scores', rows=1088, v=2049, dtype='float32', top=8, temperature=0.9, masked=1),
        # a batch of given readings over a text vocabulary
        dict(name='scores_text', op='scores', rows=4095, v=32003, dtype='bfloat16', top=20, temperature=1.0, masked=0),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(('append', 'attend', 'attend', 'scores'))
    most = max(_cost(c) for c in listed() if c['op'] == op)
    while True:
        if op == 'scores':
            c = dict(op=op, rows=_log(rng, 1, 16384), v=_log(rng, 33, 65536), dtype=rng.choice(('float32', 'bfloat16')),
                     top=rng.choice((0, 1, 5, 8, 20, 32)), temperature=rng.choice((1.0, 1.0, 0.9, 0.6, 1.3)),
                     masked=rng.randrange(2))
        else:
            nh, nkv = rng.choice(HEADS)
            b = _log(rng, 1, 128)
            mix = rng.choice(('single', 'even', 'one', 'ragged'))
            n = b if mix == 'single' else b * _log(rng, 1, max(1, 4096 // b)) if mix == 'even' else _log(rng, b, 4096)
            c = dict(op=op, b=b, n=n, mix=mix, nh=nh, nkv=nkv, page=rng.choice((16, 32, 64, 128, 256)))
            if op == 'append':
                c.update(ctx=_log(rng, 1, 30000), rot=rng.choice((128, 128, 96, 64, 32)),
                         layout=rng.choice(('half', 'interleaved')), scale=rng.choice(('none', 'linear', 'yarn')),
                         norm=rng.randrange(2))
            else:
                window = rng.choice((0, 0, _log(rng, 1, 8192)))
                c.update(ctx=_log(rng, 1, 32768), window=window, sinks=rng.choice((0, 1, 4, 33, 64)) if window else 0)
        if _cost(c) <= most:
            return c


def _cost(c):
    w = work(c)
    if c['op'] == 'scores':
        return w['bytes']
    pool = c['b'] * _slots(c) * c['nkv']
    if c['op'] == 'append':
        return w['bytes'] + 0.1 * pool                          # the pool is compared whole
    # the plain form's large arrays as well
    return w['bytes'] + w['flops'] / 100 + 256 * pool + 2 * c['n'] * c['nh'] * _slots(c)


def _slots(c):
    """Slots that a row's list of pages has."""
    if c['op'] == 'append':                                     # the pool holds the last pages alone
        return c['page'] * (2 + c['n'] // c['page'] // c['b'])
    return -(-(c['ctx'] + c['n']) // c['page']) * c['page']


def _pasts(c):
    """What rows hold before the step, evenly over their distribution."""
    return [c['ctx']] if c['b'] <= 2 else [c['ctx'] * (i + 0.5) / 32 for i in range(32)]


def work(c):
    op = c['op']
    if op == 'scores':
        size = 4 if c['dtype'] == 'float32' else 2
        return dict(bytes=c['rows'] * (c['v'] * size + 8 + 16 + 12 * c['top']), flops=c['rows'] * c['v'] * 5)
    b, n, nh, nkv = c['b'], c['n'], c['nh'], c['nkv']
    if op == 'append':                                          # q, k, v in; q out, k and v into the cache
        return dict(bytes=n * (nh + 2 * nkv) * D * 4, flops=n * (nh + nkv) * D * 6)
    counts = [n / b] * b if c['mix'] != 'one' else [n - b + 1] + [1] * (b - 1)
    seen = keys = 0.0
    for m in set(counts):
        for past in _pasts(c):
            share = counts.count(m) / len(_pasts(c))
            at = torch.arange(max(1, round(m)), dtype=torch.float64) + past + 1     # slots up to each token
            vis = at if not c['window'] else torch.minimum(at, c['window'] + (at - c['window']).clamp(0, c['sinks']))
            seen += share * float(vis.mean()) * m
            keys += share * min(past + m, c['window'] + m + c['sinks'] if c['window'] else past + m)
    return dict(bytes=2 * n * nh * D * 2 + keys * nkv * 4 * D, flops=4 * D * nh * seen)


# ------------------------------------------------------------------------------------------------------------ inputs
def _counts(c, g):
    b, n = c['b'], c['n']
    if c['mix'] in ('single', 'even'):
        return [n // b] * b
    if c['mix'] == 'one':
        return [n - b + 1] + [1] * (b - 1)
    cut = torch.randint(0, n + 1, (b - 1,), generator=g, device='cuda').sort().values.tolist()
    return [y - x for x, y in zip([0] + cut, cut + [n])]


def _rope(c):
    """Radians per position [rot / 2] (64 bits, on the host) and the amplitude: base 10^6; linear: positions divided by 4;
    yarn: 8 times the 32768 positions of training, frequencies of 32 turns and more in them kept, of one turn or less
    divided, a ramp between."""
    half = c['rot'] // 2
    freq = torch.tensor([1e6 ** (-i / half) for i in range(half)], dtype=torch.float64)
    if c['scale'] == 'linear':
        return freq / 4, 1.0
    if c['scale'] == 'yarn':
        at = [c['rot'] * math.log(32768 / (2 * math.pi * turns)) / (2 * math.log(1e6)) for turns in (32, 1)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), c['rot'] - 1)
        ramp = ((torch.arange(half, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return freq * (1 - ramp) + freq / 8 * ramp, 0.1 * math.log(8) + 1
    return freq, 1.0


def prepare(case, seed):
    c = dict(case)
    dev = 'cuda'
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    st = dict(case=c)
    if c['op'] == 'scores':
        rows, v = c['rows'], c['v']
        # logits of a trained head: unit noise around a common slope, a few ids far ahead; the last ids may be suppressed
        x = torch.randn(rows, v, generator=g, device=dev) - 3 * torch.rand(v, generator=g, device=dev)
        gone = max(1, v // 512) if c['masked'] else 0
        peak = torch.randint(0, v - gone, (rows, 4), generator=g, device=dev)
        far, at = 12 * torch.rand(rows, 4, generator=g, device=dev), torch.arange(rows, device=dev)
        for i in range(4):
            x[at, peak[:, i]] += far[:, i]
        if gone:
            x[:, v - gone:] = float('-inf')
        st['logits'] = x.to(getattr(torch, c['dtype']))
        if own:
            st['lib'] = _lib('sampling')
        # most given tokens are likely ones
        any_id = torch.randint(0, v - gone, (rows,), generator=g, device=dev)
        st['tokens'] = torch.where(torch.rand(rows, generator=g, device=dev) < 0.8, peak[:, 0], any_id)
        return st
    b, n, nh, nkv, page = c['b'], c['n'], c['nh'], c['nkv'], c['page']
    counts = _counts(c, g)
    past = [c['ctx']] * b if b <= 2 else torch.randint(0, c['ctx'] + 1, (b,), generator=g, device=dev).tolist()
    spans = [(p, p + m) for p, m in zip(past, counts)]          # the slots of each row's new tokens
    width = -(-(c['ctx'] + n) // page)
    st['spans'] = spans
    st['lengths'] = torch.tensor([e for _, e in spans], dtype=torch.int64, device=dev)
    cut = [0]
    for m in counts:
        cut.append(cut[-1] + m)
    st['offsets'] = None if c['mix'] == 'single' else torch.tensor(cut, dtype=torch.int64, device=dev)
    # pages in use are spread over the pool; of an append's rows only those that the step writes are there
    first = [s // page if c['op'] == 'append' else 0 for s, _ in spans]
    need = [-(-e // page) - f for f, (_, e) in zip(first, spans)]
    pages = b * width if c['op'] == 'attend' else n // page + 2 * b
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.full((b, width), -1, dtype=torch.int32)
    used = 0
    for r in range(b):
        table[r, first[r]:first[r] + need[r]] = order[used:used + need[r]]
        used += need[r]
    st['table'] = table.to(dev)
    if c['op'] == 'append':
        st['keys'], st['values'] = (torch.zeros(pages, nkv, page, D, dtype=torch.bfloat16, device=dev)
                                    for _ in range(2))
        st['qkv'] = torch.randn(n, (nh + 2 * nkv) * D, generator=g, device=dev).to(torch.bfloat16)
        st['q_norm'], st['k_norm'] = (((1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16)
                                       for _ in range(2)) if c['norm'] else (None, None))
        freq, st['amplitude'] = _rope(c)
        st['freq'] = freq.to(dev)
        if own:
            st['lib'] = lib = _lib('paged')
            scale = dict(none=None, linear=dict(kind='linear', factor=4.0),
                         yarn=dict(kind='yarn', factor=8.0, original=32768))[c['scale']]
            st['rotary'] = lib.Rotary(c['rot'], base=1e6, layout=c['layout'], scaling=scale)
            st['cache'] = lib.PagedCache(st['keys'], st['values'])
        return st
    # keys as the k norm leaves them, the first slots drawing attention as a trained model's do
    u = torch.randn(nkv, 1, D, generator=g, device=dev)
    u = u / u.square().mean(-1, keepdim=True).sqrt()
    k = torch.randn(pages, nkv, page, D, generator=g, device=dev, dtype=torch.bfloat16)
    v = torch.randn(pages, nkv, page, D, generator=g, device=dev, dtype=torch.bfloat16)
    head = st['table'][:, 0].long()
    head = head[head >= 0]
    k[head, :, :4] = (0.5 * k[head, :, :4].float() + 0.5 * u).to(torch.bfloat16)
    q = torch.randn(n, nh, D, generator=g, device=dev)
    st['q'] = (q + 0.3 * u.view(1, nkv, 1, D).expand(1, nkv, nh // nkv, D).reshape(1, nh, D)).to(torch.bfloat16)
    st['keys'], st['values'] = k, v
    if own:
        st['lib'] = _lib('paged')
        st['cache'] = st['lib'].PagedCache(k, v)
    return st


# -------------------------------------------------------------------------------------------------------- plain form
def _plain_append(st):
    c = st['case']
    nh, nkv, rot, page = c['nh'], c['nkv'], c['rot'], c['page']
    x = st['qkv'].float().view(c['n'], nh + 2 * nkv, D)
    slot = torch.cat([torch.arange(s, e, device='cuda') for s, e in st['spans']])
    row = torch.cat([torch.full((e - s,), r, device='cuda') for r, (s, e) in enumerate(st['spans'])])
    turn = slot.double()[:, None] * st['freq'] / (2 * math.pi)
    angle = (2 * math.pi * (turn - turn.round())).float()
    cos, sin = angle.cos()[:, None] * st['amplitude'], angle.sin()[:, None] * st['amplitude']

    def turned(h, w):
        if w is not None:
            h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.float()
        a, rest = h[..., :rot], h[..., rot:]
        if c['layout'] == 'half':
            p, m = a[..., :rot // 2], a[..., rot // 2:]
            a = torch.cat((p * cos - m * sin, m * cos + p * sin), -1)
        else:
            p, m = a[..., 0::2], a[..., 1::2]
            a = torch.stack((p * cos - m * sin, m * cos + p * sin), -1).flatten(-2)
        return torch.cat((a, rest), -1).to(torch.bfloat16)
    q = turned(x[:, :nh], st['q_norm'])
    at = st['table'][row, slot // page].long()
    st['keys'][at, :, slot % page] = turned(x[:, nh:nh + nkv], st['k_norm'])
    st['values'][at, :, slot % page] = x[:, nh + nkv:].to(torch.bfloat16)
    return q, st['keys'], st['values']


def _attention(q, k, v, p, c):
    """q [.., nh, n, D] of tokens at slots p [.., n] over k / v [.., nkv, s, D]."""
    nh, n = q.shape[-3:-1]
    nkv, s = k.shape[-3:-1]
    j = torch.arange(s, device='cuda')
    seen = j <= p[..., None]
    if c['window']:
        seen &= (j > p[..., None] - c['window']) | (j < c['sinks'])
    z = torch.matmul(q.float().reshape(q.shape[:-3] + (nkv, nh // nkv * n, D)), k.float().transpose(-1, -2))
    z = z.mul_(D ** -0.5).view(q.shape[:-3] + (nkv, nh // nkv, n, s))
    z.masked_fill_(~seen[..., None, None, :, :], float('-inf'))
    top = z.amax(-1, keepdim=True)
    z.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = z.sum(-1, keepdim=True)
    z.div_(torch.where(total == 0, torch.ones_like(total), total))
    return torch.matmul(z.view(q.shape[:-3] + (nkv, nh // nkv * n, s)), v.float()).view(q.shape).to(torch.bfloat16)


def _plain_attend(st):
    c = st['case']
    q, table = st['q'], st['table'].clamp(min=0)
    if c['mix'] == 'single':
        k, v = (st[x][table.long()].transpose(1, 2).flatten(2, 3) for x in ('keys', 'values'))
        return _attention(q.view(c['b'], c['nh'], 1, D), k, v, st['lengths'][:, None] - 1, c).view(q.shape)
    out = torch.empty_like(q)
    t = 0
    for r, (s, e) in enumerate(st['spans']):
        if e > s:
            at = table[r, :-(-e // c['page'])].long()
            k, v = (st[x][at].transpose(0, 1).flatten(1, 2)[:, :e] for x in ('keys', 'values'))
            p = torch.arange(s, e, device='cuda')
            out[t:t + e - s] = _attention(q[t:t + e - s].transpose(0, 1), k, v, p, c).transpose(0, 1)
            t += e - s
    return out


def _plain_scores(st):
    c = st['case']
    raw, tok = st['logits'].float(), st['tokens'][:, None]
    x = raw / c['temperature']
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    logz = total.log()
    entropy = logz[:, 0] - (e * x.masked_fill(e == 0, 0)).sum(-1) / total[:, 0]
    mine = raw.gather(1, tok)
    ids = torch.arange(c['v'], device='cuda')
    rank = ((raw > mine) | ((raw == mine) & (ids < tok))).sum(-1)
    best = torch.sort(raw, dim=-1, descending=True, stable=True).indices[:, :c['top']]
    return (x.gather(1, tok) - logz)[:, 0], entropy, rank, best, x.gather(1, best) - logz


def run(st):
    c = st['case']
    if not own:
        return dict(append=_plain_append, attend=_plain_attend, scores=_plain_scores)[c['op']](st)
    if c['op'] == 'append':
        q = st['lib'].append(st['qkv'], st['cache'], st['table'], st['lengths'], offsets=st['offsets'],
                             rotary=st['rotary'], q_norm=st['q_norm'], k_norm=st['k_norm'], eps=EPS)
        return q, st['keys'], st['values']
    if c['op'] == 'attend':
        return st['lib'].attend(st['q'], st['cache'], st['table'], st['lengths'], offsets=st['offsets'],
                                window=c['window'] or None, sinks=c['sinks'])
    return tuple(st['lib'].token_scores(st['logits'], st['tokens'], top=c['top'], temperature=c['temperature']))


# ----------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_append(st):
    c = st['case']
    nh, nkv, rot, page = c['nh'], c['nkv'], c['rot'], c['page']
    q = torch.zeros(c['n'], nh, D, dtype=torch.float64, device='cuda')
    keys, values = (torch.zeros(st['keys'].shape, dtype=torch.float64, device='cuda') for _ in range(2))
    freq, amp = _rope(c)
    # the pair of each rotated dim, and its sign in the product with the sine
    dim = torch.arange(D)
    if c['layout'] == 'half':
        lower = dim < rot // 2
        other, which = torch.where(lower, dim + rot // 2, dim - rot // 2), dim % max(rot // 2, 1)
    else:
        lower = dim % 2 == 0
        other, which = torch.where(lower, dim + 1, dim - 1), dim // 2
    turned = dim < rot
    other = torch.where(turned, other, dim).cuda()
    sign = torch.where(turned, torch.where(lower, -1.0, 1.0), 0.0).double().cuda()
    per = torch.where(turned, freq[which.clamp(max=rot // 2 - 1)], torch.zeros(())).cuda()
    gain = torch.where(turned, amp, 1.0).double().cuda()
    t = 0
    for r, (s, e) in enumerate(st['spans']):
        if e == s:
            continue
        h = st['qkv'][t:t + e - s].double().view(e - s, nh + 2 * nkv, D)
        p = torch.arange(s, e, device='cuda')
        angle = p.double()[:, None, None] * per

        def rotated(y, w):
            if w is not None:
                y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            return gain * (y * torch.cos(angle) + sign * y[..., other] * torch.sin(angle))
        q[t:t + e - s] = rotated(h[:, :nh], st['q_norm'])
        at = st['table'][r].long()[p // page]
        keys[at, :, p % page] = rotated(h[:, nh:nh + nkv], st['k_norm'])
        values[at, :, p % page] = h[:, nh + nkv:]
        t += e - s
    return q, keys, values


def _exact_attend(st):
    c = st['case']
    group = c['nh'] // c['nkv']
    out = torch.zeros(st['q'].shape, dtype=torch.float64, device='cuda')
    t = 0
    for r, (s, e) in enumerate(st['spans']):
        if e == s:
            continue
        at = st['table'][r, :-(-e // c['page'])].long()
        p = torch.arange(s, e, device='cuda')[:, None]
        j = torch.arange(e, device='cuda')[None]
        hidden = j > p
        if c['window']:
            hidden |= (p - j >= c['window']) & (j >= c['sinks'])
        for h in range(c['nkv']):
            k, v = (st[x][at, h].reshape(-1, D)[:e].double() for x in ('keys', 'values'))
            for i in range(h * group, h * group + group):
                z = st['q'][t:t + e - s, i].double() @ k.T / math.sqrt(D)
                out[t:t + e - s, i] = torch.softmax(z.masked_fill_(hidden, -math.inf), -1) @ v
        t += e - s
    return out


def _exact_scores(st):
    c = st['case']
    parts = []
    for x, tok in zip(st['logits'].split(512), st['tokens'].split(512)):
        logp = torch.log_softmax(x.double() / c['temperature'], -1)
        entropy = -torch.special.xlogy(logp.exp(), logp.exp()).sum(-1)
        order = torch.argsort(-x.double(), dim=-1, stable=True)
        rank = (order == tok[:, None]).int().argmax(-1)
        best = order[:, :c['top']]
        parts.append((logp.gather(1, tok[:, None])[:, 0], entropy, rank, best, logp.gather(1, best)))
    return tuple(torch.cat(p) for p in zip(*parts))


def exact(case, seed):
    st = prepare(case, seed)
    return dict(append=_exact_append, attend=_exact_attend, scores=_exact_scores)[case['op']](st)
