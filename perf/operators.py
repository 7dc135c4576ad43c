"""Measured cases of the long-speech operators (``flashb.longform``): attention with a sliding window and sink tokens,
a KV cache held in 4 bits, and eviction from a cache by accumulated attention weight.

``run`` computes each operator in plain torch operations (``own`` false) or calls the library (``own`` true); ``exact``
gives the same outputs from the definitions in 64 bits.

Row b of a cache holds its keys in slots [start_b, len_b); the token at slot p sees slot j when start_b <= j <= p and
(j > p - window or j < start_b + sinks).  A token without a visible key gives 0.
"""
import math
import os
import sys

import torch

own = False

D = 128
LUT = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)      # the magnitudes of a 4-bit e2m1 value
HEADS = ((16, 4), (8, 2), (8, 8), (16, 8), (16, 2))  # (query heads, key/value heads): the backbone's, the depth model's, others


def _lib():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'breeze-tts-2-flash_b200')
    if root not in sys.path:
        sys.path.insert(0, root)
    from flashb import longform
    return longform


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one stream (a conditional / unconditional pair) late in a long reading, on a short window: pure latency
        dict(name='window_decode_one', op='window_decode', b=2, nh=16, nkv=4, s=2048, window=512, sinks=4, pad=1),
        # 64 streams of different ages in one step, the window's bytes beyond L2
        dict(name='window_decode_many', op='window_decode', b=128, nh=16, nkv=4, s=4096, window=2048, sinks=4, pad=1),
        # a short ragged prompt of one stream, left padded
        dict(name='window_prefill_short', op='window_prefill', b=2, nh=16, nkv=4, l=197, past=0, window=128, sinks=4,
             pad=1),
        # a long text prompt in one pass
        dict(name='window_prefill_long', op='window_prefill', b=1, nh=16, nkv=4, l=8192, past=0, window=1024, sinks=4,
             pad=0),
        # the new token of 64 streams goes into the 4-bit cache and is read back
        dict(name='kv4_store_token', op='kv4_store', b=128, nh=16, nkv=4, s=2048, l=1),
        # the prompts of 8 rows go into the 4-bit cache and are read back for the prompt's own attention
        dict(name='kv4_store_prompt', op='kv4_store', b=8, nh=16, nkv=4, s=4500, l=4097),
        # one stream over its 4-bit cache
        dict(name='kv4_decode_one', op='kv4_decode', b=2, nh=16, nkv=4, s=2741, pad=0),
        # 32 streams of different ages over long 4-bit caches
        dict(name='kv4_decode_many', op='kv4_decode', b=64, nh=16, nkv=4, s=8192, pad=1),
        # one stream, the attention weight of each slot added up for a later eviction
        dict(name='scored_decode_one', op='scored_decode', b=2, nh=16, nkv=4, s=1000, pad=0),
        # 32 streams, the same
        dict(name='scored_decode_many', op='scored_decode', b=64, nh=16, nkv=4, s=4096, pad=1),
        # one stream's cache halved
        dict(name='evict_one', op='evict', b=2, nh=16, nkv=4, s=2048, keep=1023, sinks=4, recent=256, pad=0),
        # 32 streams' caches cut to a quarter at once
        dict(name='evict_many', op='evict', b=64, nh=16, nkv=4, s=8192, keep=2048, sinks=4, recent=512, pad=1),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(('window_decode', 'window_prefill', 'kv4_store', 'kv4_decode', 'scored_decode', 'evict'))
    most = max(_cost(c) for c in listed() if c['op'] == op)
    while True:
        nh, nkv = rng.choice(HEADS)
        c = dict(op=op, b=_log(rng, 1, 128), nh=nh, nkv=nkv)
        if op == 'window_decode':
            c.update(s=_log(rng, 16, 16384), window=_log(rng, 1, 8192), sinks=rng.choice((0, 1, 4, 33, 64)))
        elif op == 'window_prefill':
            c.update(l=_log(rng, 1, 8192), past=rng.choice((0, 0, _log(rng, 1, 4096))), window=_log(rng, 16, 8192),
                     sinks=rng.choice((0, 1, 4, 33, 64)))
        elif op == 'kv4_store':
            l = _log(rng, 1, 8192)
            c.update(s=l + rng.randrange(0, 512), l=l)
        elif op in ('kv4_decode', 'scored_decode'):
            c.update(s=_log(rng, 16, 16384))
        else:
            s = _log(rng, 64, 16384)
            keep = rng.randrange(s // 8 + 2, s)
            sinks = rng.choice((0, 1, 4))
            c.update(s=s, keep=keep, sinks=min(sinks, keep), recent=rng.randrange(0, max(1, keep - 4)))
        if op != 'kv4_store':
            c.update(pad=rng.randrange(2))
        if _cost(c) <= most:
            return c


def _cost(c):
    w = work(c)
    # the plain form's large arrays as well: every query against every key of a prefill, every slot of a cache
    if c['op'] == 'window_prefill':
        return c['b'] * c['nh'] * c['l'] * (c['l'] + c['past'])
    return w['bytes'] + 512 * c['b'] * c['nkv'] * c['s']


def _mean_keys(c):
    """Mean visible keys of a row whose length is uniform in [1, s]."""
    s = c['s']
    cap = min(s, c['window'] + c['sinks']) if 'window' in c else s
    return (cap * (cap + 1) / 2 + (s - cap) * cap) / s


def work(c):
    b, nh, nkv = c['b'], c['nh'], c['nkv']
    op = c['op']
    io = 2 * b * nh * D * 2                                    # q in, out out
    if op in ('window_decode', 'scored_decode', 'kv4_decode'):
        keys = b * nkv * _mean_keys(c)
        per = 4 * D if op != 'kv4_decode' else 2 * (D // 2 + D // 16)
        extra = 8 * b * nkv * c['s'] if op == 'scored_decode' else 0
        return dict(bytes=keys * per + io + extra, flops=4 * D * keys * (nh // nkv))
    if op == 'window_prefill':
        n, past, w, sk = c['l'], c['past'], c['window'], c['sinks']
        p = torch.arange(past, past + n, dtype=torch.float64)
        win = torch.clamp(p + 1, max=float(w))
        seen = float((win + torch.clamp(torch.minimum(p + 1 - win, torch.tensor(float(sk), dtype=torch.float64)),
                                        min=0)).sum())
        keys = min(past + n, w + n + sk)
        return dict(bytes=io * n + 4 * D * b * nkv * keys, flops=4 * D * b * nh * seen)
    if op == 'kv4_store':
        rows = 2 * b * nkv * c['l']
        # read bf16, write codes and scales; read codes and scales, write bf16
        return dict(bytes=rows * 2 * (2 * D + D // 2 + D // 16), flops=rows * D * 4)
    # a row shorter than `keep` moves as it is; lengths as in _ages
    s, keep = c['s'], c['keep']
    live = s - s // 16 if b <= 2 else (s + 1) / 2
    rows = min(live, keep) if b <= 2 else keep - keep * (keep - 1) / (2 * s)
    return dict(bytes=b * nkv * (2 * rows * 2 * 2 * D + 4 * live + 8 * keep), flops=b * nkv * live)


# ------------------------------------------------------------------------------------------------------------ inputs
def _heads(c, g, n, q_len=1):
    """Queries, keys and values as the q/k norms leave them (unit variance), the first tokens of each row drawing
    attention as the sinks of a trained model do."""
    dev = 'cuda'
    b, nh, nkv = c['b'], c['nh'], c['nkv']
    u = torch.randn(1, nkv, 1, D, generator=g, device=dev)
    u = u / u.square().mean(-1, keepdim=True).sqrt()
    k = torch.randn(b, nkv, n, D, generator=g, device=dev, dtype=torch.bfloat16)
    v = torch.randn(b, nkv, n, D, generator=g, device=dev, dtype=torch.bfloat16)
    k[:, :, :4] = (0.5 * k[:, :, :4].float() + 0.5 * u).to(torch.bfloat16)
    q = torch.randn(b, q_len, nh, D, generator=g, device=dev)
    q = (q + 0.3 * u.view(1, 1, nkv, 1, D).expand(1, 1, nkv, nh // nkv, D).reshape(1, 1, nh, D)).to(torch.bfloat16)
    return q.transpose(1, 2), k, v                              # q [b, nh, q_len, D], a view as projections give it


def _ages(c, g):
    """Lengths of rows of different ages, and the left padding of their prompts."""
    b, s = c['b'], c['s']
    if b <= 2:
        length = torch.full((b,), s - s // 16, dtype=torch.int64, device='cuda')
    else:
        length = torch.randint(1, s + 1, (b,), generator=g, device='cuda')
        length[0] = s
    start = None
    if c.get('pad'):
        start = torch.randint(0, 1 + max(1, s // 64), (b,), generator=g, device='cuda')
    return length, start


def _split4(x):
    """The e2m1 codes (two per byte, the even element in the low half) and e4m3 block scales of x [..., D], as bytes."""
    blk = x.float().unflatten(-1, (D // 16, 16))
    s8 = (blk.abs().amax(-1) / 6).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = s8.float().unsqueeze(-1)
    a = blk.abs()
    code = sum(((a > t * s) if n % 2 == 0 else (a >= t * s)).to(torch.uint8)
               for n, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code = torch.where(s > 0, code | ((blk < 0).to(torch.uint8) << 3), torch.zeros_like(code)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), s8.view(torch.uint8)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    op = c['op']
    st = dict(case=c, scaling=D ** -0.5)
    if op == 'window_prefill':
        n, past = c['l'], c['past']
        q, k, v = _heads(c, g, past + n, n)
        st.update(q=q, k=k, v=v, past=past)
        st['start'] = torch.randint(0, 1 + min(16, n - 1), (c['b'],), generator=g, device='cuda') if c['pad'] else None
        return st
    if op == 'kv4_store':
        _, k, v = _heads(c, g, c['l'])
        length = torch.randint(0, c['s'] - c['l'] + 1, (c['b'], 1), generator=g, device='cuda')
        st.update(k=k, v=v, slots=length + torch.arange(c['l'], device='cuda'))
        if own:
            st['cache'] = _lib().KV4Cache.empty(c['b'], c['nkv'], c['s'])
        return st
    q, k, v = _heads(c, g, c['s'])
    length, start = _ages(c, g)
    st.update(q=q, length=length, start=start)
    if op == 'kv4_decode':
        kq, ks = _split4(k)
        vq, vs = _split4(v)
        st.update(kq=kq, ks=ks, vq=vq, vs=vs)
        if own:
            st['cache'] = _lib().KV4Cache(kq, ks, vq, vs)
        return st
    st.update(k=k, v=v)
    if op in ('scored_decode', 'evict'):
        # a few slots hold most of the weight; small numbers are common, exact ties too
        acc = torch.empty(c['b'], c['nkv'], c['s'], device='cuda').exponential_(1.0, generator=g).pow(3)
        acc[torch.rand(acc.shape, generator=g, device='cuda') < 0.2] = 0.0
        st['acc'] = acc
    if own:
        st['cache'] = _lib().KVCache(k, v)
    if op == 'evict':
        st['into_k'], st['into_v'] = torch.zeros_like(k), torch.zeros_like(v)
        if own:
            st['into'] = _lib().KVCache(st['into_k'], st['into_v'])
    return st


# -------------------------------------------------------------------------------------------------------- plain form
def _softmax_pv(q, k, v, seen, scaling):
    """out [b, n, nh, D] and the weights [b, nkv, g, n, s] of q [b, nh, n, D] over k / v [b, nkv, s, D] where seen
    ([b, 1, 1, n, s])."""
    b, nh, n, _ = q.shape
    nkv = k.shape[1]
    qg = q.float().reshape(b, nkv, nh // nkv * n, D)
    s = torch.matmul(qg, k.float().transpose(2, 3)).view(b, nkv, nh // nkv, n, -1).mul_(scaling)
    s.masked_fill_(~seen, float('-inf'))
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = torch.matmul(s.view(b, nkv, nh // nkv * n, -1), v.float()).view(b, nh, n, D)
    return out.transpose(1, 2).to(torch.bfloat16), s


def _seen(pos, start, s, window=None, sinks=0):
    """[b, 1, 1, n, s]: which of the s slots the tokens at slots pos [b, n] see."""
    j = torch.arange(s, device=pos.device)
    p = pos[:, :, None]
    st = torch.zeros_like(pos[:, :1]) if start is None else start[:, None]
    st = st[:, :, None]
    m = (j >= st) & (j <= p)
    if window is not None:
        m &= (j > p - window) | (j < st + sinks)
    return m[:, None, None]


def _join4(q, s):
    """float32 values of codes q [..., D/2] and block scales s [..., D/16]."""
    code = torch.stack((q & 15, q >> 4), -1).flatten(-2)
    m = (code & 7).float()
    mag = torch.where(m < 2, m * 0.5, (1 + 0.5 * (code & 1).float()) * torch.exp2(torch.floor(m * 0.5) - 1))
    x = torch.where(code > 7, -mag, mag).unflatten(-1, (D // 16, 16))
    return (x * s.view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def _plain(st):
    c = st['case']
    op = c['op']
    if op == 'window_prefill':
        pos = torch.arange(st['past'], st['past'] + c['l'], device='cuda')[None].expand(c['b'], -1)
        seen = _seen(pos, st['start'], st['past'] + c['l'], c['window'], c['sinks'])
        return _softmax_pv(st['q'], st['k'], st['v'], seen, st['scaling'])[0]
    if op == 'kv4_store':
        return tuple(_join4(*_split4(x)).to(torch.bfloat16) for x in (st['k'], st['v']))
    if op == 'evict':
        j = torch.arange(c['s'], device='cuda')
        n = st['length'][:, None, None]
        lo = torch.zeros_like(n) if st['start'] is None else st['start'][:, None, None]
        live = (j >= lo) & (j < n)
        always = live & ((j < lo + c['sinks']) | (j >= n - c['recent']))
        key = st['acc'].masked_fill(always, float('inf')).masked_fill(~live, float('-inf'))
        slot = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :c['keep']]
        ok = torch.gather(live.expand_as(key), 2, slot)
        slot, order = torch.sort(torch.where(ok, slot, c['s']), dim=-1)
        ok = torch.gather(ok, 2, order)
        at = slot.clamp(max=c['s'] - 1)
        rows = at[..., None].expand(-1, -1, -1, D)
        k = torch.gather(st['k'], 2, rows).masked_fill(~ok[..., None], 0)
        v = torch.gather(st['v'], 2, rows).masked_fill(~ok[..., None], 0)
        acc = torch.gather(st['acc'], 2, at).masked_fill(~ok, 0)
        length = (n - lo).clamp(min=0, max=c['keep']).view(-1)
        return torch.where(ok, slot, -1).int(), length, k, v, acc
    pos = st['length'][:, None] - 1
    seen = _seen(pos, st['start'], c['s'], c.get('window'), c.get('sinks', 0))
    if op == 'kv4_decode':
        k, v = _join4(st['kq'], st['ks']), _join4(st['vq'], st['vs'])
        return _softmax_pv(st['q'], k, v, seen, st['scaling'])[0]
    out, p = _softmax_pv(st['q'], st['k'], st['v'], seen, st['scaling'])
    return out if op == 'window_decode' else (out, st['acc'] + p.sum((2, 3)))


def run(st):
    if not own:
        return _plain(st)
    c = st['case']
    op = c['op']
    lf = _lib()
    if op == 'window_decode':
        return lf.decode(st['q'], st['cache'], st['length'], starts=st['start'], window=c['window'], sinks=c['sinks'])
    if op == 'window_prefill':
        return lf.prefill(st['q'], st['k'], st['v'], window=c['window'], sinks=c['sinks'], starts=st['start'])
    if op == 'kv4_store':
        st['cache'].store(st['k'], st['v'], st['slots'])
        return st['cache'].read(st['slots'])
    if op == 'kv4_decode':
        return lf.decode(st['q'], st['cache'], st['length'], starts=st['start'])
    if op == 'scored_decode':
        acc = torch.empty_like(st['acc'])
        return lf.decode(st['q'], st['cache'], st['length'], starts=st['start'], acc=st['acc'], acc_out=acc), acc
    kept, length, acc = lf.evict(st['cache'], st['acc'], st['length'], c['keep'], into=st['into'], starts=st['start'],
                                 sinks=c['sinks'], recent=c['recent'])
    return kept, length, st['into_k'][:, :, :c['keep']], st['into_v'][:, :, :c['keep']], acc


# ----------------------------------------------------------------------------------------- the definitions in 64 bits
def _values4(x):
    """x [n, D] in 64 bits, each block of 16 on the 4-bit grid of its scale."""
    blk = x.double().reshape(-1, 16)
    want = (blk.abs().amax(1) / 6).clamp(max=448.0)
    e = torch.floor(torch.log2(want.clamp(min=2.0 ** -6))).clamp(min=-6)
    step = torch.exp2(e - 3)                                    # e4m3: 3 fraction bits, exponents from -6
    s = torch.round(want / step) * step                         # round() goes to even at ties
    grid = torch.tensor(LUT, dtype=torch.float64, device=x.device)
    a = blk.abs() / torch.where(s > 0, s, torch.ones_like(s))[:, None]
    near = torch.zeros_like(a)
    for i in range(1, 8):
        mid = (grid[i - 1] + grid[i]) / 2
        near = torch.where((a > mid) | ((a == mid) & (i % 2 == 0)), grid[i], near)
    return (torch.sign(blk) * near * s[:, None]).reshape(x.shape)


def _exact_row(q, k, v, seen, scaling):
    """One row and head group: q [g, n, D], k / v [s, D], seen [n, s] -> out [g, n, D], weights [g, n, s]."""
    z = torch.einsum('gnd,sd->gns', q.double(), k.double()) * scaling
    z = torch.where(seen, z, torch.full_like(z, float('-inf')))
    p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
    return torch.einsum('gns,sd->gnd', p, v.double()), p


def exact(case, seed):
    st = prepare(case, seed)
    c = st['case']
    op = c['op']
    if op == 'kv4_store':
        return tuple(_values4(x.reshape(-1, D)).reshape(x.shape) for x in (st['k'], st['v']))
    b, nh, nkv = c['b'], c['nh'], c['nkv']
    if op == 'evict':
        keep, s = c['keep'], c['s']
        kept = torch.full((b, nkv, keep), -1, dtype=torch.int32)
        length = torch.zeros(b, dtype=torch.int64)
        k = torch.zeros(b, nkv, keep, D, dtype=torch.float64, device='cuda')
        v = torch.zeros_like(k)
        acc = torch.zeros(b, nkv, keep, dtype=torch.float64, device='cuda')
        weight = st['acc'].cpu()
        for r in range(b):
            lo = 0 if st['start'] is None else int(st['start'][r])
            hi = int(st['length'][r])
            n = max(0, hi - lo)
            length[r] = min(n, keep)
            for h in range(nkv):
                if n <= keep:
                    rows = torch.arange(lo, lo + n)
                else:
                    mid = weight[r, h, lo + c['sinks']:hi - c['recent']]
                    best = torch.argsort(mid, descending=True, stable=True)[:keep - c['sinks'] - c['recent']]
                    rows = torch.cat((torch.arange(lo, lo + c['sinks']), lo + c['sinks'] + best.sort().values,
                                      torch.arange(hi - c['recent'], hi)))
                m = rows.numel()
                kept[r, h, :m] = rows.int()
                at = rows.cuda()
                k[r, h, :m], v[r, h, :m] = st['k'][r, h, at].double(), st['v'][r, h, at].double()
                acc[r, h, :m] = st['acc'][r, h, at].double()
        return kept, length, k, v, acc
    g = nh // nkv
    n = c.get('l', 1)
    s = c['s'] if 's' in c else st['past'] + c['l']
    out = torch.zeros(b, n, nh, D, dtype=torch.float64, device='cuda')
    acc = st['acc'].double() if op == 'scored_decode' else None
    j = torch.arange(s, device='cuda')
    for r in range(b):
        lo = 0 if st['start'] is None else int(st['start'][r])
        p = torch.arange(st['past'], s, device='cuda')[:, None] if op == 'window_prefill' else st['length'][r:r + 1, None] - 1
        seen = (j >= lo) & (j <= p)
        if 'window' in c:
            seen = seen & ((p - j < c['window']) | (j - lo < c['sinks']))
        for h in range(nkv):
            if op == 'kv4_decode':
                k, v = (_join64(st[x + 'q'][r, h], st[x + 's'][r, h]) for x in 'kv')
            else:
                k, v = st['k'][r, h], st['v'][r, h]
            for i in range(h * g, h * g + g) if n > 1 else (None,):       # a head at a time where there are many tokens
                at = slice(h * g, h * g + g) if i is None else slice(i, i + 1)
                o, w = _exact_row(st['q'][r, at], k, v, seen, st['scaling'])
                out[r, :, at] = o.transpose(0, 1)
                if acc is not None:
                    acc[r, h] += w.sum((0, 1))
    return out if acc is None else (out, acc)


def _join64(q, s):
    grid = torch.tensor(LUT + tuple(-x for x in LUT), dtype=torch.float64, device=q.device)
    x = grid[torch.stack((q % 16, q // 16), -1).flatten(-2).int()]
    return x * s.view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)
