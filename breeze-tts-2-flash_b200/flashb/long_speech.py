"""A long reading on a bounded cache: the backbone prefill and decode step of ``flashb.backbone`` / ``flashb.prefill`` with
their attention and cache replaced by ``flashb.longform`` -- a sliding window with sink tokens, a 4-bit cache, eviction by
attention weight, in any combination.

    speech = LongSpeech(graph, slots=1024, four_bits=True, window=512, sinks=4)
    speech.prefill(inputs_embeds)                 # [B, L, H]; starts: left padding per row
    for frame in ...:
        graph.input_ids_buf.copy_(ids)
        speech.step()                             # graph.hidden_buf, logits_buf, cfg_logits_buf as after a decode step

``graph`` carries the attributes that ``flashb.backbone.fused_decode_step`` reads (an official ``BackboneGraph``, or
``flashb.engine.SyntheticBackboneGraph``); its own static cache and mask are not used, so give it the smallest
``max_seq_len`` that its other uses need, and the reading's length to ``positions``: a rotary table of that many entries
(512 bytes each, all that grows with the reading; None: the graph's table, ``max_seq_len`` + 1).  Keys enter the cache
after their rotary embedding, so their slot may change while their position stays; a reading that reaches the end of the
table raises.  With ``keep`` the caches are evicted to that many slots when they are full, each layer by its own weights
(those of the decode steps: the prompt's slots begin at 0); without it a full cache raises.  ``reset`` empties them for
another reading.

    python -m flashb.long_speech --frames 200 --slots 256 --four-bits --window 128 --keep 192
"""
import argparse
import time

import torch

from . import backbone as bb
from . import kernels, longform
from ._native import FB_ERR_ARG, FB_ERR_STATE, FlashbError


def rotary_table(graph, n, device):
    """cos / sin [n, 128] bf16 of positions 0 .. n - 1 as the graph's own table has them."""
    if hasattr(graph, 'model'):
        with torch.no_grad():
            x = torch.zeros(1, n, 128, dtype=torch.bfloat16, device=device)
            cos, sin = graph.model.rotary_emb(x, torch.arange(n, device=device)[None])
        return tuple(t[0].to(torch.bfloat16).contiguous() for t in (cos, sin))
    from .engine import rope_table
    return rope_table(graph.cfg.theta, 128, n, device)


class LongSpeech:
    def __init__(self, graph, slots, four_bits=False, window=None, sinks=4, keep=None, recent=None, decay=1.0,
                 positions=None):
        st = bb._prep(graph)
        if st is None:
            raise FlashbError(FB_ERR_ARG, 'long speech: the graph is outside the fused decode step')
        if keep is not None and not 0 < keep < slots:
            raise FlashbError(FB_ERR_ARG, f'long speech: keep {keep} of {slots} slots')
        self.graph, self.st, self.slots = graph, st, slots
        self.window, self.sinks, self.keep, self.decay = window, sinks, keep, decay
        self.recent = max(0, min(keep // 4, keep - sinks)) if keep is not None and recent is None else recent or 0
        if sinks < 0 or self.recent < 0 or (keep is not None and sinks + self.recent > keep):
            raise FlashbError(FB_ERR_ARG, f'long speech: {sinks} first and {self.recent} last slots of the {keep} that stay')
        if window is not None and window < 1:
            raise FlashbError(FB_ERR_ARG, f'long speech: a window of {window}')
        L0 = st['layers'][0]
        B, self.NH, self.NKV = st['B'], L0.wq.shape[0] // 128, L0.wk.shape[0] // 128
        dev = self.device = L0.wq.device
        n = len(st['layers'])

        def cache():
            if four_bits:
                return longform.KV4Cache.empty(B, self.NKV, slots, device=dev)
            return longform.KVCache(*(torch.zeros(B, self.NKV, slots, 128, dtype=torch.bfloat16, device=dev)
                                      for _ in range(2)))
        self.caches = [cache() for _ in range(n)]
        # eviction moves layer i's slots into the spare cache, which then becomes layer i's; the old one is the next spare
        self.spare = cache() if keep is not None else None
        self.acc = [torch.zeros(B, self.NKV, slots, device=dev) for _ in range(n)] if keep is not None else None
        self.spare_acc = torch.zeros(B, self.NKV, slots, device=dev) if keep is not None else None
        self.lengths = torch.zeros(B, dtype=torch.int64, device=dev)
        self.starts = torch.zeros(B, dtype=torch.int64, device=dev)
        self.used = 0                                     # the largest length (every row grows by one a step)
        if positions is not None and positions < 1:
            raise FlashbError(FB_ERR_ARG, f'long speech: a rotary table of {positions} positions')
        self.cos_tab, self.sin_tab = ((st['cos_tab'], st['sin_tab']) if positions is None else
                                      rotary_table(graph, positions, dev))
        self.table = self.cos_tab.shape[0]                # positions that the rotary table has
        self.next = 0                                     # no row's next position is beyond it
        self.rows = torch.arange(B, device=dev)
        self.zero = torch.zeros(1, dtype=torch.int64, device=dev)
        self.new_k, self.new_v = (torch.empty(B, self.NKV, 1, 128, dtype=torch.bfloat16, device=dev) for _ in range(2))

    def reset(self):
        """Empty caches for another reading; nothing is allocated."""
        for t in (self.lengths, self.starts, *(self.acc or ())):
            t.zero_()
        self.used = self.next = 0

    def _put(self, cache, k, v, slots):
        """k / v [B, NKV, L, 128] to slots [B, L]."""
        if cache.bits == 4:
            cache.store(k, v, slots)
        else:
            for dst, src in ((cache.keys, k), (cache.values, v)):
                dst[self.rows[:, None], :, slots] = src.transpose(1, 2)

    def _mlp(self, Lw, ao, x):
        fx = kernels.fused()
        h1 = torch.empty_like(x)
        fx.gemv_resid(ao, Lw.wo, x, h1)
        act = torch.empty(x.shape[0], Lw.wg.shape[0], dtype=torch.bfloat16, device=x.device)
        if x.shape[0] > bb.ROWS_NORM_APART:
            xn = torch.empty_like(x)
            fx.rmsnorm(h1, Lw.ln2_w, Lw.ln2_eps, xn)
            fx.gemv_gateup(xn, None, Lw.ln2_eps, Lw.wg, Lw.wu, act)
        else:
            fx.gemv_gateup(h1, Lw.ln2_w, Lw.ln2_eps, Lw.wg, Lw.wu, act)
        y = torch.empty_like(x)
        fx.gemv_resid(act, Lw.wd, h1, y)
        return y

    def _qkv(self, Lw, x):
        fx = kernels.fused()
        qkv = torch.empty(x.shape[0], Lw.wq.shape[0] + 2 * Lw.wk.shape[0], dtype=torch.bfloat16, device=x.device)
        if x.shape[0] > bb.ROWS_NORM_APART:
            xn = torch.empty_like(x)
            fx.rmsnorm(x, Lw.ln1_w, Lw.ln1_eps, xn)
            fx.gemv_seg(xn, None, Lw.ln1_eps, Lw.wq, Lw.wk, Lw.wv, qkv)
        else:
            fx.gemv_seg(x, Lw.ln1_w, Lw.ln1_eps, Lw.wq, Lw.wk, Lw.wv, qkv)
        return qkv

    def prefill(self, inputs_embeds, starts=None):
        """The prompt [B, L, H] bf16 (row b's tokens from ``starts[b]`` on, clamped to 0 .. L; positions count from there)
        into empty caches (a first reading's, or after ``reset``).  Returns the hidden states [B, L, H] after the final
        norm."""
        fx, st = kernels.fused(), self.st
        B, L, H = inputs_embeds.shape
        if L > self.slots or self.used:
            raise FlashbError(FB_ERR_STATE, f'long speech: a prompt of {L} into {self.slots} slots, {self.used} in use')
        if L > self.table and (starts is None or L - max(0, int(starts.min())) > self.table):
            raise FlashbError(FB_ERR_STATE, f'long speech: a prompt of {L} with a rotary table of {self.table} positions')
        if starts is not None:
            self.starts.copy_(starts).clamp_(0, L)
        at = torch.arange(L, device=self.device)
        pos = (at[None] - self.starts[:, None]).clamp_(min=0).contiguous()
        slots = at[None].expand(B, L)
        k, v = (torch.empty(B, self.NKV, L, 128, dtype=torch.bfloat16, device=self.device) for _ in range(2))
        x = inputs_embeds.reshape(B * L, H).contiguous()
        for Lw, cache in zip(st['layers'], self.caches):
            qkv = self._qkv(Lw, x)
            fx.prefill_qkv(qkv, B, L, self.NH, self.NKV, Lw.qn_w, Lw.kn_w, Lw.qk_eps, self.cos_tab, self.sin_tab, pos, at,
                           k, v)
            q = qkv.as_strided((B, self.NH, L, 128), (L * qkv.stride(0), 128, qkv.stride(0), 1))
            self._put(cache, k, v, slots)
            # attend to what later steps will find in the cache
            kk, vv = cache.read(at) if cache.bits == 4 else (k, v)
            ao = longform.prefill(q, kk, vv, window=self.window, sinks=self.sinks, starts=self.starts, scaling=Lw.scaling)
            x = self._mlp(Lw, ao.view(B * L, -1), x)
        hidden = torch.empty(B, L, H, dtype=torch.bfloat16, device=self.device)
        fx.rmsnorm(x, st['norm_w'], st['norm_eps'], hidden.view(B * L, H))
        self.used = self.next = L
        self.lengths.fill_(L)
        self.graph.position_ids.copy_((L - self.starts).view(B, 1))
        return hidden

    def step(self):
        """One decode step on the graph's buffers; row b's token goes to slot ``lengths[b]`` at position
        ``graph.position_ids[b]``, and both move on by one."""
        g, st, fx = self.graph, self.st, kernels.fused()
        B = st['B']
        if self.next >= self.table:
            # past the table a token would get no rotary embedding and its key no place; the rows may be padded, so look
            self.next = int(g.position_ids.max())
            if self.next >= self.table:
                raise FlashbError(FB_ERR_STATE, f'long speech: all {self.table} positions of the rotary table are in use')
        if self.used == self.slots:
            self._evict()
        slots = self.lengths.view(B, 1).clone()
        self.lengths += 1
        self.used += 1
        self.next += 1
        pos = g.position_ids.view(-1)
        fx.embed_rope(g.input_ids_buf.view(B, -1), st['vocab'], st['embed'], pos, self.cos_tab, self.sin_tab, st['x0'],
                      st['cos'], st['sin'])
        x = st['x0']
        for i, (Lw, cache) in enumerate(zip(st['layers'], self.caches)):
            qkv = self._qkv(Lw, x)
            fx.prefill_qkv(qkv, B, 1, self.NH, self.NKV, Lw.qn_w, Lw.kn_w, Lw.qk_eps, self.cos_tab, self.sin_tab, pos,
                           self.zero, self.new_k, self.new_v)
            self._put(cache, self.new_k, self.new_v, slots)
            q = qkv.as_strided((B, self.NH, 1, 128), (qkv.stride(0), 128, qkv.stride(0), 1))
            ao = longform.decode(q, cache, self.lengths, starts=self.starts, window=self.window, sinks=self.sinks,
                                 scaling=Lw.scaling, acc=self.acc[i] if self.acc is not None else None, decay=self.decay)
            x = self._mlp(Lw, ao.view(B, -1), x)
        hb = g.hidden_buf.view(B, -1)
        blk = getattr(g, 'cfg_block', B)
        if blk == B and B <= 16:
            fx.lm_head_cfg(x, st['norm_w'], st['norm_eps'], st['lm_head32'], g.guidance_scale, hb, g.logits_buf,
                           g.cfg_logits_buf)
        else:
            fx.lm_head_cfg_blocks(x, st['norm_w'], st['norm_eps'], st['lm_head32'], g.guidance_scale, blk, hb, g.logits_buf,
                                  g.cfg_logits_buf)
        g.position_ids += 1

    def _evict(self):
        if self.keep is None:
            raise FlashbError(FB_ERR_STATE, f'long speech: all {self.slots} slots are in use')
        for i, cache in enumerate(self.caches):
            _, n, acc = longform.evict(cache, self.acc[i], self.lengths, self.keep, into=self.spare, starts=self.starts,
                                       sinks=self.sinks, recent=self.recent, acc_into=self.spare_acc)
            self.caches[i], self.spare = self.spare, cache
            self.acc[i], self.spare_acc = acc, self.acc[i]
        self.lengths.copy_(n)
        self.starts.zero_()
        self.used = self.keep

    def cache_bytes(self):
        """Bytes of one layer's cache."""
        c = self.caches[0]
        ts = (c.kq, c.vq, c.ks, c.vs) if c.bits == 4 else (c.keys, c.values)
        return sum(t.numel() * t.element_size() for t in ts)


def main(argv=None):
    from .engine import BackboneConfig, SyntheticBackboneGraph
    ap = argparse.ArgumentParser(description='A long reading on a bounded cache (synthetic weights)')
    ap.add_argument('--frames', type=int, default=200)
    ap.add_argument('--prompt', type=int, default=100)
    ap.add_argument('--slots', type=int, default=512)
    ap.add_argument('--layers', type=int, default=28)
    ap.add_argument('--batch', type=int, default=2)
    ap.add_argument('--four-bits', action='store_true')
    ap.add_argument('--window', type=int)
    ap.add_argument('--sinks', type=int, default=4)
    ap.add_argument('--keep', type=int)
    a = ap.parse_args(argv)
    cfg = BackboneConfig(layers=a.layers)
    g = SyntheticBackboneGraph(cfg, batch_size=a.batch, max_seq_len=1)
    s = LongSpeech(g, a.slots, four_bits=a.four_bits, window=a.window, sinks=a.sinks, keep=a.keep,
                   positions=a.prompt + a.frames)
    gen = torch.Generator().manual_seed(1)
    s.prefill(torch.randn(a.batch, a.prompt, cfg.hidden, generator=gen).to(torch.bfloat16).cuda())
    ids = torch.randint(0, cfg.vocab, (a.frames, a.batch, 1, cfg.codebooks), generator=gen).cuda()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for f in range(a.frames):
        g.input_ids_buf.copy_(ids[f])
        s.step()
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    print(f'{a.frames} frames of {a.batch} rows, {a.slots} slots a layer ({s.cache_bytes() / 1e6:.2f} MB), '
          f'{1e3 * t / a.frames:.2f} ms a frame, logits finite: {bool(torch.isfinite(g.cfg_logits_buf).all())}')


if __name__ == '__main__':
    main()
