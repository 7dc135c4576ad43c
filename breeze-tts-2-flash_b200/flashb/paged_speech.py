"""Many readings at once on one pool of pages: the backbone of ``flashb.backbone`` / ``flashb.prefill`` over
``flashb.paged``.  Each step takes any number of new tokens of each row -- a chunk of one stream's prompt beside the next
frames of the others -- and a row takes pages as it grows and gives them back when it ends.

    speech = PagedSpeech(graph, rows=64, pages=2048)
    hidden = speech.extend(embeds, [200, 0, 1, ...])     # [T, H]: 200 prompt tokens of row 0, a frame of row 2, ...
    logits = speech.logits(hidden[last])                 # fp32, of the tokens asked for
    scores = speech.score(hidden, tokens, top=5)         # log probabilities of given tokens (``flashb.sampling``)
    speech.release(0)                                    # the row ends: its pages go back

``graph`` carries the weights that ``flashb.backbone.fused_decode_step`` reads (an official ``BackboneGraph``, or
``flashb.engine.SyntheticBackboneGraph``); its own cache, mask and position buffers are not used, so its ``max_seq_len``
may be 1.  Positions are the row's own slots, embedded by ``rotary`` (None: as the graph's model does); it has no table
that could end, and may be scaled for readings longer than the training's.  With ``window`` the pages that no later token
can see (those behind the window and past the first ``sinks`` slots) are given back as the row grows.

    python -m flashb.paged_speech --rows 8 --frames 100 --chunk 64 --window 512
"""
import argparse
import time

import torch

from . import backbone as bb
from . import kernels, paged
from ._native import FB_ERR_ARG, FB_ERR_STATE, FlashbError
from .long_speech import LongSpeech
from .sampling import token_scores

ROWS_LOGITS = 128                                          # rows of hidden states that the lm_head takes at once


def graph_rotary(graph, device):
    """The rotary positions of the graph's model."""
    if hasattr(graph, 'model'):
        emb = graph.model.rotary_emb
        return paged.Rotary(2 * emb.inv_freq.numel(), freq=emb.inv_freq.double(),
                            amplitude=float(getattr(emb, 'attention_scaling', 1.0)), device=device)
    return paged.Rotary(128, base=graph.cfg.theta, device=device)


class PagedSpeech:
    def __init__(self, graph, rows, pages, page=64, max_slots=None, window=None, sinks=0, rotary=None):
        """``rows`` readings on ``pages`` pages of ``page`` slots, each of at most ``max_slots`` (None: all pages)."""
        st = bb._prep(graph)
        if st is None:
            raise FlashbError(FB_ERR_ARG, 'paged speech: the graph is outside the fused decode step')
        if rows < 1 or pages < 1 or page < 16 or page & (page - 1):
            raise FlashbError(FB_ERR_ARG, f'paged speech: {rows} rows on {pages} pages of {page} slots')
        if (window is not None and window < 1) or sinks < 0:
            raise FlashbError(FB_ERR_ARG, f'paged speech: a window of {window} and {sinks} first slots')
        if max_slots is not None and max_slots < 1:
            raise FlashbError(FB_ERR_ARG, f'paged speech: {max_slots} slots a row')
        L0 = st['layers'][0]
        dev = self.device = L0.wq.device
        self.st, self.page, self.window, self.sinks = st, page, window, sinks
        self.codebooks = graph.input_ids_buf.shape[-1]
        self.NH, self.NKV = L0.wq.shape[0] // 128, L0.wk.shape[0] // 128
        self.rotary = graph_rotary(graph, dev) if rotary is None else rotary
        self.caches = [paged.PagedCache.empty(pages, self.NKV, page, device=dev) for _ in st['layers']]
        self.slots = pages * page if max_slots is None else max_slots      # of a row, at most
        self.width = -(-self.slots // page)
        self.free = list(range(pages - 1, -1, -1))          # pages of no row; the same page of every layer's pool
        self.pages = [[] for _ in range(rows)]              # each row's, -1: given back
        self.gone = [0] * rows                              # how many pages from the sinks' on a row has given back
        self.used = [0] * rows                              # each row's slots
        self._host = torch.full((rows, self.width), -1, dtype=torch.int32)
        self.table = self._host.to(dev)
        self.lengths = torch.zeros(rows, dtype=torch.int64, device=dev)

    _qkv, _mlp = LongSpeech._qkv, LongSpeech._mlp

    def _take(self, counts):
        """Pages for the step's tokens; all of them or none."""
        want = [-(-(self.used[r] + n) // self.page) - len(self.pages[r]) if n else 0 for r, n in enumerate(counts)]
        for r, n in enumerate(counts):
            if n and self.used[r] + n > self.slots:
                raise FlashbError(FB_ERR_STATE, f'paged speech: row {r} at {self.used[r] + n} slots, {self.slots} at most')
        if sum(want) > len(self.free):
            raise FlashbError(FB_ERR_STATE, f'paged speech: {sum(want)} pages wanted, {len(self.free)} free')
        for r, n in enumerate(want):
            for _ in range(n):
                self._host[r, len(self.pages[r])] = self.free[-1]
                self.pages[r].append(self.free.pop())
        return any(want)

    def _trim(self):
        """Pages that no later token can see: behind the window of the next one, past the sinks."""
        first = -(-self.sinks // self.page)
        some = False
        for r, used in enumerate(self.used):
            end = (used + 1 - self.window) // self.page if used >= self.window else 0     # pages all before it
            for i in range(max(first, self.gone[r]), min(end, len(self.pages[r]))):
                if self.pages[r][i] >= 0:
                    self.free.append(self.pages[r][i])
                    self.pages[r][i] = self._host[r, i] = -1
                    some = True
            self.gone[r] = max(self.gone[r], end)
        return some

    def release(self, row):
        """The row's reading ends: it is empty, its pages are free."""
        self.free += [p for p in reversed(self.pages[row]) if p >= 0]
        self.pages[row], self.used[row], self.gone[row] = [], 0, 0
        self._host[row] = -1
        self.table.copy_(self._host)
        self.lengths[row] = 0

    def embed(self, ids):
        """The input embeddings [T, H] of frames ``ids`` [T, codebooks] int64."""
        st = self.st
        if ids.device != self.device or ids.dtype != torch.int64 or ids.dim() != 2 or ids.shape[1] != self.codebooks:
            raise FlashbError(FB_ERR_ARG, f'paged speech: ids [T, {self.codebooks}] int64 on {self.device}')
        ids = ids.contiguous()
        x = torch.empty(ids.shape[0], st['embed'].shape[1], dtype=torch.bfloat16, device=self.device)
        if ids.shape[0] == 0:
            return x
        cs = torch.empty(2, ids.shape[0], 128, dtype=torch.bfloat16, device=self.device)
        pos = torch.zeros(ids.shape[0], dtype=torch.int64, device=self.device)
        kernels.fused().embed_rope(ids, st['vocab'], st['embed'], pos, st['cos_tab'], st['sin_tab'], x, cs[0], cs[1])
        return x

    def extend(self, embeds, counts):
        """The next ``counts[r]`` tokens of each row r, one row's after the other's in ``embeds`` [T, H] bf16.  Returns
        their hidden states [T, H] after the final norm.  Raises, with nothing changed, when an argument is wrong or pages run
        out."""
        if embeds.device != self.device or embeds.dtype != torch.bfloat16 or embeds.dim() != 2 or (
                embeds.shape[1] != self.st['embed'].shape[1]):
            raise FlashbError(FB_ERR_ARG, f'paged speech: embeds [T, {self.st["embed"].shape[1]}] bf16 on {self.device}')
        T = embeds.shape[0]
        if len(counts) != len(self.used) or min(counts) < 0 or sum(counts) != T:
            raise FlashbError(FB_ERR_ARG, f'paged speech: counts of {len(counts)} rows and {sum(counts)} tokens for '
                                          f'{len(self.used)} rows and {T}')
        if T == 0:
            return embeds.clone()
        changed = self._take(counts)
        if changed:
            self.table.copy_(self._host)
        table, lengths, offsets = self.table, self.lengths, None
        if max(counts) > 1:
            n = torch.tensor(counts, dtype=torch.int64)
            offsets = torch.cat((n.new_zeros(1), n.cumsum(0))).to(self.device)
            self.lengths += n.to(self.device)
        elif T == len(counts):
            self.lengths += 1
        else:
            # at most one token a row: the rows that have one, in the form of single tokens, so that what a frame's attention
            # rounds does not hang on who else is idle
            rows = torch.tensor([r for r, m in enumerate(counts) if m], dtype=torch.int64).to(self.device)
            self.lengths[rows] += 1
            table, lengths = self.table[rows], self.lengths[rows]
        for r, m in enumerate(counts):
            self.used[r] += m
        fx, st = kernels.fused(), self.st
        x = embeds.contiguous()
        for Lw, cache in zip(st['layers'], self.caches):
            qkv = self._qkv(Lw, x)
            q = paged.append(qkv, cache, table, lengths, offsets=offsets, rotary=self.rotary, q_norm=Lw.qn_w, k_norm=Lw.kn_w,
                             eps=Lw.qk_eps, out=qkv[:, :self.NH * 128].view(T, self.NH, 128))
            ao = paged.attend(q, cache, table, lengths, offsets=offsets, window=self.window, sinks=self.sinks,
                              scaling=Lw.scaling)
            x = self._mlp(Lw, ao.view(T, -1), x)
        hidden = torch.empty_like(x)
        fx.rmsnorm(x, st['norm_w'], st['norm_eps'], hidden)
        if self.window is not None and self._trim():
            self.table.copy_(self._host)
        return hidden

    def logits(self, hidden):
        """The lm_head's logits [n, V] fp32 of hidden states [n, H]."""
        W = self.st['lm_head32']
        out = torch.empty(hidden.shape[0], W.shape[0], dtype=torch.float32, device=self.device)
        for a in range(0, hidden.shape[0], ROWS_LOGITS):
            kernels.fused().lm_head_rows(hidden[a:a + ROWS_LOGITS], W, out[a:a + ROWS_LOGITS])
        return out

    def score(self, hidden, tokens, top=0, temperature=1.0):
        """What the model says of the given next tokens [n] after hidden states [n, H]: ``flashb.sampling.TokenScores``."""
        return token_scores(self.logits(hidden), tokens, top=top, temperature=temperature)


def main(argv=None):
    from .engine import BackboneConfig, SyntheticBackboneGraph
    ap = argparse.ArgumentParser(description='Readings of different ages on one pool of pages (synthetic weights)')
    ap.add_argument('--rows', type=int, default=8)
    ap.add_argument('--frames', type=int, default=100)
    ap.add_argument('--prompt', type=int, default=200, help='tokens of the longest prompt')
    ap.add_argument('--chunk', type=int, default=64, help='prompt tokens of a step')
    ap.add_argument('--pages', type=int, default=256)
    ap.add_argument('--page', type=int, default=64)
    ap.add_argument('--layers', type=int, default=28)
    ap.add_argument('--window', type=int)
    ap.add_argument('--sinks', type=int, default=4)
    ap.add_argument('--yarn', type=float, help='factor of the scaled rotary positions')
    a = ap.parse_args(argv)
    cfg = BackboneConfig(layers=a.layers)
    g = SyntheticBackboneGraph(cfg, batch_size=2, max_seq_len=1)
    rotary = None
    if a.yarn:
        rotary = paged.Rotary(128, base=cfg.theta, scaling=dict(kind='yarn', factor=a.yarn, original=32768))
    s = PagedSpeech(g, a.rows, a.pages, page=a.page, window=a.window, sinks=a.sinks if a.window else 0, rotary=rotary)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randn(max(1, a.prompt * (r + 1) // a.rows), cfg.hidden, generator=gen).to(torch.bfloat16).cuda()
               for r in range(a.rows)]
    ids = torch.randint(0, cfg.vocab, (a.frames, a.rows, cfg.codebooks), generator=gen).cuda()
    fed, frames = [0] * a.rows, [0] * a.rows
    steps, given = 0, []
    torch.cuda.synchronize()
    t = time.perf_counter()
    while min(frames) < a.frames:
        # one chunk of a prompt a step, the next frame of every row whose prompt is done
        counts, parts, chunk, live = [], [], a.chunk, []
        for r in range(a.rows):
            left = prompts[r].shape[0] - fed[r]
            n = min(left, chunk) if left else int(frames[r] < a.frames)
            if left:
                parts.append(prompts[r][fed[r]:fed[r] + n])
                fed[r] += n
                chunk -= n
            elif n:
                parts.append(s.embed(ids[frames[r], r:r + 1]))
                frames[r] += 1
                live.append((sum(counts), r))
            counts.append(n)
        hidden = s.extend(torch.cat(parts), counts)
        steps += 1
        if live:                                           # how likely the given next frames' first codebook was
            at = torch.tensor([i for i, _ in live], device='cuda')
            nxt = torch.stack([ids[min(frames[r], a.frames - 1), r, 0] for _, r in live])
            given.append(s.score(hidden[at], nxt).logprob)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    lp = torch.cat(given)
    print(f'{a.rows} rows, {sum(len(p) for p in prompts)} prompt tokens and {a.rows * a.frames} frames in {steps} steps, '
          f'{1e3 * t / steps:.2f} ms a step; {len(s.free)} of {a.pages} pages free; mean log probability {float(lp.mean()):.3f}')


if __name__ == '__main__':
    main()
