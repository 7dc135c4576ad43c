"""The backbone over pages against the framework's own prefill and decode step, fed in chunks, released and reused."""
import pytest
import torch

from gpu_util import E2E_TOL, assert_close, np32

pytestmark = pytest.mark.gpu


def _graph(layers=3, S=96, B=2):
    from flashb.engine import BackboneConfig, SyntheticBackboneGraph
    cfg = BackboneConfig(layers=layers)
    return cfg, SyntheticBackboneGraph(cfg, batch_size=B, max_seq_len=S, seed=5)


def _x(cfg, n, seed):
    return torch.randn(n, cfg.hidden, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


def _speech(g, **kw):
    from flashb.paged_speech import PagedSpeech
    kw.setdefault('pages', 40)
    kw.setdefault('page', 16)
    return PagedSpeech(g, kw.pop('rows', 2), **kw)


def test_prompt_and_frames_are_the_decode_step():
    from flashb.prefill import prefill_forward
    L, frames = 37, 4
    cfg, g = _graph()
    s = _speech(g)
    x = _x(cfg, 2 * L, 7).view(2, L, -1)
    low = torch.finfo(torch.bfloat16).min
    i, j = torch.arange(L, device='cuda')[:, None], torch.arange(96, device='cuda')
    mask = torch.where(j <= i, 0.0, low).to(torch.bfloat16).expand(2, 1, L, 96).contiguous()
    pos = torch.arange(L, device='cuda').expand(2, L).contiguous()
    kv = [(c.keys, c.values) for c in g.static_cache.layers]
    want, logits = prefill_forward(g._bb_state, x, mask, pos, torch.arange(L, device='cuda'), kv)
    # row 0 in chunks beside row 1 all at once
    parts = [s.extend(torch.cat((x[0, :10], x[1])), [10, L]), s.extend(x[0, 10:11], [1, 0]), s.extend(x[0, 11:], [L - 11, 0])]
    got = torch.cat((parts[0][:10], parts[1], parts[2]))
    assert_close(np32(got), np32(want[0]), E2E_TOL, 'prompt of row 0')
    assert_close(np32(parts[0][10:]), np32(want[1]), E2E_TOL, 'prompt of row 1')
    assert_close(s.logits(got[-1:]).cpu().numpy(), logits[:1].cpu().numpy(), E2E_TOL, 'logits')
    g.set_position(L)
    gen = torch.Generator().manual_seed(6)
    for f in range(frames):
        ids = torch.randint(0, cfg.vocab, (2, cfg.codebooks), generator=gen).cuda()
        g.input_ids_buf.copy_(ids.view(2, 1, -1))
        g.decode_step(advance=f > 0)
        h = s.extend(s.embed(ids), [1, 1])
        assert_close(np32(h), np32(g.hidden_buf.view(2, -1)), E2E_TOL, f'hidden of frame {f}')
        assert_close(s.logits(h).cpu().numpy(), g.logits_buf.cpu().numpy(), E2E_TOL, f'logits of frame {f}')


def test_rows_come_and_go():
    """A released row's pages serve another reading, which reads as if it were alone."""
    cfg, g = _graph(layers=2)
    s = _speech(g, rows=3, pages=9)
    a, b, c = (_x(cfg, n, n) for n in (50, 60, 40))
    ha, hb = (lambda h: (h[:50], h[50:]))(s.extend(torch.cat((a, b)), [50, 60, 0]))
    assert len(s.free) == 1
    from flashb._native import FB_ERR_STATE, FlashbError
    before = s.lengths.clone()
    with pytest.raises(FlashbError) as e:
        s.extend(torch.cat((a[:1], c)), [1, 0, 40])
    assert e.value.rc == FB_ERR_STATE and torch.equal(s.lengths, before) and len(s.free) == 1 and s.used == [50, 60, 0]
    s.release(1)
    hc = s.extend(c, [0, 0, 40])
    alone = _speech(g, rows=1, pages=9)
    assert torch.equal(alone.extend(c, [40]), hc)
    assert_close(np32(hb), np32(_speech(g, rows=1, pages=9).extend(b, [60])), E2E_TOL, 'row 1')
    assert_close(np32(ha), np32(_speech(g, rows=1, pages=9).extend(a, [50])), E2E_TOL, 'row 0')


def test_window_gives_pages_back():
    """With a window the pool is bounded, and what is given back was not seen."""
    cfg, g = _graph(layers=2)
    # what the first token of a chunk sees lies in 1 + ceil((33 + 15) / 16) pages, the longest chunk in ceil((60 + 15) / 16)
    small, big = (_speech(g, rows=1, pages=n, window=33, sinks=5, max_slots=400) for n in (9, 40))
    x = _x(cfg, 300, 3)
    at = 0
    for n in (40, 1, 1, 30, 7, 16, 16, 1, 60, 1, 20, 1, 1, 40, 1, 1):
        h = small.extend(x[at:at + n], [n])
        w = big.extend(x[at:at + n], [n])
        assert torch.equal(h, w)
        at += n
        assert 9 - len(small.free) <= 1 + -(-(33 + 15) // 16) + 1
        for t in small.caches[0].keys, small.caches[0].values:       # what no row holds may be anything
            t[small.free] = float('nan')
    assert small.used == [at]


def test_scores_of_a_given_reading():
    from flashb.sampling import token_scores
    cfg, g = _graph(layers=2)
    s = _speech(g, pages=40)
    h = s.extend(_x(cfg, 300, 4), [140, 160])
    tokens = torch.randint(0, cfg.vocab, (300,), generator=torch.Generator().manual_seed(5)).cuda()
    got = s.score(h, tokens, top=3, temperature=0.8)
    logits = s.logits(h)
    assert logits.shape == (300, cfg.vocab)
    want = torch.log_softmax(logits.double() / 0.8, -1)
    assert torch.allclose(got.logprob.double(), want.gather(1, tokens[:, None])[:, 0], rtol=1e-5, atol=1e-5)
    assert torch.equal(got.top_ids, logits.topk(3).indices)
    assert all(torch.equal(p, q) for p, q in zip(got, token_scores(logits, tokens, top=3, temperature=0.8)))


def test_bad_steps_are_refused():
    from flashb._native import FlashbError
    from flashb.paged_speech import PagedSpeech
    cfg, g = _graph(layers=1)
    s = _speech(g, max_slots=32)
    x = _x(cfg, 40, 1)
    for counts in ([1], [3, -1], [1, 2], [1, 1, 1]):
        with pytest.raises(FlashbError):
            s.extend(x[:2], counts)
    with pytest.raises(FlashbError):
        s.extend(x[:33], [33, 0])
    assert s.extend(x[:0], [0, 0]).shape == (0, cfg.hidden) and s.used == [0, 0]
    for kw in (dict(rows=0, pages=4), dict(rows=1, pages=0), dict(rows=1, pages=4, page=24), dict(rows=1, pages=4, window=0),
               dict(rows=1, pages=4, sinks=-1)):
        with pytest.raises(FlashbError):
            PagedSpeech(g, **kw)


def test_command():
    from flashb import paged_speech
    paged_speech.main(['--rows', '3', '--layers', '2', '--frames', '12', '--prompt', '50', '--chunk', '16', '--page', '16',
                       '--pages', '40', '--window', '32', '--yarn', '4'])
