"""GPU tests of the long-speech path: the backbone on bounded caches against the decode step over the whole sequence."""
import pytest
import torch

from gpu_util import E2E_TOL, assert_close, np32

pytestmark = pytest.mark.gpu


def _pair(B, S, **kw):
    from flashb.engine import BackboneConfig, SyntheticBackboneGraph
    from flashb.long_speech import LongSpeech
    cfg = BackboneConfig(layers=3)
    g = SyntheticBackboneGraph(cfg, batch_size=B, max_seq_len=S, seed=5)
    g2 = SyntheticBackboneGraph(cfg, batch_size=B, max_seq_len=S, weights_from=g)
    return cfg, g, g2, LongSpeech(g2, **kw)


def _ids(cfg, B, n):
    return torch.randint(0, cfg.vocab, (n, B, 1, cfg.codebooks), generator=torch.Generator().manual_seed(6)).cuda()


@pytest.mark.parametrize('B', [2, 20])
def test_whole_cache_is_the_decode_step(B):
    """No window, no eviction, room for everything: the framework's own prefill and decode step."""
    from flashb.prefill import prefill_forward
    L, frames = 37, 5
    cfg, g, _, s = _pair(B, 64, slots=64)
    x = torch.randn(B, L, cfg.hidden, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).cuda()
    starts = torch.randint(0, 9, (B,), generator=torch.Generator().manual_seed(8)).cuda()
    low = torch.finfo(torch.bfloat16).min
    i, j = torch.arange(L, device='cuda')[:, None], torch.arange(64, device='cuda')
    mask = torch.where((j <= i) & (j >= starts[:, None, None]), 0.0, low).to(torch.bfloat16).view(B, 1, L, 64)
    pos = (torch.arange(L, device='cuda') - starts[:, None]).clamp(min=0)
    kv = [(c.keys, c.values) for c in g.static_cache.layers]
    want, _ = prefill_forward(g._bb_state, x, mask, pos, torch.arange(L, device='cuda'), kv)
    got = s.prefill(x, starts)
    live = (torch.arange(L, device='cuda') >= starts[:, None])
    assert_close(np32(got[live]), np32(want[live]), E2E_TOL, 'prefill hidden')
    g.set_position(L, starts.cpu())
    for f, ids in enumerate(_ids(cfg, B, frames)):
        g.input_ids_buf.copy_(ids)
        s.graph.input_ids_buf.copy_(ids)
        g.decode_step(advance=f > 0)
        s.step()
        assert_close(np32(s.graph.hidden_buf), np32(g.hidden_buf), E2E_TOL, f'hidden of frame {f}')
        assert_close(s.graph.cfg_logits_buf.cpu().numpy(), g.cfg_logits_buf.cpu().numpy(), E2E_TOL, f'logits of frame {f}')


def test_four_bits_is_the_cache_it_reads_back():
    """A step over the 4-bit caches is a step over bf16 caches that hold what they stand for."""
    from flashb.long_speech import LongSpeech
    cfg, g, g2, s = _pair(2, 200, slots=128, four_bits=True, window=40, sinks=3)
    x = torch.randn(2, 70, cfg.hidden, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    s.prefill(x, torch.tensor([0, 6], device='cuda'))
    b = LongSpeech(g, 128, window=40, sinks=3)
    at = torch.arange(128, device='cuda')
    for c4, c in zip(s.caches, b.caches):
        k, v = c4.read(at)
        c.keys.copy_(k)
        c.values.copy_(v)
    b.lengths.copy_(s.lengths)
    b.starts.copy_(s.starts)
    b.used = s.used
    g.position_ids.copy_(g2.position_ids)
    ids = _ids(cfg, 2, 1)[0]
    g.input_ids_buf.copy_(ids)
    g2.input_ids_buf.copy_(ids)
    # the new token: 4 bits against bf16 in one of 40 slots of each layer, so only near
    s.step()
    b.step()
    assert_close(np32(g2.hidden_buf), np32(g.hidden_buf), 0.25, 'hidden')
    k, v = s.caches[0].read(torch.tensor([70], device='cuda'))
    import longform_ref as ref
    for got, c in ((k, b.caches[0].keys), (v, b.caches[0].values)):
        assert torch.equal(got.cpu().double(), ref.quantise(c[:, :, 70:71].cpu()))


@pytest.mark.parametrize('four_bits', [False, True])
def test_eviction_keeps_the_reading_going(four_bits):
    cfg, _, g, s = _pair(2, 200, slots=64, four_bits=four_bits, keep=40, sinks=4)
    x = torch.randn(2, 50, cfg.hidden, generator=torch.Generator().manual_seed(10)).to(torch.bfloat16).cuda()
    s.prefill(x, torch.tensor([0, 12], device='cuda'))
    for f, ids in enumerate(_ids(cfg, 2, 45)):
        g.input_ids_buf.copy_(ids)
        s.step()
        assert torch.isfinite(g.cfg_logits_buf).all()
        assert s.used <= 64 and int(s.lengths.max()) <= s.used
    assert int(g.position_ids[0, 0]) == 95 and int(g.position_ids[1, 0]) == 83
    total = s.acc[0].sum((1, 2))
    assert torch.isfinite(total).all() and (total > 0).all()


def test_full_cache_without_eviction_raises():
    from flashb._native import FlashbError
    cfg, _, g, s = _pair(2, 64, slots=20)
    s.prefill(torch.zeros(2, 20, cfg.hidden, dtype=torch.bfloat16, device='cuda'))
    with pytest.raises(FlashbError):
        s.step()
    with pytest.raises(FlashbError):
        s.prefill(torch.zeros(2, 1, cfg.hidden, dtype=torch.bfloat16, device='cuda'))


def test_command():
    from flashb import long_speech
    long_speech.main(['--layers', '2', '--frames', '30', '--prompt', '20', '--slots', '32', '--keep', '24', '--four-bits',
                      '--window', '16'])
