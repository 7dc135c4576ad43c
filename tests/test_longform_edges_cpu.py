"""CPU checks of the long-speech entry points at their edges: refusals, the device of a call, the rotary table."""
import types

import pytest
import torch


def test_rotary_table_is_the_graphs_own():
    """From the graph's rotary module where it has one (an official graph), else from its configuration."""
    from flashb.engine import BackboneConfig, rope_table
    from flashb.long_speech import rotary_table
    cos, sin = rope_table(1e6, 128, 50, 'cpu')

    class Rotary:
        def __call__(self, x, pos):
            assert x.dtype == torch.bfloat16 and pos.tolist() == [list(range(50))]
            return cos.float()[None], sin.float()[None]
    official = types.SimpleNamespace(model=types.SimpleNamespace(rotary_emb=Rotary()))
    for g in (official, types.SimpleNamespace(cfg=BackboneConfig())):
        c, s = rotary_table(g, 50, 'cpu')
        assert torch.equal(c, cos) and torch.equal(s, sin) and c.dtype == torch.bfloat16 and c.is_contiguous()
