"""CPU: ``prefill_attention="chunk"`` is refused where its attention does not serve, before anything is
allocated."""

from types import SimpleNamespace

import pytest

from superl8_serve_b200.config import tiny
from superl8_serve_b200.engine import DecodePipeline


@pytest.mark.parametrize("block_size", [0, 12, 48, 512])
def test_block_sizes(block_size):
    with pytest.raises(ValueError, match="power of two"):
        DecodePipeline([SimpleNamespace(cfg=tiny())], batch=1, block_size=block_size,
                       prefill_attention="chunk")


@pytest.mark.parametrize("kw", [{"head_dim": 64}, {"num_attention_heads": 258, "num_key_value_heads": 2}])
def test_heads(kw):
    with pytest.raises(ValueError, match="head_dim of 128"):
        DecodePipeline([SimpleNamespace(cfg=tiny(**kw))], batch=1, prefill_attention="chunk")
