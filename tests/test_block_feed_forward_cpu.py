"""``mlp`` in a block's configuration: what says that there is none, what is refused, and where."""
from __future__ import annotations

from collections import OrderedDict

import pytest

from semambaxlinoss_b200.mamba_block import MambaBlock, create_block

CFG = {"ssm": "gated_lru", "d_state": 4, "d_conv": 3, "expand": 2}


@pytest.mark.parametrize("none", [None, False])
def test_no_feed_forward_half(none):
    assert create_block(16, dict(CFG, mlp=none)).mlp is None
    block = MambaBlock(16, dict(CFG, mlp=none, bidirectional=False)).forward_blocks[0]
    assert block.mlp is None and not hasattr(block, "norm2")
    hybrid = {"ssm": "hybrid", "mlp": none, "backbone_1": dict(CFG, mlp=none), "backbone_2": CFG}
    assert create_block(16, hybrid).norm2 is not None


@pytest.mark.parametrize("bad", [True, 1, 0, "silu", 128, [], ("silu",)])
def test_what_is_no_configuration_is_refused(bad):
    with pytest.raises(ValueError, match="mlp must be"):
        create_block(16, dict(CFG, mlp=bad))
    with pytest.raises(ValueError, match="mlp must be"):
        MambaBlock(16, dict(CFG, mlp=bad))


def test_any_mapping_is_taken():
    assert create_block(16, dict(CFG, mlp=OrderedDict(hidden_features=24))).mlp.fc1.weight.shape == (48, 16)


@pytest.mark.parametrize("where", ["backbone_1", "backbone_2"])
def test_backbones_refuse_a_feed_forward_half(where):
    cfg = {"ssm": "hybrid", "backbone_1": CFG, "backbone_2": CFG}
    cfg[where] = dict(CFG, mlp={})
    with pytest.raises(ValueError, match="feed-forward"):
        create_block(16, cfg)
