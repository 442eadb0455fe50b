"""The attention module's positions on the host: what it refuses before any kernel."""

from __future__ import annotations

import pytest
import torch

from boltz_mlx_amd.layers.attentionv2 import AttentionPairBias
from boltz_mlx_amd.layers.positions import RelativeBias


def test_position_bias_without_positions():
    m = AttentionPairBias(32, None, 2, compute_pair_bias=False)
    with pytest.raises(ValueError, match="rel_bias needs pos"):
        m.with_grad(torch.zeros(1, 5, 32), None, torch.ones(1, 5), rel_bias=RelativeBias(2))
