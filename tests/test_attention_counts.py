"""Counts past 32 bits: the C entry points take samples, heads, buckets and distances as int, and a count that wraps would be another
call's. Broadcast views make such counts without memory. No device calls: counts are checked before devices."""

from __future__ import annotations

import pytest
import torch

from boltz_mlx_amd import autograd as A
from boltz_mlx_amd import kernels as K

MANY = 2 ** 32 + 1  # 1 in 32 bits


def refused(what, call):
    with pytest.raises(ValueError, match="too many " + what):
        call()


@pytest.mark.parametrize("of", [K, A])
def test_attention_counts(of):
    x = torch.zeros(1, 1, 1)
    q = x.expand(MANY, 1, 8)
    refused("samples", lambda: of.attention(q, q, q, 1))
    refused("samples", lambda: of.attention(q, q, q, 1, multiplicity=MANY))
    wide = x.expand(1, 1, 8 * MANY)
    refused("heads", lambda: of.attention(wide, wide, wide, MANY))


def test_attention_bwd_counts():
    q = torch.zeros(1, 1, 8).expand(MANY, 1, 8)
    refused("samples", lambda: K.attention_bwd(q, q, q, q, 1, q, torch.zeros(1, 1, 1, 2).expand(MANY, 1, 1, 2)))


@pytest.mark.parametrize("of", [K, A])
def test_qk_norm_rope_counts(of):
    q, k = torch.zeros(1, 1).expand(1, 2 * MANY), torch.zeros(1, 2)
    refused("heads", lambda: of.qk_norm_rope(q, k, None, None, MANY))
    refused("heads", lambda: of.qk_norm_rope(k, q, None, None, 1))


@pytest.mark.parametrize("of", [K, A])
def test_rel_bias_counts(of):
    b, pos = K.rel_buckets([0], device="cpu"), torch.arange(1)
    refused("heads", lambda: of.rel_bias(torch.zeros(2, 1).expand(2, MANY), b, pos))
    refused("buckets", lambda: of.rel_bias(torch.zeros(1, 1).expand(MANY, 1), b._replace(count=MANY), pos))
    refused("distances", lambda: of.rel_bias(torch.zeros(2, 1), b._replace(lut=torch.empty(MANY, dtype=torch.uint8)), pos))


def test_rel_bias_bwd_counts():
    b, pos = K.rel_buckets([0], device="cpu"), torch.arange(1)
    refused("heads", lambda: K.rel_bias_bwd(torch.zeros(1, 1, 1).expand(MANY, 1, 1), b, pos))
