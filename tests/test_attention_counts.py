"""Counts past 32 bits: the C entry points take samples, heads, buckets and distances as int, and a count that wraps would be another
call's. Broadcast views make such counts without memory. No device calls: counts are checked before devices."""

from __future__ import annotations

import pytest
import torch

from boltz_mlx_amd import _lib
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


def test_workspace_sizes_of_what_is_refused():
    """Sizes whose products pass 64 bits, and such as no launch holds: -1, from the questions as from the calls."""
    lib = _lib.load()
    for S, H, N, M in ((1 << 27, 1 << 15, 1 << 22, 1), (1 << 26, 1 << 15, 1 << 22, 1), (2 ** 31 - 1, 65535, 1 << 22, 1 << 22), (2 ** 31 - 1, 65535, 1, 1),
                       (1 << 20, 16, 5, 7), (4, 129, 1 << 22, 7), (128, 3, 5, 1 << 22)):
        assert lib.bzpf_attention_ws(S, H, 8, N, M) == -1, (S, H, N, M)
        assert lib.bzpf_attention_bwd_ws(1, S, H, 8, N, M, 1) == -1, (S, H, N, M)
    assert lib.bzpf_attention_ws(1, 1, 128, 1 << 22, 1 << 22) == 0 < lib.bzpf_attention_bwd_ws(0, 1, 1, 128, 1 << 22, 1 << 22, 1)
    assert lib.bzpf_rel_bias_bwd_ws(65535, 65535, 1, 1 << 29, 256) == -1 == lib.bzpf_rel_bias_bwd_ws(65535, 17, 1, 1, 8)
    assert lib.bzpf_rel_bias_bwd_ws(65535, 16, 1, 1, 8) > 0
