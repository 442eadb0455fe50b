"""Positions in the sequence attention, for training and fine-tuning: a learned relative position bias by buckets and the norms
of queries and keys for each head with the position rotation. (The reference's attention takes neither: its pair bias comes
from z alone, boltz_mlx/layers/attentionv2.py:59-83.) AttentionPairBias.with_grad takes both.
"""

from __future__ import annotations

import torch

from boltz_mlx_amd import autograd as A
from boltz_mlx_amd import kernels as K


class RelativeBias(torch.nn.Module):
    """A bias [(B,) H, N, N] for the attention, learned for each bucket of the tokens' distance: one for each distance from
    -reach to reach, those beyond in the last ones (or the buckets between the integers `edges`), and one for tokens of
    different chains. Zero at first."""

    def __init__(self, num_heads: int, reach: int = 32, edges=None) -> None:
        super().__init__()
        b = K.rel_buckets(K.clipped_edges(reach) if edges is None else edges, other=True, device="cpu")
        self.lo, self.count = b.lo, b.count
        self.register_buffer("lut", b.lut, persistent=False)
        self.table = torch.nn.Parameter(torch.zeros(b.count, num_heads))

    def buckets(self) -> K.RelBuckets:
        return K.RelBuckets(self.lut, self.lo, self.count, True)

    def forward(self, pos: torch.Tensor, chain=None, add=None, out_dtype=None) -> torch.Tensor:
        """pos: int32 or int64 [N] or [B, N]; chain: of pos's shape and type; add: a pair bias of the output's shape and type, added in the same pass.
        With gradients for the table and add."""
        return A.rel_bias(self.table, self.buckets(), pos, group_q=chain, add=add, out_dtype=out_dtype)


class QKNorm(torch.nn.Module):
    """The norms of queries and keys for each head of `head_dim` channels, with weights for each, and the rotation of the first
    `rotary` channels (default all) by the token's position."""

    def __init__(self, head_dim: int, eps: float = 1e-5, base: float = 10000.0, rotary=None, interleaved: bool = False) -> None:
        super().__init__()
        self.head_dim, self.eps, self.base, self.rotary, self.interleaved = head_dim, eps, base, rotary, interleaved
        self.q_weight = torch.nn.Parameter(torch.ones(head_dim))
        self.k_weight = torch.nn.Parameter(torch.ones(head_dim))

    def forward(self, q: torch.Tensor, k: torch.Tensor, pos=None, out_dtype=None):
        """q, k [.., H * head_dim] -> the same, contiguous, in out_dtype (default theirs), with gradients; pos as in
        kernels.qk_norm_rope."""
        return A.qk_norm_rope(q, k, self.q_weight, self.k_weight, q.shape[-1] // self.head_dim, pos, self.eps, self.base,
                              self.rotary, self.interleaved, out_dtype)
