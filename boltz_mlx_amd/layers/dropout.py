"""Dropout of the trunk's training recipe: the layers' updates of the pair and MSA streams are dropped with one draw for
each row of pairs, each column, or each element, scaled by 1 / (1 - p) and added to the stream. (The reference runs
inference only: its layers keep a `dropout` argument that nothing reads, boltz_mlx/layers/pairformer.py:23-57.)
"""

from __future__ import annotations

import torch

from boltz_mlx_amd import autograd as A


class Dropout(torch.nn.Module):
    """Drops in training mode and passes its input on in evaluation mode. shared: None (each element has a draw), "row" or
    "column" (one for each row / column of a [.., I, J, D] tensor). site: this module's place in the model (0 to 65535);
    modules with the same site and generator state draw alike."""

    def __init__(self, p: float, shared=None, site: int = 0) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"Dropout: p must lie in [0, 1], got {p}")
        self.p, self.shared, self.site = float(p), shared, site

    def extra_repr(self) -> str:
        return f"p={self.p}, shared={self.shared!r}, site={self.site}"

    def forward(self, x: torch.Tensor, rng: torch.Tensor) -> torch.Tensor:
        """rng: the step's generator state (kernels.dropout_rng)."""
        return A.dropout(x, self.p, rng, self.site, self.shared) if self.training and self.p > 0 else x

    def add_ln(self, z: torch.Tensor, y: torch.Tensor, ln, rng: torch.Tensor, out_dtype=None):
        """(z + self(y), ln of that) in one kernel: a layer's update of the fp32 stream z and the next module's LayerNorm
        (ln: a LayerNorm module, whose output takes out_dtype, by default y's type)."""
        return A.dropout_add_ln(z, y, ln.weight, ln.bias, ln.eps, self.p if self.training else 0.0, rng, self.site,
                                self.shared, out_dtype)
