"""The training operators with gradients: LayerNorm, dropout and the residual update, as autograd nodes of the torch binding
(csrc/bzpf_torch.cpp) over the kernels that boltz_mlx_amd.kernels offers without gradients. (The modules of
boltz_mlx_amd.layers run inference only, as the reference does; layers.norm and layers.dropout offer these functions.)

Once differentiable: a backward pass with create_graph raises. What a function saves is its input (the residual update:
its output z_new), the weight and the generator's state; changing one of them in place before the backward pass, with torch
or with a wrapper of boltz_mlx_amd.kernels that writes its argument, raises torch's error there, so advance the generator (rng[1] += 1) after the step's backward pass.

To capture a step into a HIP graph, run no eager backward pass over the same leaves whose graph is still alive, and take
the gradients inside the capture with torch.autograd.grad (or call the *_bwd functions of boltz_mlx_amd.kernels).
"""

from __future__ import annotations

import torch

from boltz_mlx_amd import kernels as K


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, out_dtype=torch.float32) -> torch.Tensor:
    """kernels.layer_norm with gradients for x, weight and bias."""
    return K.call("grad_layer_norm", x, weight, bias, eps, out_dtype)


def dropout(x: torch.Tensor, p: float, rng, site: int = 0, shared=None) -> torch.Tensor:
    """kernels.dropout with its gradient: the same draws on the output's gradient, formed again from (rng, site)."""
    return K.call("grad_dropout", x, p, rng, site, K._shared("dropout", shared))


def dropout_add_ln(z: torch.Tensor, y: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, p: float = 0.0, rng=None,
                   site: int = 0, shared=None, out_dtype=None):
    """kernels.dropout_add_ln, (z + dropout(y), its LayerNorm), with gradients for z, y, weight and bias; the backward
    pass is one kernel (and the sum of the parameters' partial gradients)."""
    return K.call("grad_dropout_add_ln", z, y, weight, bias, eps, p, rng, site, K._shared("dropout_add_ln", shared),
                  out_dtype)
