"""The training operators with gradients: LayerNorm, dropout, the residual update and the sequence attention with its
positions, as autograd nodes of the torch binding (csrc/bzpf_torch.cpp, csrc/bzpf_torch_attn.cpp) over the kernels that
boltz_mlx_amd.kernels offers without gradients. (The modules of boltz_mlx_amd.layers run inference only, as the reference
does, but for their with_grad functions; layers.norm, layers.dropout and layers.positions offer these.)

Once differentiable: a backward pass with create_graph raises. What a function saves is its inputs (the residual update:
its output z_new and the weight; the attention: its output and two numbers a row too) and the generator's state; changing one
of them in place before the backward pass, with torch or with a wrapper of boltz_mlx_amd.kernels that writes its argument,
raises torch's error there, so advance the generator (rng[1] += 1) after the step's backward pass.

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


def rel_bias(table: torch.Tensor, buckets: K.RelBuckets, pos_q, pos_k=None, group_q=None, group_k=None, add=None,
             out_dtype=None) -> torch.Tensor:
    """kernels.rel_bias with gradients for table and add."""
    return K.call("grad_rel_bias", table, *buckets, pos_q, pos_k, group_q, group_k, add, out_dtype)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, w_q, w_k, H: int, pos=None, eps: float = 1e-5, base: float = 10000.0,
                 rotary=None, interleaved: bool = False, out_dtype=None):
    """kernels.qk_norm_rope with gradients for q, k and the weights; the norms are formed again in the backward pass."""
    return K.call("grad_qk_norm_rope", q, k, w_q, w_k, H, pos, eps, base, rotary, interleaved, out_dtype)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, H: int, g=None, bias=None, mask=None,
              multiplicity: int = 1) -> torch.Tensor:
    """kernels.attention's output with gradients for q, k, v, g and bias. It saves these, its output and two numbers a row: no
    probabilities."""
    return K.call("grad_attention", q, k, v, H, g, bias, mask, multiplicity)
