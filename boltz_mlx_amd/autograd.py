"""The training operators with gradients: LayerNorm, dropout and the residual update, as torch.autograd functions over
the kernels of boltz_mlx_amd.kernels (the modules of boltz_mlx_amd.layers run inference only, as the reference does).

Once differentiable: the gradients themselves carry no graph. What a function saves is its input (the residual update:
its output z_new), the weight and the generator's state; changing one of them in place before the backward pass raises
torch's error, so advance the generator (rng[1] += 1) after the step's backward pass.

To capture a step into a HIP graph, run no eager backward pass over the same leaves whose graph is still alive, and take
the gradients inside the capture with torch.autograd.grad (or call the *_bwd kernels).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from boltz_mlx_amd import kernels as K


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        x = x.contiguous()
        ctx.save_for_backward(x, weight)
        ctx.eps, ctx.bias_dtype = eps, None if bias is None else bias.dtype
        return K.layer_norm(x, weight, bias, eps, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dx, dw, db = K.layer_norm_bwd(dy, x, weight, ctx.eps, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return dx, _as(dw, weight), _as(db, ctx.bias_dtype), None, None


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, site, shared):
        ctx.save_for_backward(rng)
        ctx.args = p, site, shared
        return K.dropout(x, p, rng, site, shared)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, site, shared = ctx.args
        return K.dropout(dy, p, ctx.saved_tensors[0], site, shared), None, None, None, None


class _DropoutAddLN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, y, weight, bias, eps, p, rng, site, shared, out_dtype):
        z_new, ln = K.dropout_add_ln(z, y, weight, bias, eps, p, rng, site, shared, out_dtype)
        ctx.save_for_backward(z_new, weight, rng)
        ctx.args = eps, p, site, shared, y.dtype, None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return z_new, ln

    @staticmethod
    @once_differentiable
    def backward(ctx, dz_new, dln):
        z_new, weight, rng = ctx.saved_tensors
        eps, p, site, shared, y_dtype, bias_dtype = ctx.args
        dz = dy = dw = db = None
        if dln is not None:
            dz, dy, dw, db = K.dropout_add_ln_bwd(dz_new, dln, z_new, weight, eps, p, rng, site, shared, y_dtype,
                                                  ctx.needs_input_grad[2], ctx.needs_input_grad[3])
        elif dz_new is not None:  # the LayerNorm's output was not used
            dz, dy = dz_new, K.dropout(dz_new, p, rng, site, shared, out_dtype=y_dtype)
        return dz, dy, _as(dw, weight), _as(db, bias_dtype), None, None, None, None, None, None


def _as(grad, like):
    """A parameter's gradient in its type (`like`: the parameter, or its type)."""
    return None if grad is None else grad.to(like.dtype if isinstance(like, torch.Tensor) else like)


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, out_dtype=torch.float32) -> torch.Tensor:
    """kernels.layer_norm with gradients for x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps, out_dtype)


def dropout(x: torch.Tensor, p: float, rng, site: int = 0, shared=None) -> torch.Tensor:
    """kernels.dropout with its gradient: the same draws on the output's gradient, formed again from (rng, site)."""
    return _Dropout.apply(x, p, rng, site, shared)


def dropout_add_ln(z: torch.Tensor, y: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, p: float = 0.0, rng=None,
                   site: int = 0, shared=None, out_dtype=None):
    """kernels.dropout_add_ln, (z + dropout(y), its LayerNorm), with gradients for z, y, weight and bias; the backward
    pass is one kernel (and the sum of the parameters' partial gradients)."""
    return _DropoutAddLN.apply(z, y, weight, bias, eps, p, rng, site, shared, out_dtype)
