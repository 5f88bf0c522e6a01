"""Layer norm on the gfx950 kernels: `torch.nn.LayerNorm`'s arguments and state, and in `forward`
the residual add that stands in front of a pre-norm layer.

The norm's parameters are replicated, not sharded: a layer norm acts on whole rows, which every
tensor-parallel rank of the reference has at this place (its Linear gathers them), so there is no
counterpart in the reference, whose models use torch's own.
"""

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import ops


class _LayerNorm(torch.autograd.Function):
    """(y, h) of rows x, h = x or round(x + residual)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, h, mean, rstd = ops.layer_norm_fwd(x, weight, bias, eps, residual=residual)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if h is None else h, weight, mean, rstd)
        ctx.param_dtype = None if bias is None else bias.dtype
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        h, weight, mean, rstd = ctx.saved_tensors
        need_x, need_residual, need_weight, need_bias = ctx.needs_input_grad[:4]
        if dy is None:   # (only the sum was used)
            dx, dweight, dbias = dsum, None, None
        else:
            dx, dweight, dbias = ops.layer_norm_bwd(dy, h, weight, mean, rstd, dsum, need_x or need_residual, need_weight,
                                                    need_bias, ctx.param_dtype)
        return dx if need_x else None, dx if need_residual else None, dweight, dbias, None


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5, residual=None):
    """F.layer_norm with the same arguments, on the HIP kernels.  With `residual`: (norm(x + residual), x + residual),
    the sum rounded to its type and normalised as it is rounded.

    Parameters are of x's type or fp32; under autocast the norm is fp32, as torch's is (64 bits are refused with and without)."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not shape or tuple(x.shape[x.dim() - len(shape):]) != shape:
        raise ValueError("layer_norm: expected the last dimensions to be %s, got %s" % (shape, tuple(x.shape)))
    for p in (weight, bias):
        if p is not None and tuple(p.shape) != shape:
            raise ValueError("layer_norm: parameter is %s, expected %s" % (tuple(p.shape), shape))
    if residual is not None and residual.shape != x.shape:
        raise ValueError("layer_norm: residual is %s, expected %s" % (tuple(residual.shape), tuple(x.shape)))
    if torch.is_autocast_enabled("cuda"):
        x, residual, weight, bias = (t.float() if t is not None and t.dtype in (torch.float16, torch.bfloat16) else t
                                     for t in (x, residual, weight, bias))
    rows, n = x.shape, math.prod(shape)
    as_rows = [t if t is None else t.reshape(-1, n) for t in (x, residual)]
    params = [p if p is None else p.reshape(-1) for p in (weight, bias)]
    # (without gradients too the autograd function is what refuses a tangent, for which it has no rule, and what a trace
    # records; a trace may run with gradients later, so that the function always keeps what they need)
    if torch.is_grad_enabled() or forward_ad._current_level >= 0 or torch.jit.is_tracing():
        out = _LayerNorm.apply(*as_rows, *params, eps)
    else:
        y, h, _, _ = ops.layer_norm_fwd(as_rows[0], *params, eps, residual=as_rows[1], save=False)
        out = y if h is None else (y, h)
    return out.reshape(rows) if residual is None else (out[0].reshape(rows), out[1].reshape(rows))


class LayerNorm(torch.nn.Module):
    """`torch.nn.LayerNorm`'s arguments, parameters and state dict.  `forward(x)` is norm(x);
    `forward(x, residual)` is (norm(x + residual), x + residual)."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__()
        self.normalized_shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
        self.eps, self.elementwise_affine = eps, elementwise_affine
        self.weight = self.bias = None
        if elementwise_affine:
            self.weight = torch.nn.Parameter(torch.ones(self.normalized_shape, device=device, dtype=dtype))
            if bias:
                self.bias = torch.nn.Parameter(torch.zeros(self.normalized_shape, device=device, dtype=dtype))

    def forward(self, x, residual=None):
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps, residual)

    def extra_repr(self):
        return "%s, eps=%g, elementwise_affine=%s, bias=%s" % (self.normalized_shape, self.eps, self.elementwise_affine,
                                                               self.bias is not None)
