"""Root-mean-square norm in front of the MoE MLP, differentiable (the reference's examples take their norms from torch)."""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import ops


class _RMSNorm(torch.autograd.Function):
    """(y, total): one HIP kernel each way, and a small one for the weight gradient."""

    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        n = ops.rms_norm(x, weight, eps, residual=residual, want_rstd=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(n.total, weight, n.rstd)
        return (n.y, n.total) if residual is not None else n.y

    @staticmethod
    def backward(ctx, grad_y, grad_total=None):
        # (the decorator costs as much host time as a launch, and says nothing where no graph is made of the backward)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad_y, grad_total)


def _backward(ctx, grad_y, grad_total):
    total, weight, rstd = ctx.saved_tensors
    need_x, need_w, _, need_r = ctx.needs_input_grad
    if grad_y is None:                                   # y was not used
        return grad_total if need_x else None, None, None, grad_total if need_r else None
    # shapes and types are the forward's, which it checked
    g_x, g_w = ops._rms_norm_backward(grad_y.contiguous(), total, weight, rstd, None if grad_total is None else grad_total.contiguous(),
                                      need_x or need_r, need_w, ops._type_code(total, "total"))
    return g_x if need_x else None, g_w, None, g_x if need_r else None


_backward_once = once_differentiable(_backward)


def rms_norm(x, weight, eps=1e-5, residual=None):
    """y = total / sqrt(mean(total^2) + eps) * weight over the last dimension, total = x + residual rounded to x's type.
    Returns y, or (y, total) with a residual, both differentiable."""
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    weight = weight.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        return _RMSNorm.apply(x, weight, float(eps), residual)
    n = ops.rms_norm(x, weight, eps, residual=residual)
    return n.y if residual is None else (n.y, n.total)


class RMSNorm(nn.Module):
    """``rms_norm`` with its weight.  ``forward(x)`` gives y, ``forward(x, residual)`` (y, x + residual)."""

    def __init__(self, d_model, eps=1e-5):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(d_model))

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, self.eps, residual)

    def extra_repr(self):
        return f"{self.weight.shape[0]}, eps={self.eps}"
