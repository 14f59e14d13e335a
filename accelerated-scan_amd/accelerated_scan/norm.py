"""Gated norm of rows, the norm behind the scan of a gated layer.

``gated_norm(x, gate, weight)`` equals
``x * rsqrt(mean(x**2, -1) + eps) * weight * silu(gate)`` in one pass over memory, forward and backward: the
outputs of ``delta.gated_delta_scan`` or ``delta.gated_delta_step`` are normalised per head and gated by a
projection of the layer's input before they leave it.  In elementary operations the same is a dozen passes.
The reference has no operator of this kind.
"""

import torch
from torch.autograd.function import once_differentiable

from . import _abi, _ops

_REAL_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, gate, weight):
    """The passing case builds no message."""
    _ops.no_tangents(x, gate, weight)
    dtype, device, shape = x.dtype, x.device, x.shape
    if (dtype in _REAL_DTYPES and gate.dtype == dtype and weight.dtype == dtype and gate.shape == shape
            and weight.shape == shape[-1:] and len(shape) > 0 and x.is_cuda and gate.device == device
            and weight.device == device and x.is_contiguous() and gate.is_contiguous() and weight.is_contiguous()):
        return
    if x.dim() < 1 or gate.shape != x.shape or weight.shape != x.shape[-1:]:
        raise RuntimeError(
            f"accelerated_scan: expected x and gate of one shape and weight of its last axis, got {tuple(x.shape)}, "
            f"{tuple(gate.shape)} and {tuple(weight.shape)}"
        )
    if x.dtype not in _REAL_DTYPES or gate.dtype != x.dtype or weight.dtype != x.dtype:
        raise RuntimeError(
            f"accelerated_scan: unsupported tensor dtypes {x.dtype}, {gate.dtype}, {weight.dtype}: expecting x, gate "
            "and weight all bfloat16, float16 or float32"
        )
    for name, t in (("x", x), ("gate", gate), ("weight", weight)):
        if not t.is_cuda or t.device != x.device:
            raise RuntimeError(f"accelerated_scan: expected {name} to be a device tensor on the device of x")
        if not t.is_contiguous():
            raise RuntimeError(f"accelerated_scan: expected {name} to be contiguous")


def _forward(x, gate, weight, eps):
    if _ops.capturing():
        return _ops.gated_norm(x, gate, weight, eps)
    out = torch.empty_like(x)
    if x.numel():
        _abi.gated_norm(x, gate, weight, eps, out)
    return out


class GatedNorm(torch.autograd.Function):
    """Autograd node: saves the inputs, recomputes the norm."""

    @staticmethod
    def forward(ctx, x, gate, weight, eps):
        ctx.save_for_backward(x, gate, weight)
        ctx.eps = eps
        return _forward(x, gate, weight, eps)

    @staticmethod
    def backward(ctx, d_out):
        if torch.is_grad_enabled() and not _ops.capturing():  # create_graph: no second derivatives
            return once_differentiable(_gradients)(ctx, d_out)
        return _gradients(ctx, d_out)


def _gradients(ctx, d_out):
    x, gate, weight = ctx.saved_tensors
    return (*_ops.gated_norm_backward_run(x, gate, weight, d_out.contiguous(), ctx.eps), None)


def gated_norm(x, gate, weight, eps=1e-6):
    """Normalise the rows of ``x`` by their root mean square, scale them by ``weight`` and gate them.

    Arguments:
        x (torch.Tensor): shape (..., width), contiguous; fp32, bf16 or fp16.
        gate (torch.Tensor): the shape and dtype of x, contiguous; enters as ``gate * sigmoid(gate)``.
        weight (torch.Tensor): shape (width,), the dtype of x.
        eps (float): added to the mean of the squares.

    Returns:
        (torch.Tensor): the shape of x; differentiable once, in reverse mode, in x, gate and weight.
    """
    _check(x, gate, weight)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or weight.requires_grad):
        return GatedNorm.apply(x, gate, weight, float(eps))
    return _forward(x, gate, weight, float(eps))
