"""``mask_iou`` -- drop-in for kaolin/metrics/render.py:18-40.

The silhouette loss of the DIB-R training step (examples/tutorial/ian_dibr.py:264-265):
``1 - mean_b(sum(l * r) / (sum(l + r - l * r) + 1e-10))``.  Forward: one HIP pass over both masks
(per-view fp64 partial sums, ordered finish, no host sync); backward: one elementwise HIP pass
(kaolin_amd/csrc/kd_metrics.hip).  The sums are accumulated in fp64, so fp32 results agree with
the reference's fp32 reductions to their rounding error, not bit for bit.

``surface_cross_entropy`` -- the loss that ties pixel features to a rendered mesh: the softmax
cross entropy of each pixel's features against a table of embeddings with a row per face (or
vertex), at the ``face_idx`` of a rasterization (kaolin_amd/csrc/kd_xent.hpp).  The (pixels, rows)
logits are never stored.
"""
import torch
from torch.autograd import Function

from .. import _C
from .._derivatives import first_only, has_tangent

__all__ = ['mask_iou', 'surface_cross_entropy']


class MaskIouHip(Function):
    """torch.autograd.Function over kd_mask_iou_forward / kd_mask_iou_backward."""

    @staticmethod
    def forward(ctx, lhs_mask, rhs_mask):
        loss, stats, _ = _C.mask_iou_forward(lhs_mask, rhs_mask)
        ctx.save_for_backward(lhs_mask, rhs_mask, stats)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        lhs, rhs, stats = ctx.saved_tensors
        gl, gr = _C.mask_iou_backward(grad_loss, lhs, rhs, stats, ctx.needs_input_grad[0],
                                      ctx.needs_input_grad[1])
        return gl, gr


def mask_iou(lhs_mask, rhs_mask):
    r"""Compute the Intersection over Union of two segmentation masks
    (kaolin/metrics/render.py:18-40).

    Args:
        lhs_mask (torch.Tensor): (batch_size, height, width), float32 or float64, on a GPU.
        rhs_mask (torch.Tensor): same shape.

    Returns:
        (torch.Tensor): the IoU loss, a scalar.
    """
    batch_size, height, width = lhs_mask.shape
    assert rhs_mask.shape == lhs_mask.shape
    return MaskIouHip.apply(lhs_mask, rhs_mask)


class SurfaceCrossEntropyHip(Function):
    """torch.autograd.Function over kd_surface_xent_forward / _backward."""

    @staticmethod
    def forward(ctx, features, embeddings, labels, scale, reduction):
        need = ctx.needs_input_grad[:2]
        loss, state = _C.metrics.surface_xent_forward(features, embeddings, labels, scale,
                                                      reduction, *need)
        ctx.save_for_backward(labels, state)
        ctx.shape, ctx.dtype, ctx.need = embeddings.shape, features.dtype, need
        ctx.scale, ctx.reduction = scale, reduction
        ctx.set_materialize_grads(False)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        if not torch.is_grad_enabled():
            return _grad(ctx, grad_loss)
        with torch.no_grad():
            grads = _grad(ctx, grad_loss)
        return first_only('surface_cross_entropy', grads)


def _grad(ctx, grad_loss):
    if grad_loss is None:
        return (None,) * 5
    if has_tangent(grad_loss):
        raise NotImplementedError('surface_cross_entropy: no forward mode')
    labels, state = ctx.saved_tensors
    gx, ge = _C.metrics.surface_xent_backward(
        grad_loss, labels, ctx.shape, ctx.dtype, ctx.scale, ctx.reduction, state, *ctx.need,
        *ctx.needs_input_grad[:2])
    return gx, ge, None, None, None


def surface_cross_entropy(features, embeddings, labels, scale=1.0, reduction='mean'):
    r"""Softmax cross entropy of pixel features against every row of a table of embeddings:
    ``cross_entropy(scale * features @ embeddings.T, labels)`` over the pixels whose label names
    a row, without the logits.

    Args:
        features (torch.Tensor): (\*labels.shape, num_channels), float32, float16 or bfloat16, on
            a GPU; 1 to 256 channels.
        embeddings (torch.Tensor): (num_rows, num_channels), the same type: a row per face or
            vertex.
        labels (torch.Tensor): any shape, int64, e.g. the (batch_size, height, width) ``face_idx``
            of :func:`kaolin_amd.render.mesh.dibr_rasterization`.  Values outside [0, num_rows) (the
            background, -1) take no part: no loss, zero gradient, whatever the features hold.
        scale (float): the logits' factor (an inverse temperature).
        reduction (str): 'mean' over the pixels that take part (0 if there are none), 'sum', or
            'none' (a loss per pixel, 0 where the label names no row).

    Returns:
        (torch.Tensor): the loss, float32.  Gradients come in the inputs' type; logits, sums and
        the loss are held in 32 bits.  16-bit probabilities enter the gradients' products rounded
        to the inputs' type.  Second derivatives raise a RuntimeError,
        forward mode a NotImplementedError.
    """
    if not (torch.is_grad_enabled() and (features.requires_grad or embeddings.requires_grad)) \
            and not has_tangent(features, embeddings):
        return _C.metrics.surface_xent_forward(features, embeddings, labels, scale, reduction)[0]
    return SurfaceCrossEntropyHip.apply(features, embeddings, labels, scale, reduction)
