"""``surface_embedding``: a learned table with a row per face (or vertex) of a mesh, looked up at the
``face_idx`` image of a rasterization or at the faces' corners.

In plain PyTorch this is ``scale * embeddings[index]`` with the background masked, whose gradient
is an unordered scatter.  Here the forward is one HIP pass and the backward sorts the indices and
adds each row's gradients in the indices' order (kaolin_amd/csrc/kd_embedding.hip): the same bits
on every run.
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ... import _C
from ..._derivatives import has_tangent

__all__ = ['surface_embedding']


class SurfaceEmbeddingHip(Function):
    """torch.autograd.Function over kd_surface_embedding_forward / _backward."""

    @staticmethod
    def forward(ctx, index, embeddings, scale):
        out, ctx.plan = _C.render.mesh.surface_embedding_forward(index, embeddings, scale, True)
        ctx.save_for_backward(index)
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        # (the guard against second derivatives costs time that a plain backward need not spend)
        return _guarded_grad(ctx, grad_out) if torch.is_grad_enabled() else _grad(ctx, grad_out)


def _grad(ctx, grad_out):
    if grad_out is None:
        return None, None, None
    if has_tangent(grad_out):
        raise NotImplementedError('surface_embedding: no forward mode')
    index, = ctx.saved_tensors
    return None, _C.render.mesh.surface_embedding_backward(grad_out, index, ctx.plan), None


_guarded_grad = once_differentiable(_grad)


def surface_embedding(index, embeddings, scale=1.0):
    r"""Look up a table of embeddings at a face (or vertex) index: ``scale * embeddings[index]``,
    zeros where the index names no row.

    With the ``face_idx`` of :func:`rasterize` / :func:`dibr_rasterization` this renders per-face
    features into the image (the background, -1, is zero); with a mesh's ``faces`` (F, 3) it
    gathers per-vertex features to the (F, 3, D) corners that a rasterizer takes.

    Args:
        index (torch.Tensor): any shape, int64, on a GPU.  Values outside [0, num_rows) name no
            row: they give zeros and take no part in the gradient.
        embeddings (torch.Tensor): (num_rows, num_channels), or (batch_size, num_rows,
            num_channels) with index of shape (batch_size, ...): a table per batch entry.
            float32, float64, float16 or bfloat16.
        scale (float): a common factor.

    Returns:
        (torch.Tensor): (\*index.shape, num_channels), in embeddings' type; products are rounded
        to it once, and the gradient's sums are held in 32 bits (64 for float64).  Forward mode
        raises a NotImplementedError.
    """
    if not (torch.is_grad_enabled() and embeddings.requires_grad) and not has_tangent(embeddings):
        return _C.render.mesh.surface_embedding_forward(index, embeddings, scale)[0]
    return SurfaceEmbeddingHip.apply(index, embeddings, scale)
