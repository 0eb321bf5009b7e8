"""What an autograd function without second derivatives or a forward mode has to refuse."""
import torch
from torch.autograd import Function
from torch.autograd.forward_ad import unpack_dual

__all__ = ['first_only', 'has_tangent']


def has_tangent(*tensors):
    """Whether one of them is dual (torch.autograd.forward_ad).  Such a tensor need not require a
    gradient, and its data can be read like any other's: an operator that leaves autograd out would
    give a result without a tangent."""
    return any(unpack_dual(t).tangent is not None for t in tensors)


class _FirstOnly(Function):
    """Hands gradients on; differentiating them raises."""

    @staticmethod
    def forward(ctx, name, anchor, *grads):
        ctx.name = name
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f'{ctx.name}: second derivatives are not implemented')


def first_only(name, grads):
    """The gradients of a backward call that is recorded (create_graph): they depend on the inputs, so
    they come with a graph, one that raises.  (torch's once_differentiable gives them none where the
    incoming gradient needs none, and a term of theirs in a loss is then left out silently.)"""
    here = [i for i, g in enumerate(grads) if g is not None]
    grads = list(grads)
    if here:
        anchor = torch.empty((), requires_grad=True)
        for i, g in zip(here, _FirstOnly.apply(name, anchor, *[grads[i] for i in here])):
            grads[i] = g
    return tuple(grads)
