"""CPU: gradients without second derivatives raise where they are differentiated."""
import pytest
import torch

from kaolin_amd._derivatives import first_only


class _Cube(torch.autograd.Function):
    """x^3 whose gradient is first_only's."""

    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return x ** 3

    @staticmethod
    def backward(ctx, grad):
        x, = ctx.saved_tensors
        with torch.no_grad():
            out = 3 * x * x * grad
        return first_only('cube', (out,))[0]


def test_a_gradient_in_a_loss_raises():
    x = torch.tensor([2.0, 3.0], requires_grad=True)
    y = _Cube.apply(x).sum()
    g, = torch.autograd.grad(y, x, create_graph=True)
    assert torch.equal(g, torch.tensor([12.0, 27.0])) and g.requires_grad
    with pytest.raises(RuntimeError, match='cube: second derivatives'):
        (y + g.pow(2).sum()).backward()


def test_none_stays_none():
    a = torch.ones(2)
    out = first_only('x', (None, a, None))
    assert out[0] is None and out[2] is None and torch.equal(out[1], a)
    assert first_only('x', (None, None)) == (None, None)


def test_tangents_are_seen():
    import torch.autograd.forward_ad as fw
    from kaolin_amd._derivatives import has_tangent
    a = torch.ones(3)
    assert not has_tangent(a)
    with fw.dual_level():
        assert has_tangent(a, fw.make_dual(a, a))
        assert not has_tangent(a)
        with torch.no_grad():
            assert has_tangent(fw.make_dual(a, a))
