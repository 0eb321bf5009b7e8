"""GPU: surface_cross_entropy over the range of its arguments: incoming gradients, logits, features
and tables of any size, infinities, rows that are alike, derivatives of its gradients."""
import math

import pytest
import torch

from test_gpu_xent import _check, _reference

pytestmark = pytest.mark.gpu

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


def _run(x, e, y, scale, reduction, grad):
    from kaolin_amd.metrics.render import surface_cross_entropy
    x, e = x.detach().requires_grad_(True), e.detach().requires_grad_(True)
    loss = surface_cross_entropy(x, e, y, scale, reduction)
    return (loss.detach(), *torch.autograd.grad(loss, [x, e], grad))


def _subnormal_step(dt):
    return torch.finfo(dt).tiny * torch.finfo(dt).eps


@pytest.mark.parametrize('power', [-123, -119, -66, 66, 119, 123])
@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_incoming_gradients_scale_the_result(dname, power):
    """Incoming gradients times a power of two, zeros among them, give the gradients times it: the same
    digits, a subnormal result off by at most one of its steps and an infinite one where it must be."""
    dt, f = TYPES[dname], 2.0 ** power
    g = torch.Generator().manual_seed(20)
    n, V, D = 300, 20, 40
    e = torch.nn.functional.normalize(torch.randn(V, D, generator=g), dim=1)
    y = torch.randint(0, V, (n,), generator=g)
    # mostly wrong: the probability of a row that is not the label is next to 1
    x = e[(y + 1) % V] + 0.1 * torch.randn(n, D, generator=g)
    x, e, y = x.to(DEV, dt), e.to(DEV, dt), y.to(DEV)
    grad = torch.rand(n, generator=g).to(DEV) + 0.25
    grad[::3] = 0
    base = _run(x, e, y, 8.0, 'none', grad)
    got = _run(x, e, y, 8.0, 'none', grad * f)
    for a, b in zip(got[1:], base[1:]):
        want = (b.double() * f).to(dt)
        near = (a.double() - want.double()).abs() <= _subnormal_step(dt)
        assert (near | (a == want)).all(), float(a.float().abs().max())
        assert not torch.isnan(a).any()


@pytest.mark.parametrize('dname', ['f32', 'bf16'])
def test_features_whose_squares_vanish(dname):
    """Features of 1e-23, whose squares are 0 in 32 bits, and a scale of 1e22: logits of some hundred,
    whose exponentials need the running maximum."""
    dt = TYPES[dname]
    g = torch.Generator().manual_seed(21)
    n, V, D = 300, 50, 256
    x = torch.where(torch.rand(n, D, generator=g) < 0.5, -1e-23, 1e-23).to(DEV, dt)
    e = (torch.randn(V, D, generator=g) * 100).to(DEV, dt)
    y = torch.randint(0, V, (n,), generator=g).to(DEV)
    grad = torch.rand(n, generator=g).to(DEV) + 0.25
    want = list(_reference(x, e, y, 1e22, 'none', grad))
    assert 300 < float(want[0].max()) < 2000
    # A probability below 2^-126 is subnormal or 0 in 32 bits, off by at most that, and so is 1 - p of a
    # label whose logit is some 100 above the others: times |g| scale |e| (or |x|) a term.  The bounds of
    # _reference leave 1e-37 for it, which is for scales next to 1.
    gs = 2.0 ** -126 * 1e22 * grad.double()
    want[3] = want[3] + 2 * gs[:, None] * e.double().abs().sum(0)
    want[5] = want[5] + 2 * gs @ x.double().abs()
    got = _run(x, e, y, 1e22, 'none', grad)
    assert all(torch.isfinite(t).all() for t in got)
    _check(got, want)
