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


LARGE = [(dname, D, size) for dname in ('f32', 'f16', 'bf16') for D in (16, 64, 130, 256)
         for size in (10.0, 300.0, 1e4, 1e9, 1e16) if dname != 'f16' or size < 1e4]


@pytest.mark.parametrize('dname,D,size', LARGE)
def test_large_logits_choose_one_row(dname, D, size):
    """Logits of 1e3 to 1e33 in pixels whose largest logit is so far above the others that their
    probabilities are below exp(-50), V of them below `rest`: the loss is the difference of two logits, the gradients are those of a
    choice.  A logit is off by dz (see test_gpu_xent), a probability of 1 by its rounding and that of an
    exponential near 0, 2^-21 in all, and the sums are of exact terms."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    dt, scale = TYPES[dname], 0.75
    g = torch.Generator().manual_seed(22)
    n, V = 700, 150
    x = (torch.randn(n, D, generator=g) * size).to(DEV, dt)
    e = (torch.randn(V, D, generator=g) * size).to(DEV, dt)
    y = torch.randint(0, V, (n,), generator=g).to(DEV)
    grad = ((torch.rand(n, generator=g) + 0.25) / 1024).to(DEV)
    z = scale * (x.double() @ e.double().t())
    dz = ((6 if dname == 'f32' else 1) * D + 8) * 2.0 ** -24 * scale * (
        x.double().abs() @ e.double().abs().t()).amax(1)
    top, best = z.topk(2, 1)
    clear = top[:, 0] - top[:, 1] > 2 * dz + 50
    assert clear.sum() > 20
    y = torch.where(clear, y, -1)
    y[:40] = torch.where(clear[:40], best[:40, 0], -1)  # some of them right
    u = torch.finfo(dt).eps / 2
    ok = (y >= 0).double()
    want = ok * (top[:, 0] - z[torch.arange(n, device=DEV), y.clamp(min=0)])
    gs = grad.double() * scale * ok
    hot = torch.zeros(n, V, dtype=torch.float64, device=DEV)
    hot[torch.arange(n, device=DEV), best[:, 0]] += 1
    hot[torch.arange(n, device=DEV), y.clamp(min=0)] -= 1
    gx = gs[:, None] * (hot @ e.double())
    ge = (hot * gs[:, None]).t() @ x.double()
    up = u if dname != 'f32' else 2.0 ** -23
    small = 2.0 ** -25 if dname == 'f16' else 1e-37
    # what the other rows add: to the loss, and to a gradient times the largest element
    rest = V * math.exp(-50)
    tx = (up + 2.0 ** -21) * gs[:, None] * (hot.abs() @ e.double().abs()) + u * gx.abs() + small \
        + rest * gs[:, None] * e.double().abs().max()
    te = (up + (n + 32) * 2.0 ** -24) * (hot.abs() * gs[:, None]).t() @ x.double().abs() \
        + u * ge.abs() + small + rest * gs.sum() * x.double().abs().max()
    loss, dx, de = _run(x, e, y, scale, 'none', grad)
    for out in (loss, surface_cross_entropy(x, e, y, scale, 'none')):
        assert ((out.double() - want).abs() <= 2 * dz + 8 * 2.0 ** -24 * want + rest).all()
    assert ((dx.double() - gx).abs() <= tx).all(), float(((dx.double() - gx).abs() - tx).max())
    assert ((de.double() - ge).abs() <= te).all(), float(((de.double() - ge).abs() - te).max())
    # the sum's gradients, whose kernels differ
    one = torch.tensor(2.0 ** -10, device=DEV)
    want_e = _run(x, e, y, scale, 'none', one.expand(n).contiguous())
    got = _run(x, e, y, scale, 'sum', one)
    terms = 2.0 ** -10 * scale * (hot.abs() * ok[:, None]).t() @ x.double().abs()
    tol = 2 * (up + (n + 32) * 2.0 ** -24) * terms + 2 * u * want_e[2].double().abs() + small \
        + rest * 2.0 ** -10 * n * x.double().abs().max()
    assert ((got[2].double() - want_e[2].double()).abs() <= tol).all()


@pytest.mark.parametrize('reduction', ['none', 'sum'])
@pytest.mark.parametrize('size', [1.0, 6.0, 40.0, 300.0, 3000.0])
@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_probabilities_add_up_to_one(dname, size, reduction):
    """With a feature that is 1 in every pixel the rows' gradients of that channel add up to
    scale sum_i g_i (sum_v p_iv - 1) = 0, whatever the logits' size: both walks have to form the same
    logits.  A probability p is off by its exponent's rounding, p (|log2 p| + 8) 2^-24, which is at
    most 2^-20 for all of a pixel's together (p |log2 p| < 0.54, 200 rows), the sum's by
    (V + 16) 2^-24, an operand's rounding by u_p; a row's sum by (n + 8) 2^-24 and u."""
    dt, scale = TYPES[dname], 1.0
    g = torch.Generator().manual_seed(23)
    n, V, D = 900, 200, 48
    x = (torch.randn(n, D, generator=g) * size).to(DEV, dt)
    e = (torch.randn(V, D, generator=g) * size).to(DEV, dt)
    x[:, 0] = 1
    y = torch.randint(0, V, (n,), generator=g).to(DEV)
    y[:300] = (x[:300].float() @ e.float().t()).argmax(1)
    grad = (torch.rand(n, generator=g) + 0.25).to(DEV) if reduction == 'none' else \
        torch.tensor(0.75, device=DEV)
    _, _, de = _run(x, e, y, scale, reduction, grad)
    gs = float(grad.double().expand(n).sum()) * scale
    u = torch.finfo(dt).eps / 2
    up = u if dname != 'f32' else 2.0 ** -22
    col = de[:, 0].double()
    # 16 bits: the offset of a walk of logits up to 2^10 (fp16) or 2^12 is one number, off by 2^-25 of it
    offset = {'f32': 0.0, 'f16': 2.0 ** -15, 'bf16': 2.0 ** -13}[dname]
    bound = 2 * gs * (2.0 ** -20 + (V + 16 + n + 8) * 2.0 ** -24 + up + offset) + u * float(col.abs().sum())
    if dname == 'f16':
        bound += V * 2.0 ** -25
    assert abs(float(col.sum())) <= bound, (float(col.sum()), bound)
    assert float(col.abs().max()) > 0


@pytest.mark.parametrize('n', [10, 100])
def test_all_logits_below_any_ordinary_number(n):
    """Logits of -1e33 to -1e31: no maximum may begin above them."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    g = torch.Generator().manual_seed(24)
    x = torch.full((n, 16), 1e18, device=DEV)
    e = -torch.rand(20, 16, generator=g).to(DEV) * 1e14
    y = torch.randint(0, 20, (n,), generator=g).to(DEV)
    z = x.double() @ e.double().t()
    want = z.amax(1) - z[torch.arange(n, device=DEV), y]
    dz = (6 * 16 + 8) * 2.0 ** -24 * z.abs().amax(1)
    got = surface_cross_entropy(x, e, y, 1.0, 'none')
    assert ((got.double() - want).abs() <= 2 * dz).all() and (got.double().amax() > 1e31)


@pytest.mark.parametrize('n', [20, 300])
@pytest.mark.parametrize('where', ['row', 'label', 'positive', 'pixel', 'all rows'])
@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_infinite_elements(dname, where, n):
    """An infinite element of the table or of a pixel: losses and gradients are finite, infinite and NaN
    where those of the formulas in 64 bits are (a row whose logits are all minus infinity takes no part),
    and the finite ones are right: probabilities off by 2^-18 (logits below 2^4), rounded to u."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    dt = TYPES[dname]
    g = torch.Generator().manual_seed(25)
    V, D, bad = 40, 24, 17
    x = (torch.rand(n, D, generator=g) * 0.5 + 0.1).to(DEV, dt)
    e = (torch.randn(V, D, generator=g) * 0.5).to(DEV, dt)
    y = torch.randint(0, V - 1, (n,), generator=g).to(DEV)
    y = torch.where(y >= bad, y + 1, y)  # no label is the bad row
    if where in ('row', 'label', 'positive'):
        e[bad, 3] = math.inf if where == 'positive' else -math.inf
        if where == 'label':
            y[5:8] = bad
    else:
        if where == 'all rows':
            e[:, 3] = e[:, 3].abs() + 0.125
        x[7, 3] = -math.inf
    grad = (torch.rand(n, generator=g) + 0.25).to(DEV)
    x64, e64 = x.double().requires_grad_(True), e.double().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(x64 @ e64.t(), y, reduction='none')
    wx, we = torch.autograd.grad(want, [x64, e64], grad.double())
    u = torch.finfo(dt).eps / 2
    cap = lambda t: torch.where(torch.isfinite(t), t, torch.zeros_like(t)).abs().double()  # noqa: E731
    gsum = grad.double().sum()
    sizes = (2.0 ** -18 + 0 * want, (2 * u + 2.0 ** -18) * 2 * grad.double()[:, None] * cap(e).amax(0),
             (2 * u + 2.0 ** -18) * 2 * gsum * cap(x).amax() + 0 * we)
    loss, dx, de = _run(x, e, y, 1.0, 'none', grad)
    if where == 'label':
        # The walk leaves a label's own row out of the weighted sum as 0 times it, and 0 times infinity is
        # NaN: where the label's row is infinite (and the loss too) an infinity of dX is NaN here.
        assert not torch.isfinite(dx[5:8, 3]).any() and not torch.isfinite(wx[5:8, 3]).any()
        dx[5:8, 3], wx[5:8, 3] = 0, 0
    for got, ref, size in zip((loss, dx, de), (want.detach(), wx, we), sizes):
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), where
        assert torch.equal(torch.isinf(got), torch.isinf(ref)), where
        fin = torch.isfinite(ref)
        assert ((got.double() - ref).abs()[fin] <= (size + 2 * u * ref.abs())[fin]).all()
    few = surface_cross_entropy(x, e, y, 1.0, 'none')
    assert torch.equal(torch.isnan(few), torch.isnan(want))
    assert torch.equal(torch.isinf(few), torch.isinf(want))
    fin = torch.isfinite(want)
    assert ((few.double() - want).abs()[fin] <= 2.0 ** -18).all()


@pytest.mark.parametrize('which', ['features', 'embeddings', 'both'])
def test_second_derivatives_raise(which):
    """A gradient that enters a loss again raises, also where that loss has another term with a graph."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    g = torch.Generator().manual_seed(26)
    x, e = torch.randn(20, 8, generator=g).to(DEV), torch.randn(10, 8, generator=g).to(DEV)
    y = torch.randint(0, 10, (20,), generator=g).to(DEV)
    leaves = [t.requires_grad_(True) for t, w in ((x, 'features'), (e, 'embeddings'))
              if which in (w, 'both')]
    for weight in (1.0, torch.tensor(2.0, device=DEV, requires_grad=True)):
        loss = surface_cross_entropy(x, e, y) * weight
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        plain = torch.autograd.grad(surface_cross_entropy(x, e, y) * weight, leaves)
        assert all(torch.equal(a, b) for a, b in zip(grads, plain))
        for a in grads:
            with pytest.raises(RuntimeError, match='second derivatives'):
                (loss + a.pow(2).sum()).backward(retain_graph=True)
    # a recorded backward by itself is no error
    x.grad = e.grad = None
    surface_cross_entropy(x, e, y).backward(create_graph=True)
    assert all(t.grad is not None for t in leaves)
    x.grad = e.grad = None


@pytest.mark.parametrize('grad_mode', [True, False])
def test_tangents_raise(grad_mode):
    """Forward mode is refused, not dropped: dual features, tables and incoming gradients."""
    import torch.autograd.forward_ad as fw
    from kaolin_amd.metrics.render import surface_cross_entropy
    from kaolin_amd.render.mesh import surface_embedding
    g = torch.Generator().manual_seed(27)
    x, e = torch.randn(20, 8, generator=g).to(DEV), torch.randn(10, 8, generator=g).to(DEV)
    y = torch.randint(0, 10, (20,), generator=g).to(DEV)
    with fw.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = fw.make_dual
        for call in (lambda: surface_cross_entropy(dual(x, x), e, y),
                     lambda: surface_cross_entropy(x, dual(e, e), y),
                     lambda: surface_embedding(y, dual(e, e))):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(surface_embedding(y, e), e[y])
        if not grad_mode:
            return
        table = e.clone().requires_grad_(True)
        weight = dual(torch.ones(20, 8, device=DEV), torch.ones(20, 8, device=DEV))
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(surface_embedding(y, table), table, weight)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(surface_cross_entropy(x, table, y, 1.0, 'none'), table, weight[:, 0])


@pytest.mark.parametrize('D', [20, 64, 100, 256])
@pytest.mark.parametrize('V', [8, 300])
@pytest.mark.parametrize('size', [0.3, 300.0])
@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_rows_that_are_alike(dname, size, V, D):
    """Rows with a common part of 30 times their differences (a smooth table: neighbouring faces): dX is
    made of the differences, so the weights of the rows have to add up to 1.  With probabilities off by
    rho = 2 du + u_p, the weighted mean of e_v - e_y is off by 2 rho times that of |e_v - e_y|, and the
    sums of whole rows in 32 bits by (V / 8 + 32) 2^-24 of the largest element."""
    dt = TYPES[dname]
    g = torch.Generator().manual_seed(28)
    n = 500
    x = (torch.randn(n, D, generator=g) * size / 3 / D ** 0.5).to(DEV, dt)
    e = ((torch.randn(V, D, generator=g) * 0.1 + 3 * torch.randn(1, D, generator=g))).to(DEV, dt)
    y = torch.randint(0, V, (n,), generator=g).to(DEV)
    grad = (torch.rand(n, generator=g) + 0.25).to(DEV)
    x64, e64 = x.double().requires_grad_(True), e.double()
    want = torch.nn.functional.cross_entropy(x64 @ e64.t(), y, reduction='none')
    gx, = torch.autograd.grad(want, x64, grad.double())
    p = torch.softmax(x64.detach() @ e64.t(), 1)
    apart = torch.stack([(p[i, :, None] * (e64 - e64[y[i]]).abs()).sum(0) for i in range(n)])
    dz = ((6 if dname == 'f32' else 1) * D + 8) * 2.0 ** -24 * (
        x.double().abs() @ e64.abs().t()).amax(1)
    u = torch.finfo(dt).eps / 2
    rho = 2 * (3 * dz + (V + 16) * 2.0 ** -24) + (u if dname != 'f32' else 2.0 ** -23)
    if dname != 'f32':
        rho = rho + 2.0 ** -35 * V  # (fp16: terms below its normal range; small beside u in bf16)
    tol = grad.double()[:, None] * (2 * rho[:, None] * apart
                                    + (V / 8 + 32) * 2.0 ** -24 * e64.abs().max()) + u * gx.abs() * 1.01
    if dname == 'f16':
        tol = tol + 2.0 ** -25
    got = _run(x, e, y, 1.0, 'none', grad)[1]
    assert ((got.double() - gx).abs() <= tol).all(), float(((got.double() - gx).abs() / tol).max())


@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_a_captured_step_follows_its_inputs(dname):
    """The walk is chosen on the device: a captured step replayed on bounded, unbounded, large and
    infinite logits in turn, with eager work between, gives what an eager call gives."""
    dt = TYPES[dname]
    g = torch.Generator().manual_seed(29)
    n, V, D = 700, 90, 40
    base_x, base_e = torch.randn(n, D, generator=g).to(DEV), torch.randn(V, D, generator=g).to(DEV)
    y = torch.randint(-1, V, (n,), generator=g).to(DEV)
    grad = (torch.rand(n, generator=g) + 0.25).to(DEV)
    x, e = base_x.to(dt), base_e.to(dt)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(x, e, y, 0.5, 'none', grad)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _run(x, e, y, 0.5, 'none', grad)
    for size in (1.0, 200.0, 0.1, 20.0, math.inf, 1.0, 200.0):
        x.copy_(base_x * (size if math.isfinite(size) else 1.0))
        e.copy_(base_e * (size if math.isfinite(size) else 1.0))
        if not math.isfinite(size):
            e[V - 1, 0] = -math.inf
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        eager = _run(x, e, y, 0.5, 'none', grad)
        for a, b in zip(outs, eager):
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(
                torch.nan_to_num(a), torch.nan_to_num(b)), size
        torch.cuda.synchronize()


@pytest.mark.parametrize('size', [1.0, 1e3])
@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_a_table_of_one_row(dname, size):
    """Nothing to choose: no loss and no gradient, whatever the logit."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    g = torch.Generator().manual_seed(30)
    x = (torch.randn(90, 33, generator=g) * size).to(DEV, TYPES[dname])
    e = (torch.randn(1, 33, generator=g) * size).to(DEV, TYPES[dname])
    y = torch.randint(-1, 2, (90,), generator=g).to(DEV)
    for out in (*_run(x, e, y, 2.0, 'none', torch.ones(90, device=DEV)),
                surface_cross_entropy(x[:50], e, y[:50], 2.0, 'none')):
        assert (out == 0).all()


@pytest.mark.parametrize('V', [8, 200])
@pytest.mark.parametrize('D', [40, 128, 200])
@pytest.mark.parametrize('reduction', ['none', 'sum'])
@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_pixels_that_are_alike(dname, reduction, D, V):
    """An untrained table of few rows and features with a common part c of 10 times their spread: every
    pixel has next to the same probabilities, and labels as often as those say, so dE is what is left of
    large sums.  A row's sum over the pixels of (p - p^) x_i is off by the probabilities' error in two
    parts, u^2 at most and for the label's term too (32 bits: 2^-23), du of a probability relative, the
    same for all pixels, and the sum's own roundings, (n / 16 + 32) 2^-24 of its terms and their number's
    parts; rounded to u."""
    dt = TYPES[dname]
    g = torch.Generator().manual_seed(31)
    n = 40000
    x = (torch.randn(n, D, generator=g) + 10 * torch.randn(1, D, generator=g)).to(DEV, dt)
    e = (torch.randn(V, D, generator=g) * 1e-4).to(DEV, dt)
    y = (torch.arange(n) % V).to(DEV)
    grad = torch.ones(n, device=DEV) if reduction == 'none' else torch.tensor(1.0, device=DEV)
    x64, e64 = x.double(), e.double().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(x64 @ e64.t(), y, reduction='sum')
    ge, = torch.autograd.grad(want, e64)
    z = x64 @ e64.detach().t()
    p = torch.softmax(z, 1)
    p[torch.arange(n, device=DEV), y] = 1 - p[torch.arange(n, device=DEV), y]
    terms = p.t() @ x64.abs()
    u = torch.finfo(dt).eps / 2
    two = u * u if dname != 'f32' else 2.0 ** -23
    dz = ((6 if dname == 'f32' else 1) * D + 8) * 2.0 ** -24 * float(
        (x64.abs() @ e64.detach().abs().t()).max())
    # a probability's own error: its logit's, the log sum's (V terms) and an exponential's, in 32 bits
    du = 2 * (3 * dz + (V + 16) * 2.0 ** -24)
    tol = (2 * two + du + (n / 16 + 32) * 2.0 ** -24) * terms + u * ge.abs() * 1.01 + (
        2.0 ** -25 if dname == 'f16' else 0.0)
    got = _run(x, e, y, 1.0, reduction, grad)[2]
    assert ((got.double() - ge).abs() <= tol).all(), float(((got.double() - ge).abs() / tol).max())
