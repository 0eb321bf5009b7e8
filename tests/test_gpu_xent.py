"""GPU: surface_cross_entropy (kd_xent.hpp) against the formulas in 64 bits.

Tolerances, with u the type's half step (eps / 2) and A_i = |scale| max_v sum_d |x_id e_vd|, which
bounds every logit of pixel i and the rounding of its sum:
- 16-bit products are exact and added in 32 bits, 32-bit ones are six bf16 products each: a logit is
  off by at most dz = (k D + 8) 2^-24 A_i with k = 1 or 6 (the 8: the factor's rounding, the
  exponent's multiply-add and, for 32 bits, the three products below 2^-24 that are left out);
- a sum of N positive terms in 32 bits is off by N 2^-24 relative, an exponential by 2^-22;
so the log odds U = L' - z_y are off by du = 3 dz + (V + 16) 2^-24, the loss softplus(U) by
w du (1 + du) plus its own rounding, and each probability by rho = 2 du relative.  The gradients are
sums of p e (of p x): off by (rho + u_p + N 2^-24) times the sum of the terms' sizes, u_p the
rounding of a probability to the operands' type (u, for 32 bits 2^-23), and rounded once to u.
float16: probabilities below 2^-28 of the largest gradient are subnormal operands, off by 2^-38 of
it a term, and results below its normal range are off by 2^-25.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


def _inputs(n, V, D, dt, seed=0, spread=1.0, background=0.3):
    g = torch.Generator().manual_seed(seed)
    e = torch.randn(V, D, generator=g)
    e = e / e.norm(dim=1, keepdim=True).clamp(min=1e-3)
    y = torch.randint(0, V, (n,), generator=g)
    x = e[y] + spread * torch.randn(n, D, generator=g) / math.sqrt(D)
    y[torch.rand(n, generator=g) < background] = -1
    return x.to(DEV, dt), e.to(DEV, dt), y.to(DEV)


def _reference(x, e, y, scale, reduction, grad):
    """Loss, gradients and their tolerances, in 64 bits."""
    dt = x.dtype
    V, D = e.shape
    x, e = x.detach().double(), e.detach().double()
    n = y.numel()
    ok = (y >= 0) & (y < V)
    rows = ok.nonzero().reshape(-1)
    ys, xs = y[rows], x[rows]
    r = torch.arange(rows.numel(), device=DEV)
    count = max(1, rows.numel())
    z = scale * (xs @ e.t())
    zy = z[r, ys]
    zo = z.clone()
    zo[r, ys] = -math.inf
    U = torch.logsumexp(zo, 1) - zy if V > 1 else torch.full_like(zy, -math.inf)
    loss = torch.logaddexp(U, torch.zeros_like(U))
    w = torch.sigmoid(U)
    p = torch.exp(z - (zy + loss)[:, None])
    p[r, ys] = w
    k = 1 if dt != torch.float32 else 6
    A = abs(scale) * (xs.abs() @ e.abs().t()).amax(1) if rows.numel() else zy
    dz = (k * D + 8) * 2.0 ** -24 * A
    du = 3 * dz + (V + 16) * 2.0 ** -24
    tl = w * du * (1 + du) * 1.01 + 4 * 2.0 ** -24 * loss + 1e-30
    g = grad.double().reshape(-1)
    g = g[rows] if reduction == 'none' else g.expand(rows.numel()) / (
        count if reduction == 'mean' else 1)
    u = torch.finfo(dt).eps / 2
    up = u if dt != torch.float32 else 2.0 ** -23
    sign = torch.ones_like(p)
    sign[r, ys] = -1
    gs = g * scale
    gx = (p * sign * gs[:, None]) @ e
    size_x = (p * gs.abs()[:, None]) @ e.abs()
    ge = (p * sign).t() @ (gs[:, None] * xs)
    rel = (2 * du + up)[:, None] * p * gs.abs()[:, None]
    size_e = rel.t() @ xs.abs() + (rows.numel() + 8) * 2.0 ** -24 * (
        (p * gs.abs()[:, None]).t() @ xs.abs())
    tx = (2 * du + up + (V + 8) * 2.0 ** -24)[:, None] * size_x + u * gx.abs() * 1.01 + 1e-37
    te = size_e + u * ge.abs() * 1.01 + 1e-37
    if dt == torch.float16:
        top = gs.abs().max() if rows.numel() else 0.0
        # a pixel's probabilities are scaled by its largest (but the label's): 2^-35 of w
        tx = tx + 2.0 ** -25 + 2.0 ** -30 * (w * gs.abs())[:, None] * e.abs().sum(0)
        te = te + 2.0 ** -25 + 2.0 ** -38 * top * xs.abs().sum(0)
    fx, ftx = torch.zeros(n, D, dtype=torch.float64, device=DEV), \
        torch.zeros(n, D, dtype=torch.float64, device=DEV)
    fx[rows], ftx[rows] = gx, tx
    if reduction == 'none':
        fl, ftl = torch.zeros(n, dtype=torch.float64, device=DEV), \
            torch.zeros(n, dtype=torch.float64, device=DEV)
        fl[rows], ftl[rows] = loss, tl
    else:
        div = count if reduction == 'mean' else 1
        fl, ftl = loss.sum() / div, tl.sum() / div + 2.0 ** -23 * loss.sum() / div + 1e-30
    return fl, ftl, fx, ftx, ge, te


def _run(x, e, y, scale, reduction, grad):
    from kaolin_amd.metrics.render import surface_cross_entropy
    x, e = x.detach().requires_grad_(True), e.detach().requires_grad_(True)
    loss = surface_cross_entropy(x, e, y, scale, reduction)
    return (loss, *torch.autograd.grad(loss, [x, e], grad))


def _grad(reduction, shape, seed=1):
    g = torch.Generator().manual_seed(seed)
    if reduction == 'none':
        return (torch.rand(shape, generator=g) + 0.25).to(DEV)
    return torch.tensor(0.75, device=DEV)


def _check(got, want):
    loss, gx, ge = got
    fl, tl, fx, tx, re, te = want
    assert loss.dtype == torch.float32
    assert ((loss.detach().double().reshape(fl.shape) - fl).abs() <= tl).all()
    assert ((gx.double().reshape(fx.shape) - fx).abs() <= tx).all(), \
        float(((gx.double().reshape(fx.shape) - fx).abs() - tx).max())
    assert ((ge.double() - re).abs() <= te).all(), float(((ge.double() - re).abs() - te).max())


CASES = [
    # dtype, pixels, rows, channels, scale, reduction
    ('f32', 1, 1, 1, 1.0, 'mean'), ('f32', 1, 2, 3, 2.0, 'none'), ('f32', 7, 33, 16, 5.0, 'sum'),
    ('f32', 300, 1000, 37, 10.0, 'mean'), ('f32', 130, 31, 64, 8.0, 'none'),
    ('f32', 2000, 97, 65, 12.0, 'none'), ('f32', 257, 700, 130, 9.0, 'mean'),
    ('f32', 100, 300, 256, 16.0, 'sum'), ('f32', 33, 5000, 32, -6.0, 'mean'),
    ('f16', 1, 64, 8, 4.0, 'none'), ('f16', 513, 997, 37, 8.0, 'none'),
    ('f16', 100, 2049, 64, 14.0, 'sum'), ('f16', 1000, 40, 128, 10.0, 'sum'),
    ('f16', 65, 500, 200, 16.0, 'none'), ('f16', 3000, 129, 20, 6.0, 'sum'),
    ('bf16', 1, 20000, 256, 14.0, 'none'), ('bf16', 1, 1, 64, 14.0, 'mean'),
    ('bf16', 5000, 1500, 64, 14.0, 'mean'), ('bf16', 400, 10000, 16, 20.0, 'none'),
    ('bf16', 31, 77, 100, 10.0, 'sum'), ('bf16', 900, 800, 255, 18.0, 'mean'),
    ('bf16', 20000, 3, 5, 3.0, 'none'), ('bf16', 640, 256, 32, 0.0, 'mean'),
    ('bf16', 129, 4097, 1, 30.0, 'none'),
]


@pytest.mark.parametrize('dname,n,V,D,scale,reduction', CASES, ids=str)
def test_loss_and_gradients(dname, n, V, D, scale, reduction):
    x, e, y = _inputs(n, V, D, TYPES[dname], seed=n + V + D, background=0.3 if n > 1 else 0.0)
    grad = _grad(reduction, (n,))
    got = _run(x, e, y, scale, reduction, grad)
    _check(got, _reference(x, e, y, scale, reduction, grad))
    assert (got[1][y < 0] == 0).all()
    again = _run(x, e, y, scale, reduction, grad)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # a fixed order of the sums
    # without gradients the parts of a sum can be cut elsewhere: the same bounds, not the same bits
    from kaolin_amd.metrics.render import surface_cross_entropy
    _check((surface_cross_entropy(x, e, y, scale, reduction), *got[1:]),
           _reference(x, e, y, scale, reduction, grad))


@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('n,V,D', [(1, 1, 1), (2, 33, 7), (31, 5000, 33), (32, 127, 64), (33, 129, 128),
                                   (63, 70000, 20), (64, 2000, 250), (65, 2000, 40)])
def test_losses_of_a_few_pixels(dname, reduction, n, V, D):
    """Without gradients the table is read as it stands, up to 64 pixels; a table one element off any
    alignment, a label of no row, NaN in its features."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    x, e, y = _inputs(n, V, D, TYPES[dname], seed=n + D, background=0.0)
    flat = torch.zeros(V * D + 1, device=DEV, dtype=e.dtype)
    off = flat[1:].view(V, D)
    off.copy_(e)
    if n > 1:
        y[n // 2] = V
        x[n // 2] = math.nan
    want = _reference(x, e, y, 9.0, reduction, _grad(reduction, (n,)))
    for table in (e, off):
        loss = surface_cross_entropy(x, table, y, 9.0, reduction)
        assert ((loss.double() - want[0]).abs() <= want[1]).all()
        assert torch.equal(loss, surface_cross_entropy(x, table, y, 9.0, reduction))


@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('spread,scale', [(0.02, 200.0), (0.0, 60.0), (8.0, 40.0)])
def test_far_from_even(dname, spread, scale):
    """Trained (the label's probability next to 1: its complement must keep its digits) and far
    from trained (the label's probability next to 0)."""
    x, e, y = _inputs(500, 400, 64, TYPES[dname], seed=3, spread=spread)
    grad = _grad('none', (500,))
    got = _run(x, e, y, scale, 'none', grad)
    _check(got, _reference(x, e, y, scale, 'none', grad))


@pytest.mark.parametrize('dname,size', [('f32', 1e-18), ('f32', 1e18), ('bf16', 1e-18),
                                        ('bf16', 1e18), ('f32', 1e-8), ('bf16', 1e8)])
def test_tables_of_any_size(dname, size):
    """Ordinary logits of very small and very large rows: no part of a sum may leave the range."""
    x, e, y = _inputs(300, 200, 40, TYPES[dname], seed=15)
    x, e = (x.float() / size).to(x.dtype), (e.float() * size).to(e.dtype)
    grad = _grad('none', (300,))
    got = _run(x, e, y, 6.0, 'none', grad)
    _check(got, _reference(x, e, y, 6.0, 'none', grad))
    assert (got[1][y >= 0] != 0).any() and (got[2] != 0).any()


@pytest.mark.parametrize('dname,n,V,D', [('bf16', 290000, 70, 16), ('bf16', 140000, 33, 100),
                                         ('f32', 150000, 40, 8), ('f32', 70000, 20, 129),
                                         ('f16', 70000, 50, 250), ('f16', 300, 140000, 8),
                                         ('f32', 260, 70000, 33), ('bf16', 100, 70000, 200)])
def test_more_blocks_than_workgroups(dname, n, V, D):
    """Whole blocks of held rows in turn and the rest cut across their borders, on both sides."""
    x, e, y = _inputs(n, V, D, TYPES[dname], seed=16, background=0.05)
    grad = _grad('none', (n,))
    _check(_run(x, e, y, 8.0, 'none', grad), _reference(x, e, y, 8.0, 'none', grad))


@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('train', [False, True])
def test_long_sums(dname, train):
    """A table of like rows, more pixels than workgroups hold: the loss is log V, and adding up like
    terms one by one rounds every time the same way.  In steps of 2^-24: 16 + 3 for the terms of one or
    two tiles, V / 64 for the tiles (16-bit data; 32-bit data carry what is lost: 3), 256 for the parts
    of a walk, 4 for the exponential, 16 for a logit's product with its factor (below 8 in log2, twice),
    and the loss's own 4 roundings."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    V, n = 100001, 140000
    dt = TYPES[dname]
    e = torch.tensor([0.75, -0.5, 0.375], device=DEV, dtype=dt).repeat(V, 1)
    x = torch.tensor([0.875, -0.625, 0.3125], device=DEV, dtype=dt).repeat(n, 1)
    y = torch.arange(n, device=DEV) % V
    x.requires_grad_(train)
    loss = surface_cross_entropy(x, e, y, 3.7, 'none').detach().double()
    want = math.log(V)
    steps = 19 + (3 if dname == 'f32' else V / 64) + 256 + 4 + 16 + 4 * want
    assert (loss - want).abs().max() <= steps * 2.0 ** -24


def test_backward_twice():
    """The forward's state is only read: a second backward gives the same."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    x, e, y = _inputs(700, 300, 48, torch.bfloat16, seed=17)
    x, e = x.requires_grad_(True), e.requires_grad_(True)
    grad = _grad('none', (700,))
    loss = surface_cross_entropy(x, e, y, 5.0, 'none')
    a = torch.autograd.grad(loss, [x, e], grad, retain_graph=True)
    torch.autograd.grad(loss, [x, e], grad * 1e-3, retain_graph=True)
    b = torch.autograd.grad(loss, [x, e], grad)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing."""
    sets = [(_inputs(6000, 3000, 64, torch.bfloat16, seed=18), 9.0),
            (_inputs(5000, 4000, 32, torch.float32, seed=19), 7.0)]
    one = torch.tensor(1.0, device=DEV)
    want = [_run(*a, s, 'mean', one) for a, s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for rep in range(3):
        for st, (a, s) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(_run(*a, s, 'mean', one))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, want[i % 2]))


def test_large_logits_move_the_maximum():
    """Rows of rising size: the running maximum moves in almost every block of the table."""
    x, e, y = _inputs(200, 3001, 48, torch.bfloat16, seed=4)
    e = (e.float() * torch.linspace(0.01, 30, 3001, device=DEV)[:, None]).bfloat16()
    grad = _grad('none', (200,))
    for table in (e, e.flip(0).contiguous()):
        _check(_run(x, table, y, 3.0, 'none', grad), _reference(x, table, y, 3.0, 'none', grad))


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('dname', ['f32', 'bf16'])
def test_no_pixel_takes_part(dname, reduction):
    x, e, y = _inputs(300, 50, 16, TYPES[dname])
    y = torch.where(torch.arange(300, device=DEV) % 2 == 0, -1, 50)
    loss, gx, ge = _run(x, e, y, 4.0, reduction, _grad(reduction, (300,)))
    assert (loss == 0).all() and (gx == 0).all() and (ge == 0).all()
    x, y = x[:0], y[:0]
    loss, gx, ge = _run(x, e, y, 4.0, reduction, _grad(reduction, (0,)))
    assert (loss == 0).all() and gx.shape == (0, 16) and (ge == 0).all()


def test_values_in_the_background():
    """NaN, infinities and the lowest value where the label names no row leave no trace."""
    x, e, y = _inputs(400, 90, 24, torch.float32, seed=5)
    dirty = x.clone()
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min], device=DEV)
    rows = (y < 0).nonzero().reshape(-1)
    dirty[rows] = bad[torch.arange(rows.numel(), device=DEV) % 4][:, None]
    far = torch.where(y < 0, torch.full_like(y, 2 ** 40), y)
    grad = _grad('none', (400,))
    gdirty = torch.where(y < 0, torch.full_like(grad, math.nan), grad)
    want = _run(x, e, y, 6.0, 'none', grad)
    for got in (_run(dirty, e, y, 6.0, 'none', grad), _run(x, e, far, 6.0, 'none', grad),
                _run(dirty, e, far, 6.0, 'none', gdirty)):
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_bad_values_are_not_hidden():
    x, e, y = _inputs(64, 40, 16, torch.float32, seed=6, background=0.0)
    x[5, 3] = math.nan
    loss, gx, ge = _run(x, e, y, 2.0, 'none', _grad('none', (64,)))
    assert torch.isnan(loss[5]) and torch.isnan(gx[5]).all()
    assert torch.isfinite(loss[:5]).all() and torch.isfinite(gx[6:]).all()
    assert torch.isnan(ge).all()


@pytest.mark.parametrize('which', ['features', 'embeddings'])
def test_one_gradient_only(which):
    from kaolin_amd.metrics.render import surface_cross_entropy
    x, e, y = _inputs(500, 300, 40, torch.bfloat16, seed=7)
    _, gx, ge = _run(x, e, y, 9.0, 'mean', torch.tensor(1.0, device=DEV))
    leaf = (x if which == 'features' else e).detach().requires_grad_(True)
    loss = surface_cross_entropy(leaf if which == 'features' else x,
                                 leaf if which == 'embeddings' else e, y, 9.0)
    loss.backward()
    assert torch.equal(leaf.grad, gx if which == 'features' else ge)


def test_shapes_and_strides():
    """An image of channels-first features, transposed labels, a stepped table, an expanded
    gradient."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    g = torch.Generator().manual_seed(8)
    B, H, W, D, V = 2, 19, 23, 21, 130
    x = torch.randn(B, D, H, W, generator=g).to(DEV).permute(0, 2, 3, 1)
    y = torch.randint(-1, V, (B, W, H), generator=g).to(DEV).transpose(1, 2)
    e = torch.randn(V, 2 * D, generator=g).to(DEV)[:, ::2]
    xl, el = x.detach().requires_grad_(True), e.detach().requires_grad_(True)
    loss = surface_cross_entropy(xl, el, y, 1.5, 'none')
    assert loss.shape == y.shape
    loss.sum().backward()
    one = torch.ones(B * H * W, device=DEV)
    want = _reference(x.reshape(-1, D), e, y.reshape(-1), 1.5, 'none', one)
    _check((loss.reshape(-1), xl.grad.reshape(-1, D), el.grad), want)
    # a pixel without any other dimension
    got = _run(x[0, 0, 0], e, torch.tensor(3, device=DEV), 1.5, 'none',
               torch.tensor(1.0, device=DEV))
    assert got[0].shape == () and got[1].shape == (D,)


def test_incoming_gradients_of_any_size():
    """float16 operands of the table's gradient are scaled by the largest incoming gradient."""
    x, e, y = _inputs(600, 200, 32, torch.float16, seed=9)
    base = _grad('none', (600,))
    base[::5] = 0
    _, _, ge = _run(x, e, y, 8.0, 'none', base)
    for f in (2.0 ** -12, 2.0 ** 6):
        _, gx, gf = _run(x, e, y, 8.0, 'none', base * f)
        want = _reference(x, e, y, 8.0, 'none', base * f)
        assert ((gf.double() - want[4]).abs() <= want[5]).all()
        assert ((gx.double() - want[2]).abs() <= want[3]).all()


def test_gradients_by_differences():
    """Directional differences of the 32-bit loss.  Along a unit step the third derivative of a
    pixel's loss is the third cumulant of scale e.d over the softmax, at most R^3 / (6 sqrt 3) with
    R the range, so a central difference is off by h^2 / 6 of that and by the loss's error / h."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    x, e, y = _inputs(200, 150, 24, torch.float32, seed=10)
    scale, h = 3.0, 2.0 ** -6
    one = torch.tensor(1.0, device=DEV)
    _, gx, ge = _run(x, e, y, scale, 'sum', one)
    g = torch.Generator().manual_seed(11)
    ok = (y >= 0).double()
    for which in ('x', 'e'):
        base = x if which == 'x' else e
        d = torch.randn(base.shape, generator=g).to(DEV)
        d = d / d.norm(dim=1, keepdim=True)
        if which == 'x':
            lo, hi = (surface_cross_entropy(x + s * h * d, e, y, scale, 'none').double()
                      for s in (-1, 1))
            slope = scale * (d.double() @ e.double().t())
            got = (gx.double() * d.double()).sum()
        else:
            lo, hi = (surface_cross_entropy(x, e + s * h * d, y, scale, 'none').double()
                      for s in (-1, 1))
            slope = scale * (x.double() @ d.double().t())
            got = (ge.double() * d.double()).sum()
        R = slope.amax(1) - slope.amin(1)
        trunc = (ok * R ** 3).sum() / (6 * math.sqrt(3)) * h * h / 6
        tl = _reference(x, e, y, scale, 'none', torch.ones(200, device=DEV))
        # the stepped inputs are rounded too: half a step of their size, times the slope
        step = 2.0 ** -24 * scale * ok.sum() * 4
        noise = (tl[1].sum() * 2 + step) / (2 * h) + (tl[3] if which == 'x' else tl[5]).sum()
        diff = ((hi - lo) / (2 * h)).sum()
        assert abs(diff - got) <= trunc + noise, (which, float(diff), float(got))


def test_no_second_derivative():
    from kaolin_amd.metrics.render import surface_cross_entropy
    x, e, y = _inputs(20, 10, 8, torch.float32)
    x.requires_grad_(True)
    g, = torch.autograd.grad(surface_cross_entropy(x, e, y), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals_on_the_gpu():
    from kaolin_amd.metrics.render import surface_cross_entropy as f
    from kaolin_amd.render.mesh import surface_embedding
    x, e, y = _inputs(20, 10, 8, torch.float32)
    for args, what in (((x.double(), e.double(), y), 'not implemented'),
                       ((x, e.half(), y), 'dtype'), ((x, e, y.int()), 'torch.int64'),
                       ((x[:19], e, y), 'size'), ((x, e[:, :7], y), 'size'),
                       ((x, e[None], y), 'embeddings must be'), ((x, e[:0], y), 'at least one'),
                       ((x, e, y, 1.0, 'max'), 'reduction'), ((x, e, y, math.inf), 'finite'),
                       ((x.new_zeros(4, 257), e.new_zeros(3, 257), y[:4]), '256 channels'),
                       ((x.cpu(), e, y), 'on a GPU')):
        with pytest.raises(RuntimeError, match=what):
            f(*args)
    with pytest.raises(RuntimeError, match='torch.int64'):
        surface_embedding(y.int(), e)
    with pytest.raises(RuntimeError, match='not implemented'):
        surface_embedding(y, e.long())
    with pytest.raises(RuntimeError, match='on a GPU'):
        surface_embedding(y.cpu(), e)


def test_past_32_bit_offsets():
    """More than 2^31 features: the last pixels' losses and gradients, and the table's gradient."""
    n, V, D = 8400001, 40, 256
    g = torch.Generator(device=DEV).manual_seed(12)
    e = torch.randn(V, D, generator=g, device=DEV).bfloat16() / 16
    y = torch.arange(n, device=DEV) % (V + 1) - 1
    x = torch.randn(1024, D, generator=g, device=DEV).bfloat16().repeat(n // 1024 + 1, 1)[:n]
    grad = torch.rand(n, generator=g, device=DEV)
    grad[1 << 20:-(1 << 20)] = 0  # the table's gradient: the first and the last pixels
    loss, gx, ge = _run(x, e, y, 5.0, 'none', grad)
    keep = torch.cat([torch.arange(1 << 20, device=DEV), torch.arange(n - (1 << 20), n, device=DEV)])
    want = _reference(x[keep], e, y[keep], 5.0, 'none', grad[keep])
    _check((loss[keep], gx[keep], ge), want)
    assert (gx[1 << 20:-(1 << 20)] == 0).all()


def test_other_stream():
    x, e, y = _inputs(3000, 700, 64, torch.bfloat16, seed=13)
    one = torch.tensor(1.0, device=DEV)
    want = _run(x, e, y, 10.0, 'mean', one)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _run(x, e, y, 10.0, 'mean', one)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_captured_steps_replay():
    """Two captured training steps replayed in turn, with eager work between, on changing inputs
    (the number of pixels that take part changes inside the graph)."""
    from kaolin_amd.metrics.render import surface_cross_entropy
    setups = []
    for n, V, D, dt, red in ((900, 500, 32, torch.float32, 'mean'),
                             (4000, 80, 64, torch.bfloat16, 'none')):
        x, e, y = _inputs(n, V, D, dt, seed=n)
        grad = _grad(red, (n,))
        xl, el = x.clone().requires_grad_(True), e.clone().requires_grad_(True)

        def step(xl=xl, el=el, y=y, red=red, grad=grad):
            loss = surface_cross_entropy(xl, el, y, 7.0, red)
            return (loss, *torch.autograd.grad(loss, [xl, el], grad))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        setups.append((graph, xl, el, y, red, grad, outs))
    for rep in range(3):
        for graph, xl, el, y, red, grad, outs in setups:
            with torch.no_grad():
                xl.copy_(xl.roll(5, 0))
                y[rep::3 + rep] = -1
                for o in outs:
                    o.fill_(float('nan'))
        for graph, *_ in setups:
            graph.replay()
        for graph, xl, el, y, red, grad, outs in setups:
            eager = _run(xl, el, y, 7.0, red, grad)
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), rep
        torch.cuda.synchronize()


@pytest.mark.parametrize('dname', ['f32', 'bf16'])
def test_correspondence_step(dname):
    """The operators as they are used together: per-vertex features gathered to the faces' corners
    and rendered, per-face embeddings looked up at the rendered face_idx, and the cross entropy of
    the pixels' features against every face, back to both tables and to the vertices."""
    from kaolin_amd import workloads
    from kaolin_amd.metrics.render import surface_cross_entropy
    from kaolin_amd.render.mesh import dibr_rasterization, prepare_vertices, surface_embedding
    dt = TYPES[dname]
    s = workloads.sphere_views(20, 26, 64, 64, 2, DEV)
    g = torch.Generator().manual_seed(14)
    faces, F = s['faces'], s['faces'].shape[0]
    D = 12
    vert = s['vertices'].clone().requires_grad_(True)
    vfeat = torch.randn(vert.shape[0], D, generator=g).to(DEV).requires_grad_(True)
    table = torch.randn(F, D, generator=g).to(DEV, dt).requires_grad_(True)
    fvc, fvi, nrm = prepare_vertices(vert.unsqueeze(0), faces, s['proj'],
                                     camera_transform=s['cam'])
    corners = surface_embedding(faces, vfeat, 0.5)
    assert torch.equal(corners, vfeat.detach()[faces] * 0.5)
    feats = corners.unsqueeze(0).expand(2, -1, -1, -1)
    image, soft, face_idx = dibr_rasterization(64, 64, fvc[..., 2], fvi, feats, nrm[..., 2])
    assert (face_idx >= 0).any() and (face_idx < 0).any()
    rendered = surface_embedding(face_idx, table)
    pixels = (image.to(dt) + rendered)
    loss = surface_cross_entropy(pixels, table, face_idx, 2.0)
    loss.backward()
    # the same from the definition, down to the rendered image (whose backward is tested elsewhere)
    im = image.detach().to(dt).double().requires_grad_(True)
    t64 = table.detach().double().requires_grad_(True)
    hit = face_idx >= 0
    px = im + torch.where(hit[..., None], t64[face_idx.clamp(min=0)], t64.new_zeros(()))
    ref = torch.nn.functional.cross_entropy(2.0 * px[hit] @ t64.t(), face_idx[hit])
    ref.backward()
    # bf16 pixels are rounded (2^-8), which moves logits of size |2 x.e| and what follows from them
    u = torch.finfo(dt).eps
    bound = u * 2.0 * float((px[hit].detach().abs() @ t64.detach().abs().t()).max()) * 4 + 1e-4
    assert abs(float(loss.detach()) - float(ref.detach())) <= bound
    scale = float(t64.grad.abs().max())
    assert float((table.grad.double() - t64.grad).abs().max()) <= bound * scale
    for p in (vert, vfeat, table):
        assert p.grad is not None and torch.isfinite(p.grad).all() and (p.grad != 0).any()
    # the vertex features' gradient is the corners' gradient added per vertex
    gc, = torch.autograd.grad(
        dibr_rasterization(64, 64, fvc[..., 2].detach(), fvi.detach(),
                           (c := corners.detach().requires_grad_(True)).unsqueeze(0).expand(
                               2, -1, -1, -1), nrm[..., 2].detach())[0], c,
        torch.ones_like(image))
    v = vfeat.detach().requires_grad_(True)
    gv, = torch.autograd.grad(surface_embedding(faces, v, 0.5), v, gc)
    want = torch.zeros(vfeat.shape, dtype=torch.float64, device=DEV).index_add_(
        0, faces.reshape(-1), gc.double().reshape(-1, D)) * 0.5
    size = torch.zeros_like(want).index_add_(0, faces.reshape(-1),
                                             gc.double().abs().reshape(-1, D)) * 0.5
    assert ((gv.double() - want).abs() <= 64 * 2.0 ** -24 * size).all()
