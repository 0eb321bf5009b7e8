"""GPU: surface_embedding (kd_embedding.hip) against the plain lookup in 64 bits.

Tolerances.  With u the type's half step (eps / 2): the product is exact to 2^-24 (2^-53 for
float64) and rounded once, so |out - ref| <= (u + 2^-24) |ref|.  A gradient row of m terms is added
in 32 bits: |sum - ref| <= (m + 2) 2^-24 sum |g| |scale|, and rounded once.  float16 results below
its normal range are off by up to half a subnormal step, 2^-25.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'f64': torch.float64, 'f16': torch.float16, 'bf16': torch.bfloat16}


def _half_step(dt):
    return torch.finfo(dt).eps / 2


def _wide_step(dt):
    return 2.0 ** -53 if dt == torch.float64 else 2.0 ** -24


def _reference(index, table, scale, grad=None):
    """out and, with grad, (dE, sum |g| |scale| per row, tokens per row), in 64 bits on the CPU."""
    index, table = index.cpu(), table.detach().cpu().double()
    shape = table.shape
    if table.dim() == 2:
        table, index = table.unsqueeze(0), index.unsqueeze(0)
    B, N, D = table.shape
    flat = index.reshape(B, -1) if B else index.reshape(0, 0)
    ok = (flat >= 0) & (flat < N)
    key = torch.where(ok, flat + torch.arange(B).unsqueeze(1) * N, torch.full_like(flat, B * N))
    key = key.reshape(-1)
    padded = torch.cat([table.reshape(B * N, D), torch.zeros(1, D, dtype=torch.float64)])
    out = padded[key] * scale
    if grad is None:
        return out
    g = grad.cpu().double().reshape(-1, D)
    tot = torch.zeros(B * N + 1, D, dtype=torch.float64).index_add_(0, key, g)[:-1] * scale
    mag = torch.zeros(B * N + 1, D, dtype=torch.float64).index_add_(0, key, g.abs())[:-1]
    cnt = torch.bincount(key, minlength=B * N + 1)[:-1]
    return out, tot.reshape(shape), (mag * abs(scale)).reshape(shape), cnt


def _check_out(out, ref):
    dt = out.dtype
    err = (out.detach().cpu().double().reshape(ref.shape) - ref).abs()
    tol = (_half_step(dt) + _wide_step(dt)) * ref.abs()
    if dt == torch.float16:
        tol = tol + 2.0 ** -25
    assert (err <= tol).all(), float((err - tol).max())


def _check_grad(ge, ref, mag, cnt):
    dt = ge.dtype
    assert torch.isfinite(ge).all()
    err = (ge.cpu().double() - ref).abs()
    m = (cnt.double() + 2).reshape(*ref.shape[:-1], 1)
    tol = m * _wide_step(dt) * mag * 1.01 + _half_step(dt) * ref.abs() * 1.01
    if dt == torch.float16:
        tol = tol + 2.0 ** -25
    assert (err <= tol).all(), float((err - tol).max())
    assert (ge.cpu()[cnt.reshape(ref.shape[:-1]) == 0] == 0).all()


def _index(kind, n, N, gen):
    if kind == 'random':
        return torch.randint(-1, N, (n,), generator=gen)
    if kind == 'one':  # one row for every token
        return torch.full((n,), N // 2)
    if kind == 'runs':  # an image's runs of the same face, with background
        return (torch.arange(n) // 37 * 7919) % (N + 1) - 1
    if kind == 'none':  # nothing is looked up
        return torch.randint(0, 2, (n,), generator=gen) * (N + 1) - 1
    if kind == 'wild':  # far outside
        i = torch.randint(0, N, (n,), generator=gen)
        i[::3] = 2 ** 40
        i[1::7] = -2 ** 62
        return i
    raise KeyError(kind)


def _run(index, table, scale, grad):
    from kaolin_amd.render.mesh import surface_embedding
    t = table.detach().requires_grad_(True)
    out = surface_embedding(index, t, scale)
    return out, torch.autograd.grad(out, t, grad)[0]


CASES = [
    # dtype, kind, tokens, rows, channels, scale
    ('f32', 'random', 1, 1, 1, 1.0), ('f32', 'random', 1, 1000, 3, -2.5),
    ('f32', 'random', 63, 5, 16, 0.5), ('f32', 'random', 4097, 300, 37, 1.5),
    ('f32', 'one', 20000, 10, 12, 1.0), ('f32', 'one', 70001, 3, 5, 1.0),
    ('f32', 'runs', 50000, 70000, 4, 3.0), ('f32', 'none', 5000, 100, 8, 1.0),
    ('f32', 'wild', 5000, 257, 33, 1.0), ('f32', 'random', 300, 7, 700, 1.0),
    ('f32', 'random', 9000, 200000, 20, 0.0),
    ('f64', 'random', 3001, 50, 7, 1.25), ('f64', 'one', 9000, 4, 130, 1.0),
    ('f64', 'runs', 20000, 255, 2, 1.0),
    ('f16', 'random', 8192, 256, 64, 0.125), ('f16', 'one', 30000, 2, 24, 1.0),
    ('f16', 'runs', 12345, 999, 17, 4.0), ('f16', 'random', 10, 3, 1, 1.0),
    ('bf16', 'random', 40000, 65535, 64, 8.0), ('bf16', 'runs', 100000, 500, 256, 1.0),
    ('bf16', 'one', 16385, 65536, 8, 1.0), ('bf16', 'random', 5000, 11, 300, -1.0),
    ('bf16', 'none', 1, 1, 8, 1.0), ('bf16', 'runs', 4096, 17000000, 2, 1.0),
]


@pytest.mark.parametrize('dname,kind,n,N,D,scale', CASES, ids=str)
def test_lookup_and_gradient(dname, kind, n, N, D, scale):
    dt = TYPES[dname]
    gen = torch.Generator().manual_seed(n * 31 + N + D)
    index = _index(kind, n, N, gen).to(DEV)
    table = torch.randn(N, D, generator=gen).to(DEV, dt)
    grad = torch.randn(n, D, generator=gen).to(DEV, dt)
    out, ge = _run(index, table, scale, grad)
    assert out.shape == (n, D) and out.dtype == dt and ge.dtype == dt
    ref, rg, mag, cnt = _reference(index, table, scale, grad)
    _check_out(out, ref)
    _check_grad(ge, rg, mag, cnt)
    out2, ge2 = _run(index, table, scale, grad)
    assert torch.equal(out, out2) and torch.equal(ge, ge2)  # a fixed order of the sums


@pytest.mark.parametrize('kind', ['random', 'one', 'runs', 'wild'])
@pytest.mark.parametrize('n,N,D', [(2, 1024, 40), (1023, 1025, 3), (1024, 1, 9), (1025, 3000, 300),
                                   (8191, 1024, 16), (16383, 40000, 8), (16384, 1025, 33),
                                   (16384, 2, 600), (16385, 1024, 8), (16385, 30000, 1)])
def test_around_the_sort_s_sizes(kind, n, N, D):
    """One workgroup's tokens and a token more, a digit's keys and one more, borders joined by the last
    workgroup and by a launch of their own."""
    gen = torch.Generator().manual_seed(n + N)
    index = _index(kind, n, N, gen).to(DEV)
    table = torch.randn(N, D, generator=gen).to(DEV)
    grad = torch.randn(n, D, generator=gen).to(DEV)
    out, ge = _run(index, table, 1.0, grad)
    ref, rg, mag, cnt = _reference(index, table, 1.0, grad)
    _check_out(out, ref)
    _check_grad(ge, rg, mag, cnt)
    assert torch.equal(ge, _run(index, table, 1.0, grad)[1])


@pytest.mark.parametrize('shape,N,D', [((3, 20, 30), 50, 16), ((2, 7), 9, 5), ((1, 4, 4), 6, 8),
                                       ((5, 0), 4, 3)])
def test_table_per_batch_entry(shape, N, D):
    gen = torch.Generator().manual_seed(5)
    index = torch.randint(-1, N + 1, shape, generator=gen).to(DEV)
    table = torch.randn(shape[0], N, D, generator=gen).to(DEV)
    grad = torch.randn(*shape, D, generator=gen).to(DEV)
    out, ge = _run(index, table, 2.0, grad)
    assert out.shape == (*shape, D)
    ref, rg, mag, cnt = _reference(index, table, 2.0, grad)
    _check_out(out, ref)
    _check_grad(ge, rg, mag, cnt)


def test_shared_indices_in_a_batch():
    """faces of shape (F, 3) expanded over the batch (stride 0), tables per view."""
    gen = torch.Generator().manual_seed(6)
    faces = torch.randint(0, 40, (60, 3), generator=gen).to(DEV)
    table = torch.randn(4, 40, 6, generator=gen).to(DEV)
    grad = torch.randn(4, 60, 3, 6, generator=gen).to(DEV)
    index = faces.expand(4, 60, 3)
    out, ge = _run(index, table, 1.0, grad)
    assert torch.equal(out, torch.stack([t[faces] for t in table]))
    _, rg, mag, cnt = _reference(index, table, 1.0, grad)
    _check_grad(ge, rg, mag, cnt)


@pytest.mark.parametrize('dname', ['f32', 'bf16'])
def test_strides_and_alignment(dname):
    """Transposed, stepped, expanded and misaligned inputs give what their copies give."""
    dt = TYPES[dname]
    gen = torch.Generator().manual_seed(7)
    N, D, h, w = 91, 16, 20, 33
    index = torch.randint(-1, N, (w, h), generator=gen).to(DEV).t()
    wide = torch.randn(N, 2 * D, generator=gen).to(DEV, dt)
    table = wide[:, ::2]
    grad = torch.randn(D, h, w, generator=gen).to(DEV, dt).permute(1, 2, 0)
    assert not (index.is_contiguous() or table.is_contiguous() or grad.is_contiguous())
    a = _run(index, table, 1.5, grad)
    b = _run(index.contiguous(), table.contiguous(), 1.5, grad.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # one element off a 16-byte boundary
    flat = torch.zeros(N * D + 1, device=DEV, dtype=dt)
    off = flat[1:].view(N, D)
    off.copy_(table)
    gflat = torch.zeros(h * w * D + 1, device=DEV, dtype=dt)
    goff = gflat[1:].view(h, w, D)
    goff.copy_(grad)
    assert off.data_ptr() % 16 and goff.data_ptr() % 16
    c = _run(index, off, 1.5, goff)
    assert torch.equal(a[0], c[0])
    ref, rg, mag, cnt = _reference(index, table, 1.5, grad)
    _check_grad(c[1], rg, mag, cnt)
    # the gradient of a plain sum arrives expanded (stride 0)
    from kaolin_amd.render.mesh import surface_embedding
    t = table.detach().contiguous().requires_grad_(True)
    surface_embedding(index, t).sum().backward()
    want = torch.bincount(index[index >= 0].reshape(-1), minlength=N)
    assert torch.equal(t.grad, want.unsqueeze(1).expand(N, D).to(dt))


def test_nothing_to_look_up():
    from kaolin_amd.render.mesh import surface_embedding
    for shape, N, D in (((0,), 5, 4), ((3, 0, 2), 5, 4), ((6,), 0, 4), ((6,), 5, 0)):
        index = torch.zeros(shape, dtype=torch.long, device=DEV)
        t = torch.randn(N, D, device=DEV, requires_grad=True)
        out = surface_embedding(index, t)
        assert out.shape == (*shape, D)
        if N == 0:
            assert (out == 0).all()
        ge, = torch.autograd.grad(out.sum(), t)
        assert ge.shape == t.shape and (N == 0 or D == 0 or (ge == 0).all())


def test_values_in_background_and_in_unused_rows():
    """NaN and infinities reach only what they belong to."""
    gen = torch.Generator().manual_seed(8)
    index = torch.tensor([3, -1, 0, 3, 9, 1], device=DEV)
    table = torch.randn(5, 8, generator=gen).to(DEV)
    table[2] = float('nan')  # never looked up
    table[1, 3] = float('inf')
    grad = torch.randn(6, 8, generator=gen).to(DEV)
    grad[1], grad[4] = float('nan'), float('inf')  # no row
    out, ge = _run(index, table, 2.0, grad)
    assert (out[1] == 0).all() and (out[4] == 0).all()
    assert torch.equal(out[5], table[1] * 2) and torch.equal(out[0], table[3] * 2)
    assert torch.isfinite(ge).all() and (ge[2] == 0).all() and (ge[4] == 0).all()
    assert torch.equal(ge[0], grad[2] * 2)


def test_gradient_by_differences():
    """The lookup is linear: differences in float64 are exact up to rounding."""
    from kaolin_amd.render.mesh import surface_embedding
    gen = torch.Generator().manual_seed(9)
    index = torch.randint(-1, 7, (3, 11), generator=gen).to(DEV)
    t = torch.randn(6, 5, generator=gen, dtype=torch.float64).to(DEV).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda e: surface_embedding(index, e, 1.75), (t,))


def test_no_second_derivative_and_no_gradient_asked():
    from kaolin_amd.render.mesh import surface_embedding
    index = torch.zeros(4, dtype=torch.long, device=DEV)
    t = torch.randn(3, 4, device=DEV, requires_grad=True)
    with torch.no_grad():
        assert not surface_embedding(index, t).requires_grad
    assert not surface_embedding(index, t.detach()).requires_grad
    g, = torch.autograd.grad(surface_embedding(index, t).pow(2).sum(), t, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_results_past_32_bit_offsets():
    """More than 2^31 elements in the output and in its gradient."""
    n, D, N = 8400003, 256, 1000
    index = torch.arange(n, device=DEV) * 7 % (N + 1) - 1
    table = torch.randn(N, D, device=DEV).to(torch.bfloat16)
    from kaolin_amd.render.mesh import surface_embedding
    t = table.requires_grad_(True)
    out = surface_embedding(index, t, 2.0)
    for s in (slice(0, 1000), slice(n // 2, n // 2 + 1000), slice(n - 1000, n)):
        i = index[s]
        want = torch.where((i >= 0).unsqueeze(1), table.detach()[i.clamp(min=0)] * 2,
                           torch.zeros((), device=DEV, dtype=torch.bfloat16))
        assert torch.equal(out[s], want)
    ge, = torch.autograd.grad(out, t, torch.ones_like(out))
    cnt = torch.bincount(index[index >= 0], minlength=N) * 2
    assert torch.equal(ge, cnt.unsqueeze(1).expand(N, D).to(torch.bfloat16))


def test_other_stream():
    gen = torch.Generator().manual_seed(10)
    index = torch.randint(-1, 500, (30000,), generator=gen).to(DEV)
    table = torch.randn(500, 24, generator=gen).to(DEV)
    grad = torch.randn(30000, 24, generator=gen).to(DEV)
    want = _run(index, table, 1.0, grad)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _run(index, table, 1.0, grad)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_captured_lookups_replay():
    """Two captured graphs (workspaces of their own) replayed in turn with eager work between."""
    from kaolin_amd.render.mesh import surface_embedding
    gen = torch.Generator().manual_seed(11)
    setups = []
    for n, N, D in ((5000, 300, 16), (20000, 70, 37)):
        index = torch.randint(-1, N, (n,), generator=gen).to(DEV)
        table = torch.randn(N, D, generator=gen).to(DEV)
        grad = torch.randn(n, D, generator=gen).to(DEV)
        t = table.clone().requires_grad_(True)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.autograd.grad(surface_embedding(index, t), t, grad)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = surface_embedding(index, t)
            ge, = torch.autograd.grad(out, t, grad)
        setups.append((graph, index, t, grad, out, ge))
    for rep in range(3):
        for graph, index, t, grad, out, ge in setups:
            with torch.no_grad():
                index.copy_(index.roll(17))
                t.mul_(1.25)
                grad.mul_(-0.5)
            out.fill_(float('nan'))
            ge.fill_(float('nan'))
        for graph, *_ in setups:
            graph.replay()
        for graph, index, t, grad, out, ge in setups:
            eo, eg = _run(index, t, 1.0, grad)
            assert torch.equal(out, eo) and torch.equal(ge, eg), rep
        torch.cuda.synchronize()
