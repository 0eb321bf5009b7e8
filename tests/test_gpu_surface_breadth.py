"""GPU: the surface operators' choices by size that other sizes do not reach, and their largest calls."""
import pytest
import torch

from test_gpu_embedding import _check_grad, _check_out, _index, _reference, _run

pytestmark = pytest.mark.gpu

DEV = 'cuda'
TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


def test_more_than_2_to_the_24_workgroups():
    """Rows of more than 512 vectors take a workgroup each: a grid of one dimension holds 2^24 of them."""
    from kaolin_amd.render.mesh import surface_embedding
    n, N, D = (1 << 24) + 5, 7, 4097
    if torch.cuda.mem_get_info()[0] < n * D * 2 + (1 << 33):
        pytest.skip('needs 150 GB of free device memory')
    index = torch.arange(n, device=DEV) % (N + 1) - 1
    table = torch.randn(N, D, device=DEV).half()
    out = surface_embedding(index, table, 2.0)
    for s in (slice(0, 100), slice((1 << 20) - 50, (1 << 20) + 50), slice(n - 100, n)):
        i = index[s]
        want = torch.where((i >= 0).unsqueeze(1), table[i.clamp(min=0)] * 2, table.new_zeros(()))
        assert torch.equal(out[s], want)
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize('dname,kind,n,N,D', [
    # eight tokens a thread in the sort's launches (2^19 to 2^22 tokens)
    ('f32', 'random', 600001, 100002, 37), ('f32', 'runs', 524289, 3000, 4),
    ('bf16', 'random', 2000003, 50000, 8), ('bf16', 'one', 2000003, 50000, 8),
    ('f16', 'wild', 1048577, 1 << 20, 2),
    # sixteen
    ('bf16', 'runs', 4194305, 70000, 2),
    # three and four passes in launches of their own
    ('f32', 'random', 20000, 2000000, 1), ('f32', 'one', 16385, (1 << 20) + 1, 2),
    ('bf16', 'runs', 40000, 3000000, 3), ('f32', 'wild', 70000, (1 << 30) + 1, 1),
    # borders joined by the last workgroup in several rounds: of columns, of workgroups, of both
    ('f32', 'one', 200, 9, 300), ('f32', 'runs', 200, 9, 300), ('f32', 'random', 200, 9, 600),
    ('f32', 'one', 4000, 50, 37), ('f32', 'runs', 4000, 50, 37), ('bf16', 'one', 250, 3, 1000),
    ('f32', 'one', 900, 20, 256), ('f32', 'runs', 900, 20, 256),
], ids=str)
def test_choices_by_size(dname, kind, n, N, D):
    gen = torch.Generator().manual_seed(n * 31 + N + D)
    dt = TYPES[dname]
    index = _index(kind, n, N, gen)
    if N > 1 << 25:  # the rows that are looked at are few: all of them among the last ones
        index = torch.where((index >= 0) & (index < N), N - 1 - index % 5000, index)
    index = index.to(DEV)
    grad = torch.randn(n, D, generator=gen).to(DEV, dt)
    if N > 1 << 25:
        table = torch.zeros(N, D, device=DEV, dtype=dt)
        table[-5000:] = torch.randn(5000, D, generator=gen).to(DEV, dt)
        out, ge = _run(index, table, 1.5, grad)
        inside = (index >= 0) & (index < N)
        low = torch.where(inside, index - (N - 5000), torch.full_like(index, -1))
        ref, rg, mag, cnt = _reference(low, table[-5000:], 1.5, grad)
        _check_out(out, ref)
        _check_grad(ge[-5000:], rg, mag, cnt)
        assert not ge[:-5000].any()
        return
    table = torch.randn(N, D, generator=gen).to(DEV, dt)
    out, ge = _run(index, table, 1.5, grad)
    ref, rg, mag, cnt = _reference(index, table, 1.5, grad)
    _check_out(out, ref)
    _check_grad(ge, rg, mag, cnt)
    assert torch.equal(ge, _run(index, table, 1.5, grad)[1])


@pytest.mark.parametrize('dname', ['f32', 'f16', 'bf16'])
def test_both_gradients_of_one_table(dname):
    """A rendered image plus the lookup at its face_idx against the same table: the table's gradient is
    the loss's and the lookup's, added.  From the pixels as they are (rounded), with the bounds of the
    single operators: te and tx of the cross entropy (see test_gpu_xent), tx added up over a row's
    pixels, a rounding u of each of the two gradients and of their sum, m 2^-24 for a sum of m terms."""
    from test_gpu_xent import _reference as xent_reference
    from kaolin_amd import workloads
    from kaolin_amd.metrics.render import surface_cross_entropy
    from kaolin_amd.render.mesh import dibr_rasterization, prepare_vertices, surface_embedding
    dt, D, scale = TYPES[dname], 12, 2.0
    s = workloads.sphere_views(20, 26, 64, 64, 2, DEV)
    g = torch.Generator().manual_seed(14)
    faces, F = s['faces'], s['faces'].shape[0]
    vfeat = torch.randn(s['vertices'].shape[0], D, generator=g).to(DEV)
    table = torch.randn(F, D, generator=g).to(DEV, dt).requires_grad_(True)
    fvc, fvi, nrm = prepare_vertices(s['vertices'].unsqueeze(0), faces, s['proj'],
                                     camera_transform=s['cam'])
    feats = surface_embedding(faces, vfeat, 0.5).unsqueeze(0).expand(2, -1, -1, -1)
    image, _, face_idx = dibr_rasterization(64, 64, fvc[..., 2], fvi, feats, nrm[..., 2])
    rendered = surface_embedding(face_idx, table)
    pixels = image.to(dt) + rendered
    px = pixels.detach().requires_grad_(True)
    weight = torch.tensor(64.0, device=DEV)  # (fp16 gradients well above its smallest numbers)
    loss = surface_cross_entropy(pixels, table, face_idx, scale)
    loss.backward(weight)
    y = face_idx.reshape(-1)
    want_loss, tl, gx, tx, ge, te = xent_reference(px.reshape(-1, D), table, y, scale, 'mean', weight)
    hit = y >= 0
    add = lambda t: torch.zeros(F, D, dtype=torch.float64, device=DEV).index_add_(  # noqa: E731
        0, y[hit], t[hit].double())
    u = torch.finfo(dt).eps / 2
    m = torch.bincount(y[hit], minlength=F).double()[:, None]
    look = add(gx)
    tol = te + add(tx) + (m + 2) * 2.0 ** -24 * add(gx.abs()) + u * (look.abs() + add(tx)) \
        + u * (ge + look).abs() * 1.02 + (2.0 ** -25 if dname == 'f16' else 0.0)
    assert abs(float(loss.detach()) - float(want_loss)) <= float(tl)
    got = table.grad.double()
    assert ((got - ge - look).abs() <= tol).all(), float(((got - ge - look).abs() - tol).max())
    # neither part, nor nothing, would pass
    for part in (ge, look, ge + look):
        assert (part.abs() > 4 * tol).float().mean() > 0.2
