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
