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
