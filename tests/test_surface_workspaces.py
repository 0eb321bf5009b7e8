"""CPU: workspace sizes of surface_cross_entropy, and what a scale may be."""
import numpy as np
import pytest
import torch

from kaolin_amd import _C, _lib


@pytest.mark.parametrize('esize', [2, 4])
def test_a_few_pixels_without_gradients_need_little(esize):
    """Up to 64 pixels read the table as it stands: nothing of its size is needed beside it."""
    lib = _lib.load()
    state, scratch = lib.kd_surface_xent_state_size, lib.kd_surface_xent_scratch_size
    for n in (1, 64):
        for rows, D in ((10, 3), (200000, 256)):
            assert 0 < state(n, rows, D, esize, 0, 0) <= 256
            assert 0 < scratch(n, rows, D, esize, 0, 0, 0) <= 1 << 19
            # gradients need the packed table
            table = rows * D * esize
            for need in ((1, 0), (0, 1), (1, 1)):
                assert state(n, rows, D, esize, *need) >= table
    assert state(65, 200000, 256, esize, 0, 0) >= 200000 * 256 * esize
    assert state(0, 200000, 256, esize, 0, 0) > 0


@pytest.mark.parametrize('scale', ['2', b'2', None, [2.0], 1j, 10 ** 400, True, torch.tensor(2.0)], ids=str)
def test_a_scale_is_a_number(scale):
    with pytest.raises(RuntimeError, match='scale must be a number'):
        _C._number('surface_embedding', 'scale', scale)


@pytest.mark.parametrize('scale', [2, 2.0, np.float32(2), np.int64(2), np.float16(2)], ids=repr)
def test_numbers_of_any_kind(scale):
    assert _C._number('surface_embedding', 'scale', scale) == 2.0
