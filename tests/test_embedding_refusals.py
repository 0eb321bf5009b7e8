"""CPU: what surface_embedding and surface_cross_entropy refuse, and their workspace queries."""
import pytest
import torch

from kaolin_amd import _C, _lib
from kaolin_amd.metrics.render import surface_cross_entropy
from kaolin_amd.render.mesh import surface_embedding

NEVER = torch.device('meta')  # a device without data: refused before anything is read


def _embed(**kw):
    a = dict(index=torch.zeros(4, dtype=torch.long), embeddings=torch.zeros(3, 5), scale=1.0)
    a.update(kw)
    return a['index'], a['embeddings'], a['scale']


def test_operators_need_a_gpu():
    with pytest.raises(RuntimeError, match='on a GPU'):
        surface_embedding(*_embed())
    with pytest.raises(RuntimeError, match='on a GPU'):
        surface_cross_entropy(torch.zeros(4, 5), torch.zeros(3, 5),
                              torch.zeros(4, dtype=torch.long))


@pytest.mark.parametrize('kw,what', [
    (dict(index=torch.zeros(4, dtype=torch.int32)), 'dtype torch.int64'),
    (dict(index=torch.zeros(4)), 'dtype torch.int64'),
    (dict(embeddings=torch.zeros(5)), 'embeddings must be'),
    (dict(embeddings=torch.zeros(2, 2, 3, 5)), 'embeddings must be'),
    (dict(embeddings=torch.zeros(3, 6, 5)), 'a table per batch entry'),
    (dict(scale=float('nan')), 'finite'),
    (dict(scale=float('inf')), 'finite'),
    (dict(scale=torch.tensor(2.0)), 'a number'),
    (dict(scale=True), 'a number'),
    (dict(embeddings=torch.empty(1, 2 ** 20 + 1, device=NEVER)), '2\\^20 channels'),
    (dict(embeddings=torch.empty(2 ** 31, 1, device=NEVER)), '2\\^31 embeddings'),
    (dict(index=torch.empty(2 ** 31, dtype=torch.long, device=NEVER)), '2\\^31 indices'),
], ids=str)
def test_embedding_arguments(kw, what):
    index, table, scale = _embed(**kw)
    with pytest.raises(RuntimeError, match=what):
        _C._embedding_args('surface_embedding', index, table.shape, scale)


def test_embedding_types():
    for dt in (torch.float32, torch.float64, torch.float16, torch.bfloat16):
        assert _C._sfx16(torch.zeros(1, dtype=dt), 'x')
    for dt in (torch.int64, torch.uint8, torch.complex64, torch.bool):
        with pytest.raises(RuntimeError, match='not implemented'):
            _C._sfx16(torch.zeros(1, dtype=dt), 'x')
    with pytest.raises(RuntimeError, match='not implemented'):
        _C._sfx16(torch.zeros(1, dtype=torch.float64), 'x', double=False)


def test_workspace_queries():
    lib = _lib.load()
    size = lib.kd_surface_embedding_workspace_size
    assert size(1000, 1, 50, 16, 4) > 4 * 4 * 1000
    assert size(2 ** 23, 1, 50000, 32, 2) < 2 ** 30
    for bad in ((0, 1, 50, 16, 4), (2 ** 31, 1, 50, 16, 4), (10, 0, 50, 16, 4),
                (10, 4, 2 ** 30, 16, 4), (10, 1, 50, 2 ** 20 + 1, 4), (10, 1, 50, 16, 3)):
        assert size(*bad) == 0, bad
    state, scratch = lib.kd_surface_xent_state_size, lib.kd_surface_xent_scratch_size
    assert state(1000, 50, 16, 4, 1, 1) > state(1000, 50, 16, 4, 0, 0) > 0
    assert state(0, 50, 16, 4, 1, 1) > 0  # an empty call has a gradient of zeros
    for bad in ((-1, 50, 16, 4, 1, 1), (10, 0, 16, 4, 1, 1), (10, 50, 0, 4, 1, 1),
                (10, 50, 257, 4, 1, 1), (10, 50, 16, 8, 1, 1), (2 ** 31, 50, 16, 4, 1, 1)):
        assert state(*bad) == 0 and scratch(*bad, 0) == 0 and scratch(*bad, 1) == 0, bad


def test_native_calls_refuse_before_they_launch():
    """The C entry points check sizes, pointers and workspaces on the host."""
    lib = _lib.load()
    p = 4096  # never read: every call below is refused
    for name, args, what in (
            ('kd_surface_embedding_forward_f32', (-1, 1, 5, 4, p, p, 1.0, p, None), b'indices'),
            ('kd_surface_embedding_forward_f32', (8, 3, 5, 4, p, p, 1.0, p, None), b'split'),
            ('kd_surface_embedding_forward_f32', (8, 1, 5, 4, None, p, 1.0, p, None), b'NULL'),
            ('kd_surface_embedding_forward_f32', (8, 1, 5, 4, p, None, 1.0, p, None), b'NULL'),
            ('kd_surface_embedding_backward_f16', (8, 1, 5, 4, p, p, 1.0, None, p, 1 << 30, None),
             b'NULL'),
            ('kd_surface_embedding_backward_f16', (8, 1, 5, 4, p, p, 1.0, p, p, 16, None),
             b'workspace'),
            ('kd_surface_xent_forward_bf16', (8, 5, 257, p, p, p, 1.0, 1, 1, 1, p, p, 1 << 30, p,
                                              1 << 30, None), b'channels'),
            ('kd_surface_xent_forward_bf16', (8, 0, 16, p, p, p, 1.0, 1, 1, 1, p, p, 1 << 30, p,
                                              1 << 30, None), b'embeddings'),
            ('kd_surface_xent_forward_bf16', (8, 5, 16, p, p, p, float('nan'), 1, 1, 1, p, p,
                                              1 << 30, p, 1 << 30, None), b'scale'),
            ('kd_surface_xent_forward_bf16', (8, 5, 16, p, p, p, 1.0, 3, 1, 1, p, p, 1 << 30, p,
                                              1 << 30, None), b'reduction'),
            ('kd_surface_xent_forward_bf16', (8, 5, 16, p, p, p, 1.0, 1, 1, 1, None, p, 1 << 30, p,
                                              1 << 30, None), b'loss'),
            ('kd_surface_xent_forward_bf16', (8, 5, 16, p, p, p, 1.0, 1, 1, 1, p, p, 64, p,
                                              1 << 30, None), b'workspace'),
            ('kd_surface_xent_forward_bf16', (8, 5, 16, p, p, p, 1.0, 1, 1, 1, p, p, 1 << 30, p,
                                              64, None), b'workspace'),
            ('kd_surface_xent_forward_bf16', (8, 5, 16, p, p, p, 1.0, 1, 1, 1, p, p + 16, 1 << 30, p,
                                              1 << 30, None), b'aligned'),
            ('kd_surface_embedding_backward_f16', (8, 1, 5, 4, p, p, 1.0, p, p + 16, 1 << 30, None),
             b'aligned'),
            ('kd_surface_xent_backward_f32', (8, 5, 16, p, 1.0, 1, 0, 1, p, p, p, p, 1 << 30, p,
                                              1 << 30, None), b'did not prepare'),
            ('kd_surface_xent_backward_f32', (8, 5, 16, p, 1.0, 1, 1, 1, None, p, p, p, 1 << 30, p,
                                              1 << 30, None), b'grad_loss')):
        rc = getattr(lib, name)(*args)
        assert rc != _lib.KD_OK
        assert what in lib.kd_last_error(), (what, lib.kd_last_error())
