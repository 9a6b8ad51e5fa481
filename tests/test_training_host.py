"""What the training operators refuse, without a GPU: the C ABI validates before it touches a device."""
import ctypes

import pytest
import torch

from test_cabi import _params


def _grads(**over):
    from fly_b200 import _cabi
    g = _cabi.SblGrads()
    for n in ('dout', 'row_stats', 'dq', 'dk', 'dv'):
        setattr(g, n, 4096)
    for n, v in over.items():
        setattr(g, n, v)
    return g


@pytest.mark.parametrize('over,code,fragment', [
    (dict(softmax_eps=0.1), -2, 'softmax_eps'),
    (dict(q_pos0=4, T=50), -2, 'shards'),
    (dict(sum_hi=90), -2, 'shards'),
    (dict(w=0), -1, 'local_context'),
    (dict(D=200), -2, 'D=200'),
])
def test_problems_without_gradients(sbl_lib, over, code, fragment):
    p, n = _params(**over), ctypes.c_size_t(0)
    for rc in (sbl_lib.sbl_backward_workspace_bytes(ctypes.byref(p), ctypes.byref(n)),
               sbl_lib.sbl_forward_train(ctypes.byref(p), 4096, 1 << 40, 4096, None),
               sbl_lib.sbl_backward(ctypes.byref(p), ctypes.byref(_grads()), 4096, 1 << 40, None)):
        assert rc == code and fragment in sbl_lib.sbl_last_error().decode()


def test_backward_arguments(sbl_lib):
    p, n = _params(), ctypes.c_size_t(0)
    assert sbl_lib.sbl_backward_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0
    # psi, phi and f df, all fp32
    assert n.value >= 3 * 2 * 3 * 100 * 256 * 4
    call = lambda g, ws=4096, size=n.value: sbl_lib.sbl_backward(ctypes.byref(p), g, ws, size, None)  # noqa: E731
    assert call(None) == -1
    for name in ('dout', 'row_stats', 'dq', 'dk', 'dv'):
        assert call(ctypes.byref(_grads(**{name: None}))) == -1
        assert 'non-null' in sbl_lib.sbl_last_error().decode()
    g = _grads()
    g.reserved[2] = 1
    assert call(ctypes.byref(g)) == -1
    assert call(ctypes.byref(_grads()), None) == -3
    assert call(ctypes.byref(_grads()), 4096 + 16) == -3
    assert call(ctypes.byref(_grads()), 4096, n.value - 1) == -3
    assert sbl_lib.sbl_forward_train(ctypes.byref(p), 4096, 1 << 40, None, None) == -1


def _rotary(**over):
    from fly_b200 import _cabi
    p = _cabi.SblNormRotary()
    p.dtype = p.weight_dtype = _cabi.SBL_DTYPE_F32
    p.B, p.E, p.rotary, p.eps, p.theta = 2, 64, 64, 1e-6, 10000.0
    for s in p.side:
        s.T, s.H, s.x, s.y, s.dy = 5, 3, 4096, 4096, 4096
    for n, v in over.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize('over,code,fragment', [
    (dict(dtype=3), -1, 'dtype'), (dict(weight_dtype=-1), -1, 'dtype'), (dict(E=0), -1, 'E positive'),
    (dict(B=-1), -1, 'B must be'), (dict(E=513), -2, '512'), (dict(rotary=65), -1, 'even'),
    (dict(rotary=66), -1, 'even'), (dict(rotary=-2), -1, 'even'), (dict(interleaved=2), -1, 'interleaved'),
    (dict(eps=-1.0), -1, 'eps'), (dict(eps=float('nan')), -1, 'eps'), (dict(theta=0.0), -1, 'theta'),
])
def test_norm_rotary_arguments(sbl_lib, over, code, fragment):
    p, n = _rotary(**over), ctypes.c_size_t(0)
    for rc in (sbl_lib.sbl_norm_rotary_forward(ctypes.byref(p), None),
               sbl_lib.sbl_norm_rotary_workspace_bytes(ctypes.byref(p), ctypes.byref(n)),
               sbl_lib.sbl_norm_rotary_backward(ctypes.byref(p), 4096, 1 << 30, None)):
        assert rc == code and fragment in sbl_lib.sbl_last_error().decode()


def test_norm_rotary_sides_and_workspace(sbl_lib):
    p = _rotary()
    p.side[1].x = None
    assert sbl_lib.sbl_norm_rotary_forward(ctypes.byref(p), None) == -1
    p = _rotary()
    p.side[0].H = 0
    assert sbl_lib.sbl_norm_rotary_forward(ctypes.byref(p), None) == -1
    p = _rotary()
    p.side[1].dy = None
    assert sbl_lib.sbl_norm_rotary_backward(ctypes.byref(p), None, 0, None) == -1
    p, n = _rotary(), ctypes.c_size_t(0)
    p.side[0].dweight = 4096
    assert sbl_lib.sbl_norm_rotary_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0 and n.value > 0
    assert sbl_lib.sbl_norm_rotary_backward(ctypes.byref(p), None, 0, None) == -3
    assert sbl_lib.sbl_norm_rotary_backward(ctypes.byref(p), 4096, n.value - 1, None) == -3
    # nothing to do, no device touched
    p = _rotary(B=0)
    assert sbl_lib.sbl_norm_rotary_forward(ctypes.byref(p), None) == 0


def test_tensors_are_checked():
    from fly_b200 import QKNormRotary, ops
    q = torch.randn(1, 5, 2, 8)
    with pytest.raises(ValueError, match='CUDA'):
        ops.qk_norm_rotary(q, q)
    with pytest.raises(ValueError, match='CUDA'):
        QKNormRotary(8)(q, q)
    with pytest.raises(ValueError, match='CUDA'):
        ops.sblocal_attention(q.requires_grad_(), q, q, torch.randn(4, 8), 2)


def test_norm_module():
    from fly_b200 import QKNormRotary, SBLocalAttention
    m = QKNormRotary(64, rotary_dim=32, theta=500.0, interleaved=True, eps=1e-5, init=0.5)
    assert set(m.state_dict()) == {'query_weight', 'key_weight'}
    assert (m.query_weight == 0.5).all() and m.key_weight.shape == (64,)
    with pytest.raises(ValueError):
        QKNormRotary(64, rotary_dim=33)
    with pytest.raises(ValueError):
        QKNormRotary(64, rotary_dim=66)
    layer = SBLocalAttention(16, 64, 64)
    assert layer.qk_norm is None and list(layer.state_dict()) == ['feature_map.projection_matrix']
    layer.qk_norm = m
    assert len(list(layer.parameters())) == 2
