"""Strides that the gradients on the tensor cores take or refuse, without a GPU: with a workspace that is too small a call
ends behind the check of strides and in front of the device."""
import ctypes

import pytest

from test_cabi import _params
from test_training_host import _grads


def tensor_params(T, S, d):
    p = _params(dtype=1, T=T, S=S, E=d, D=d, r=2 * d, S_total=S, sum_hi=S)
    for n in 'qkvo':
        row = 's' if n in 'kv' else 't'
        setattr(p, f'{n}_stride_b', 3 * d * max(T, S))
        setattr(p, f'{n}_stride_{row}', 3 * d)
        setattr(p, f'{n}_stride_h', d)
    return p


def tensor_grads(d, **over):
    g = _grads()
    for n in ('do', 'dq', 'dk', 'dv'):
        row = 's' if n in ('dk', 'dv') else 't'
        setattr(g, f'{n}_stride_b', 300 * d)
        setattr(g, f'{n}_stride_{row}', 3 * d)
        setattr(g, f'{n}_stride_h', d)
    for n, v in over.items():
        setattr(g, n, v)
    return g


@pytest.mark.parametrize('d', [64, 128])
def test_row_strides(d, sbl_lib):
    def call(T, S, **over):
        return sbl_lib.sbl_backward(ctypes.byref(tensor_params(T, S, d)), ctypes.byref(tensor_grads(d, **over)), 4096, 256,
                                    None)

    for name in ('do_stride_t', 'dq_stride_t', 'dk_stride_s', 'dv_stride_s'):
        T, S = (1, 90) if name.endswith('_t') else (90, 1)
        for stride in (1, 0, -8, d + 4, d - 8):
            # refused where rows follow one another, taken where there is one
            assert call(90, 90, **{name: stride}) == -1, (name, stride)
            assert '16-byte aligned' in sbl_lib.sbl_last_error().decode()
            assert call(T, S, **{name: stride}) == -3, (name, stride, sbl_lib.sbl_last_error())
    assert call(90, 90) == -3
    assert call(1, 1, dout=4098) == -1
