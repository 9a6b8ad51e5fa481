"""Gradients of batches without a real key: zeros, whatever the queries and the output's gradient are.

Such a row's normaliser is the floor of the division, so a feature over it is about 1e37 (1e24 in the kernels for any
shape): with queries of zero and gradients of one sign a sum over some hundred rows leaves the fp32 range."""
import pytest
import torch

from oracle.training_oracle import sblocal_grads
from tests.test_training_gpu import BF16_ANY, BF16_TENSOR, FP32, check, grads_of, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('d,dtype,size,tol', [(64, torch.bfloat16, 1.0, BF16_TENSOR), (128, torch.bfloat16, 1.0, BF16_TENSOR),
                                              (32, torch.bfloat16, 1e16, BF16_ANY), (32, torch.float32, 1e16, FP32)],
                         ids=['64', '128', 'any-bf16', 'any-fp32'])
@pytest.mark.parametrize('T,S', [(300, 300), (1500, 1500), (40, 700)])
def test_batches_without_keys(T, S, d, dtype, size, tol, sbl_lib):
    q, k, v, dout, W = inputs(3, T, S, 2, d, d, 2 * d, dtype, seed=5)
    lengths = torch.tensor([0, S, 0], device='cuda')
    q[0] = 0                                             # a padded batch, and one of small queries
    q[2] *= 1e-3
    dout[0], dout[2] = size, -size
    got = grads_of(q, k, v, dout, W, 24, None, lengths)
    for x in got:
        assert (x[0] == 0).all() and (x[2] == 0).all()
    one = slice(1, 2)
    check([x[one] for x in got], sblocal_grads(q[one], k[one], v[one], dout[one], W, 24), tol)
