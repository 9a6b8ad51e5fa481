"""Gradients that nobody needs are not formed, and the others are the same bits without them."""
import ctypes
import itertools

import pytest
import torch

from test_cabi import _params
from test_training_host import _grads
from test_training_strides import tensor_grads, tensor_params

NEEDS = [n for n in itertools.product((False, True), repeat=3) if any(n)]


def test_pointers_of_skipped_gradients_may_be_null(sbl_lib):
    for p, make in ((_params(), _grads), (tensor_params(90, 90, 64), lambda **over: tensor_grads(64, **over))):
        def call(p, **over):
            return sbl_lib.sbl_backward(ctypes.byref(p), ctypes.byref(make(**over)), 4096, 256, None)

        # (-3: behind every check of the gradients, the workspace is too small)
        assert call(p) == -3
        for name, bit in (('dq', 1), ('dk', 2), ('dv', 4)):
            assert call(p, **{name: None, 'skip': bit}) == -3
            assert call(p, **{name: None, 'skip': 7 - bit}) == -1
        assert call(p, dq=None, dk=None, dv=None, skip=7) == -3
        assert call(p, dout=None, skip=7) == -1
        for bits in (8, -1):
            assert call(p, skip=bits) == -1 and 'skip' in sbl_lib.sbl_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize('d,r,dtype', [(64, 128, torch.bfloat16), (128, 256, torch.bfloat16), (20, 12, torch.bfloat16),
                                       (24, 16, torch.float32)])
def test_any_part_of_the_gradients(d, r, dtype, sbl_lib):
    from fly_b200 import ops
    from tests.test_training_gpu import inputs
    q, k, v, dout, W = inputs(2, 300, 260, 3, d, d, r, dtype, seed=8)
    lengths = torch.tensor([260, 100], device='cuda')
    whole = [x.clone().requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(ops.sblocal_attention(*whole, W, 40, key_lengths=lengths), whole, dout)
    for needs in NEEDS:
        xs = [x.clone().requires_grad_(n) for x, n in zip((q, k, v), needs)]
        out = ops.sblocal_attention(*xs, W, 40, key_lengths=lengths)
        out.backward(dout)
        for x, need, y in zip(xs, needs, want):
            assert (x.grad is not None) == need and (not need or torch.equal(x.grad, y))
        # one call's graph, asked for a part
        part = [x for x, n in zip(whole, needs) if n]
        got = torch.autograd.grad(ops.sblocal_attention(*whole, W, 40, key_lengths=lengths), part, dout)
        assert all(torch.equal(a, b) for a, b in zip(got, [y for y, n in zip(want, needs) if n]))
    prob = ops.Problem(q, k, v, W, 40)
    _, stats = prob.forward_train(torch.empty(prob.workspace_bytes, dtype=torch.uint8, device='cuda'))
    every = prob.backward(dout, stats)
    for needs in NEEDS:
        got = prob.backward(dout, stats, needs=needs)
        assert all(torch.equal(a, b) if n else a is None for a, b, n in zip(got, every, needs))
