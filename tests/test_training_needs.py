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


def test_rotation_side_without_a_place_is_left_out(sbl_lib):
    from test_training_host import _rotary
    p, n = _rotary(), ctypes.c_size_t(0)
    p.side[0].y = None
    p.side[1].dweight = 4096
    assert sbl_lib.sbl_norm_rotary_forward(ctypes.byref(p), None) == -1
    # (-3: behind the checks of the sides, the workspace is missing)
    assert sbl_lib.sbl_norm_rotary_backward(ctypes.byref(p), None, 0, None) == -3
    assert sbl_lib.sbl_norm_rotary_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0 and n.value > 0
    p.side[0].dweight = 4096
    assert sbl_lib.sbl_norm_rotary_backward(ctypes.byref(p), None, 0, None) == -1
    p.side[0].dweight = p.side[1].dweight = p.side[1].y = None
    assert sbl_lib.sbl_norm_rotary_backward(ctypes.byref(p), None, 0, None) == 0      # nothing to do


@pytest.mark.gpu
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('B,T,S,Hq,Hk,E,dtype', [
    (2, 1300, 1300, 5, 2, 64, torch.bfloat16), (3, 7, 7, 16, 4, 128, torch.bfloat16), (2, 40, 90, 3, 3, 64, torch.float32),
    (2, 300, 300, 3, 2, 21, torch.float32), (2, 300, 0, 3, 2, 64, torch.float32)])
def test_any_part_of_the_rotation(B, T, S, Hq, Hk, E, dtype, interleaved, sbl_lib):
    from fly_b200 import ops
    from tests.test_norm_rotary_gpu import make
    q, k, wq, wk, dq, dk = make(B, T, S, Hq, Hk, E, dtype, seed=3)
    xs = (q, k, wq, wk)
    whole = [x.clone().requires_grad_() for x in xs]
    want = torch.autograd.grad(ops.qk_norm_rotary(*whole, interleaved=interleaved), whole, (dq, dk))
    for needs in itertools.product((False, True), repeat=4):
        if not any(needs):
            continue
        leaves = [x.clone().requires_grad_(n) for x, n in zip(xs, needs)]
        torch.autograd.backward(ops.qk_norm_rotary(*leaves, interleaved=interleaved), (dq, dk))
        for x, need, y in zip(leaves, needs, want):
            assert (x.grad is not None) == need and (not need or torch.equal(x.grad, y))
