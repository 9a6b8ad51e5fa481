"""Output gradients in the layouts that autograd hands back: dense ones that begin off a 16-byte boundary, and an axis of
one with a stride of its own.  The kernels get the same numbers, so the gradients are the same bits."""
import pytest
import torch

from tests.test_training_gpu import inputs

pytestmark = pytest.mark.gpu


def same(got, want):
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('d,r,dtype', [(64, 128, torch.bfloat16), (128, 256, torch.bfloat16), (20, 12, torch.bfloat16),
                                       (64, 128, torch.float32)])
def test_gradient_off_the_alignment(d, r, dtype, sbl_lib):
    from fly_b200 import ops
    q, k, v, dout, W = inputs(2, 90, 90, 3, d, d, r, dtype)
    xs = [x.requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(ops.sblocal_attention(*xs, W, 16), xs, dout)
    for offset in (3, 8, 1):
        odd = torch.empty(offset + dout.numel(), device='cuda', dtype=dtype)[offset:].view(dout.shape).copy_(dout)
        assert odd.is_contiguous()
        same(torch.autograd.grad(ops.sblocal_attention(*xs, W, 16), xs, odd), want)
    # the gradient of a part of one flat tensor
    aux = torch.zeros(3, device='cuda', dtype=dtype)
    flat = torch.cat([aux, ops.sblocal_attention(*xs, W, 16).flatten()])
    same(torch.autograd.grad(flat, xs, torch.cat([aux, dout.flatten()])), want)


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('B,H', [(2, 3), (1, 1)])
def test_gradient_of_one_row(B, H, d, sbl_lib):
    from fly_b200 import ops
    q, k, v, dout, W = inputs(B, 1, 70, H, d, d, 2 * d, torch.bfloat16)
    xs = [x.requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(ops.sblocal_attention(*xs, W, 16), xs, dout)
    # channels first: the axis of one comes back with stride 1
    out = ops.sblocal_attention(*xs, W, 16).permute(0, 2, 3, 1)
    same(torch.autograd.grad(out, xs, dout.permute(0, 2, 3, 1).contiguous()), want)
    for stride in (1, 4):
        odd = dout.as_strided(dout.shape, (H * d, stride, d, 1))
        same(torch.autograd.grad(ops.sblocal_attention(*xs, W, 16), xs, odd), want)


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('T,S', [(1, 70), (70, 1), (1, 1)])
def test_single_rows_with_any_stride(T, S, d, sbl_lib):
    """At the C entry, dout, dq, dk and dv of one row with row strides that a tensor map cannot have."""
    import ctypes

    from fly_b200 import _cabi, ops
    B, H = 2, 3
    q, k, v, dout, W = inputs(B, T, S, H, d, d, 2 * d, torch.bfloat16)
    prob = ops.Problem(q, k, v, W, 16)
    _, stats = prob.forward_train(torch.empty(prob.workspace_bytes, dtype=torch.uint8, device='cuda'))
    want = prob.backward(dout, stats)
    got = [torch.full_like(x, 7.0) for x in want]
    for stride in (1, 0, d + 4, -8):
        g = _cabi.SblGrads()
        for name, x, axis in (('dout', dout, 't'), ('dq', got[0], 't'), ('dk', got[1], 's'), ('dv', got[2], 's')):
            setattr(g, name, x.data_ptr())
            pre = 'do' if name == 'dout' else name
            sb, sr, sh = x.stride()[:3]
            setattr(g, f'{pre}_stride_b', sb)
            setattr(g, f'{pre}_stride_{axis}', stride if x.shape[1] == 1 else sr)
            setattr(g, f'{pre}_stride_h', sh)
        g.row_stats = stats.data_ptr()
        n = prob.backward_workspace_bytes()
        ws = torch.empty(n, dtype=torch.uint8, device='cuda')
        _cabi.check(sbl_lib.sbl_backward(ctypes.byref(prob.params), ctypes.byref(g), ws.data_ptr(), n,
                                         torch.cuda.current_stream().cuda_stream))
        same(got, want)
        for x in got:
            x.fill_(7.0)
