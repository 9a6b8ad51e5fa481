"""Calls of the gradients and of the norm and rotation that the other files do not make: heads shared by fewer keys over
many tokens, two calls at once, captured steps whose lengths and positions change, refusals.

Tolerances as in test_norm_rotary_gpu.py and test_training_gpu.py, whose checks are used; where two calls do the same
arithmetic on the same values their bits are compared."""
import pytest
import torch

from oracle.training_oracle import sblocal_grads
from tests.test_norm_rotary_gpu import check_side, make
from tests.test_training_gpu import BF16_TENSOR, check, grads_of, inputs

pytestmark = pytest.mark.gpu

# B, T, Hq, Hk, E, rotary, dtype: enough tokens that one warp takes a token's heads of both sides
MANY = [
    (2, 1300, 5, 2, 64, 64, torch.bfloat16),
    (2, 1300, 1, 9, 64, 32, torch.float32),
    (1, 2500, 3, 7, 128, 64, torch.bfloat16),
    (3, 801, 2, 1, 40, 16, torch.float32),          # 5 of 8 lanes hold a row
    (1, 2401, 4, 4, 256, 0, torch.bfloat16),
]


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('case', MANY, ids=lambda c: '-'.join(str(x) for x in c[:6]))
def test_many_tokens_with_shared_heads(case, interleaved, sbl_lib):
    from fly_b200 import ops
    B, T, Hq, Hk, E, rotary, dtype = case
    q, k, wq, wk, dq, dk = make(B, T, T, Hq, Hk, E, dtype, seed=7)
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    pos = torch.arange(T, device='cuda').flip(0) * 3 - 50
    y = ops.qk_norm_rotary(*leaves, positions=pos, rotary_dim=rotary, interleaved=interleaved)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    # an angle of a position of up to 7200 radians, rounded once as a fraction of a turn
    kw = dict(positions=pos, rotary=rotary, interleaved=interleaved)
    check_side(y[0], grads[0], grads[2], q, wq, dq, **kw)
    check_side(y[1], grads[1], grads[3], k, wk, dk, **kw)
    # positions of the keys' own, equal in value: the sides apart, the same values
    z = ops.qk_norm_rotary(*leaves, positions=pos, key_positions=pos.clone(), rotary_dim=rotary, interleaved=interleaved)
    assert torch.equal(z[0], y[0]) and torch.equal(z[1], y[1])
    # only one side has a weight, and only it wants a gradient
    z = ops.qk_norm_rotary(q.detach(), k.detach(), None, wk, positions=pos, rotary_dim=rotary, interleaved=interleaved)
    g, = torch.autograd.grad(z, (wk,), (dq, dk))
    assert torch.equal(z[1], y[1]) and torch.equal(g, grads[3])


def test_norm_rotary_refusals(sbl_lib):
    from fly_b200 import ops
    q, k, wq, wk, _, _ = make(2, 5, 5, 2, 2, 64, torch.bfloat16)
    pos = torch.arange(5, device='cuda')
    for error, args, kw in [
            (TypeError, (q.half(), k.half()), {}),
            (TypeError, (q, k.float()), {}),
            (TypeError, (q, k, wq.half(), wk.half()), {}),
            (TypeError, (q, k, wq, wk.bfloat16()), {}),
            (ValueError, (q, k[..., :32]), {}),
            (ValueError, (q, k[:1]), {}),
            (ValueError, (q[0], k[0]), {}),
            (ValueError, (q.cpu(), k), {}),
            (ValueError, (q, k.cpu()), {}),
            (ValueError, (q, k, wq[:32], wk), {}),
            (ValueError, (q, k, wq.cpu(), wk), {}),
            (ValueError, (q, k), dict(positions=pos[:4])),
            (ValueError, (q, k), dict(positions=pos.int())),
            (ValueError, (q, k), dict(positions=pos.cpu())),
            (ValueError, (q, k), dict(key_positions=pos[None].expand(3, 5))),
            (ValueError, (q, k), dict(rotary_dim=33)),
            (ValueError, (q, k), dict(rotary_dim=66)),
            (ValueError, (q, k), dict(eps=-1.0)),
            (ValueError, (q, k), dict(theta=0.0))]:
        with pytest.raises(error):
            ops.qk_norm_rotary(*args, **kw)
    wide = torch.zeros(1, 1, 1, 514, device='cuda')
    with pytest.raises(NotImplementedError):
        ops.qk_norm_rotary(wide, wide)


def test_attention_gradient_refusals(sbl_lib):
    from fly_b200 import ops
    q, k, v, dout, W = inputs(1, 40, 40, 2, 16, 16, 8, torch.float32)
    q.requires_grad_()
    out = ops.sblocal_attention(q, k, v, W, 8, softmax_eps=1e-3)   # the forward is built, its gradients are not
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(out, q, dout)
    with pytest.raises(TypeError):
        ops.sblocal_attention(q, k.bfloat16(), v, W, 8)
    prob = ops.Problem(q.detach(), k, v, W, 8)
    _, stats = prob.forward_train(torch.empty(prob.workspace_bytes, dtype=torch.uint8, device='cuda'))
    for bad in (dout[:, :-1], dout.bfloat16(), dout.cpu()):
        with pytest.raises(ValueError):
            prob.backward(bad, stats)
    # a second derivative is refused, not wrong
    out = ops.sblocal_attention(q, k, v, W, 8)
    g, = torch.autograd.grad(out, q, dout.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)


@pytest.mark.parametrize('d,dtype', [(64, torch.bfloat16), (128, torch.bfloat16), (32, torch.float32)])
def test_captured_step_sees_new_lengths(d, dtype, sbl_lib):
    """Lengths live on the device and are read by the kernels: a replayed step follows them, down to a batch without keys,
    and what an earlier replay left in its buffers does not come back."""
    from fly_b200 import ops
    q, k, v, dout, W = inputs(3, 333, 333, 2, d, d, 2 * d, dtype, seed=4)
    lengths = torch.tensor([333, 200, 129], device='cuda')
    xs = [x.requires_grad_() for x in (q, k, v)]

    def step():
        out = ops.sblocal_attention(*xs, W, 96, key_lengths=lengths)
        grads = torch.autograd.grad(out, xs, dout)
        return (out.detach(), *grads)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for new in ((333, 200, 129), (5, 333, 0), (128, 1, 333)):
        lengths.copy_(torch.tensor(new))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        ref = sblocal_grads(q.detach(), k.detach(), v.detach(), dout, W, 96, None, lengths)
        check(got, ref, BF16_TENSOR if dtype == torch.bfloat16 else 1e-5)


@pytest.mark.parametrize('d', [64, 128])
def test_two_steps_at_once(d, sbl_lib):
    """Two steps of different problems in flight on two streams: each gives what it gives alone."""
    one, two = (inputs(2, n, n, 4, d, d, 2 * d, torch.bfloat16, seed=n) for n in (900, 1111))
    alone = [grads_of(*x[:5], 64) for x in (one, two)]
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        got = []
        for s, x in zip(streams, (one, two)):
            with torch.cuda.stream(s):
                got.append(grads_of(*x[:5], 64))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('B,H,N,d,w', [(1, 17, 300, 64, 64), (2, 33, 260, 128, 64), (1, 148, 128, 64, 32),
                                       (1, 149, 129, 64, 32)])
def test_heads_and_tiles_around_the_grid(B, H, N, d, w, sbl_lib):
    """More than sixteen heads (a block of the row kernel), and one tile per SM or one more."""
    q, k, v, dout, W = inputs(B, N, N, H, d, d, 2 * d, torch.bfloat16, seed=2)
    got = grads_of(q, k, v, dout, W, w)
    check(got, sblocal_grads(q, k, v, dout, W, w, None, None), BF16_TENSOR)
