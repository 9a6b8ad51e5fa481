"""Gradients of SBLocal attention (`ops.sblocal_attention`, the module under autograd) against the definition in 64
bits, differentiated by autograd.

Metric: |x - ref| / |ref| in the 2-norm per tensor.  Tolerances:
  fp32   exponents of up to about 12 and their exp are off by 16 * 2^-24; every other step adds a few 2^-24; the sums
         outside the window are differences of sums up to 8 times as large: 8 * 20 * 2^-24 = 1e-5;
  bf16   independent roundings of half a step, 2^-8, each: the kernels for any shape round the output (through delta)
         and the result, sqrt(2) * 2^-8; the tensor-core kernels also features, summaries, g, p g and du of either
         side: sqrt(9) * 2^-8 = 1.2e-2.
"""
import pytest
import torch

from oracle.training_oracle import rel2, sblocal_dense, sblocal_grads

pytestmark = pytest.mark.gpu

FP32 = 1e-5
BF16_ANY = 2 ** 0.5 * 2.0 ** -8
BF16_TENSOR = 3 * 2.0 ** -8


def inputs(B, T, S, H, E, D, r, dtype, tau=None, seed=0):
    """Logits of unit scale, an orthogonal-block projection."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    scale = ((tau or E ** -0.5) * E) ** -0.5
    q, k = (n(B, T, H, E) * scale).to(dtype), (n(B, S, H, E) * scale).to(dtype)
    v, dout = n(B, S, H, D).to(dtype), n(B, T, H, D).to(dtype)
    blocks = -(-r // E)
    rows = torch.linalg.qr(n(blocks, E, E))[0].transpose(1, 2).reshape(-1, E)[:r]
    return q, k, v, dout, (rows * n(r, E).norm(dim=1, keepdim=True)).contiguous()


def grads_of(q, k, v, dout, W, w, tau=None, lengths=None):
    from fly_b200 import ops
    xs = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.sblocal_attention(*xs, W, w, tau, key_lengths=lengths)
    return (out.detach(), *torch.autograd.grad(out, xs, dout))


def check(got, ref, tol):
    names = ('out', 'dq', 'dk', 'dv')
    errs = {n: rel2(x, y) for n, x, y in zip(names, got, ref)}
    assert all(torch.isfinite(x).all() for x in got)
    assert max(errs.values()) <= tol, errs


GRID = [
    # B, H, T, S, E, D, r, w, tau, lengths
    (2, 3, 47, 39, 21, 17, 13, 28, 0.235, (39, 22)),
    (1, 2, 1, 5, 16, 16, 8, 4, None, None),           # one query
    (2, 1, 130, 130, 64, 64, 128, 1, None, None),     # a window of one key
    (1, 2, 65, 65, 64, 64, 128, 200, None, None),     # every key in the window
    (2, 2, 200, 300, 32, 48, 20, 33, None, (300, 7)),
    (2, 2, 300, 70, 32, 128, 20, 64, None, (70, 0)),  # rows far behind the last key; a batch without keys
    (1, 1, 190, 190, 130, 20, 30, 50, None, None),    # head dim over one column block
    (1, 1, 70, 70, 200, 128, 300, 16, None, None),
    (2, 1, 100, 100, 8, 4, 1, 10, None, (64, 100)),   # two features
    (1, 4, 513, 513, 64, 64, 128, 256, 147 ** -0.5, None),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('case', GRID, ids=lambda c: '-'.join(str(x) for x in c[:8]))
def test_gradients_any_shape(case, dtype, sbl_lib):
    B, H, T, S, E, D, r, w, tau, lengths = case
    q, k, v, dout, W = inputs(B, T, S, H, E, D, r, dtype, tau)
    lengths = torch.tensor(lengths, device='cuda') if lengths else None
    got = grads_of(q, k, v, dout, W, w, tau, lengths)
    ref = sblocal_grads(q, k, v, dout, W, w, tau, lengths)
    tensor = dtype == torch.bfloat16 and (E, D, r) == (64, 64, 128)
    check(got, ref, FP32 if dtype == torch.float32 else BF16_TENSOR if tensor else BF16_ANY)
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            assert (got[2][b, n:] == 0).all() and (got[3][b, n:] == 0).all()
            if n == 0:
                assert (got[0][b] == 0).all() and (got[1][b] == 0).all()


TENSOR = [
    # B, H, T, S, d, w, tau, lengths: both head dims of the tensor-core kernels
    (1, 1, 128, 128, 64, 64, None, None),
    (2, 3, 1000, 1000, 64, 256, None, None),
    (2, 2, 1200, 1200, 64, 8, None, (1200, 333)),
    (1, 2, 900, 2000, 64, 100, None, None),          # more keys than queries: key tiles nobody sees
    (1, 2, 2000, 900, 64, 33, None, None),           # queries behind the last key
    (3, 2, 777, 777, 64, 257, 576 ** -0.5, (777, 128, 0)),
    (1, 1, 300, 1, 64, 16, None, None),
    (2, 1, 3, 1500, 64, 2048, None, None),
    (1, 2, 1500, 1500, 64, 1000, None, (1400,)),
    (1, 1, 16, 16, 64, 256, None, None),             # a short sequence, all of it in every window
    (4, 40, 130, 130, 64, 20, None, None),           # more tiles than SMs
    (1, 1, 128, 128, 128, 64, None, None),
    (2, 2, 1000, 1000, 128, 512, None, (1000, 513)),
    (1, 2, 700, 1900, 128, 64, None, None),
    (1, 2, 1900, 700, 128, 129, None, None),
    (2, 1, 1, 1300, 128, 5, None, None),
    (1, 1, 40, 40, 128, 512, None, None),
    (2, 40, 200, 260, 128, 4000, None, None),
]


@pytest.mark.parametrize('case', TENSOR, ids=lambda c: '-'.join(str(x) for x in c[:6]))
def test_gradients_on_the_tensor_cores(case, sbl_lib):
    from fly_b200 import ops
    B, H, T, S, d, w, tau, lengths = case
    q, k, v, dout, W = inputs(B, T, S, H, d, d, 2 * d, torch.bfloat16, tau, seed=1)
    lengths = torch.tensor(lengths, device='cuda') if lengths else None
    prob = ops.Problem(q, k, v, W, w, tau, key_lengths=lengths)
    assert (prob.status_offset is not None) == (w <= 2048 or d == 128)
    got = grads_of(q, k, v, dout, W, w, tau, lengths)
    ref = sblocal_grads(q, k, v, dout, W, w, tau, lengths)
    if S == 1:   # the logits have no gradient: held to the size of what cancels in it
        size = float((dout.float().norm(dim=-1) * v.float().norm(dim=-1)).max())
        assert got[1].float().abs().max() <= BF16_TENSOR * size
        got, ref = (got[0], got[3]), (ref[0], ref[3])
        assert all(rel2(x, y) <= BF16_TENSOR for x, y in zip(got, ref))
        return
    check(got, ref, BF16_TENSOR)
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            assert (got[2][b, n:] == 0).all() and (got[3][b, n:] == 0).all()
            if n == 0:
                assert (got[0][b] == 0).all() and (got[1][b] == 0).all()


def test_gradients_of_long_sequences(sbl_lib):
    """One (batch, head) of the long configuration, against the kernels for any shape on the same inputs (which the
    tests above hold to the definition): the difference is at most the sum of both tolerances."""
    from fly_b200 import ops
    for d, N, w in ((64, 16384, 256), (128, 8192, 512)):
        q, k, v, dout, W = inputs(1, N, N, 1, d, d, 2 * d, torch.bfloat16)
        got = grads_of(q, k, v, dout, W, w)
        prob = ops.Problem(q, k, v, W, w, generic=True)
        ws = torch.empty(prob.workspace_bytes, dtype=torch.uint8, device='cuda')
        out, stats = prob.forward_train(ws)
        check(got, (out, *prob.backward(dout, stats)), BF16_TENSOR + BF16_ANY)


def test_single_key_has_no_gradient_in_the_logits(sbl_lib):
    """One key: its weight is 1 whatever the logit, so dq = dk = 0 up to roundings of dout.v, and dv = sum dout."""
    for dtype, tol in ((torch.float32, 64 * 2.0 ** -24), (torch.bfloat16, 4 * 2.0 ** -8)):
        q, k, v, dout, W = inputs(2, 5, 1, 2, 64, 64, 128, dtype)
        out, dq, dk, dv = grads_of(q, k, v, dout, W, 16)
        assert rel2(out, v.double().expand_as(out)) <= tol
        size = float((dout.float().norm(dim=-1) * v.float().norm(dim=-1)).max())
        assert dq.float().abs().max() <= tol * size and dk.float().abs().max() <= 5 * tol * size
        assert rel2(dv, dout.double().sum(1, keepdim=True)) <= tol


def test_gradients_against_differences(sbl_lib):
    """Directional differences of the definition in 64 bits: the error of a central difference at h = 1e-4 is about
    h^2 = 1e-8 of the third derivative, far under the fp32 tolerance."""
    q, k, v, dout, W = inputs(2, 90, 75, 2, 24, 20, 16, torch.float32, seed=3)
    lengths = torch.tensor([75, 40], device='cuda')
    grads = grads_of(q, k, v, dout, W, 20, None, lengths)[1:]
    g = torch.Generator(device='cuda').manual_seed(9)
    f = lambda a, b, c: float((sblocal_dense(a, b, c, W, 20, None, lengths) * dout.double()).sum())  # noqa: E731
    xs = [x.double() for x in (q, k, v)]
    for i in range(3):
        # along the gradient itself, so that the derivative is its norm and no digits cancel
        u = grads[i].double() / grads[i].double().norm()
        h = 1e-4
        up, down = list(xs), list(xs)
        up[i], down[i] = xs[i] + h * u, xs[i] - h * u
        slope = (f(*up) - f(*down)) / (2 * h)
        assert abs(slope - float(grads[i].double().norm())) <= 2 * FP32 * abs(slope)


def test_views_and_expanded_gradient(sbl_lib):
    """q, k, v out of one packed projection, and the gradient of out.sum(): an expanded scalar."""
    from fly_b200 import ops
    for E, r, dtype, tol in ((64, 128, torch.bfloat16, BF16_TENSOR), (20, 12, torch.float32, FP32)):
        g = torch.Generator(device='cuda').manual_seed(2)
        packed = (torch.randn(2, 150, 3 * 3 * E, generator=g, device='cuda') * E ** -0.25).to(dtype).requires_grad_()
        W = torch.randn(r, E, generator=g, device='cuda')
        q, k, v = packed.view(2, 150, 3, 3, E).unbind(2)
        out = ops.sblocal_attention(q, k, v, W, 40)
        scale = torch.randn(3, E, generator=g, device='cuda').to(dtype)
        got, = torch.autograd.grad((out * scale).sum(), packed)
        x = packed.detach().double().requires_grad_()
        ref = sblocal_dense(*x.view(2, 150, 3, 3, E).unbind(2), W, 40)
        want, = torch.autograd.grad((ref * scale.double()).sum(), x)
        assert rel2(got, want) <= tol
        expanded, = torch.autograd.grad(ops.sblocal_attention(q, k, v, W, 40).sum(), packed)
        want, = torch.autograd.grad(sblocal_dense(*x.view(2, 150, 3, 3, E).unbind(2), W, 40).sum(), x)
        assert rel2(expanded, want) <= tol


def test_forward_is_unchanged_under_autograd(sbl_lib):
    from fly_b200 import ops
    for E, D, r, dtype in ((64, 64, 128, torch.bfloat16), (128, 128, 256, torch.bfloat16), (21, 17, 13, torch.float32)):
        q, k, v, _, W = inputs(2, 200, 200, 2, E, D, r, dtype)
        plain = ops.sblocal_forward(q, k, v, W, 64)
        under = ops.sblocal_attention(q.requires_grad_(), k, v, W, 64)
        assert torch.equal(plain, under.detach())


def test_module_trains_with_lengths_and_norm(sbl_lib):
    """Norm and rotation, then the layer, as one program: gradients of the inputs and of the norm's weights."""
    from fly_b200 import LengthMask, QKNormRotary, SBLocalAttention
    from oracle.training_oracle import norm_rotary
    for dtype, tol in ((torch.float32, 2 * FP32), (torch.bfloat16, 12 ** 0.5 * 2.0 ** -8)):
        q, k, v, dout, W = inputs(2, 300, 300, 2, 64, 64, 128, dtype)
        layer = SBLocalAttention(64, 64, 256).cuda()
        layer.qk_norm = QKNormRotary(64, init=64 ** -0.25).cuda()
        layer.feature_map.new_feature_map('cuda')
        layer.feature_map.projection_matrix.copy_(W)
        xs = [x.requires_grad_() for x in (q, k, v)]
        lengths = torch.tensor([300, 171], device='cuda')
        out, _ = layer(*xs, key_padding_mask=LengthMask(lengths, max_len=300))
        out.backward(dout)
        ws = [layer.qk_norm.query_weight, layer.qk_norm.key_weight]
        ref = [x.detach().double().requires_grad_() for x in (*xs, *ws)]
        qn, kn = norm_rotary(ref[0], ref[3]), norm_rotary(ref[1], ref[4])
        want = torch.autograd.grad(sblocal_dense(qn, kn, ref[2], W, 64, None, lengths), ref, dout.double())
        for x, y in zip((*xs, *ws), want):
            assert rel2(x.grad, y) <= tol, rel2(x.grad, y)
        assert set(layer.state_dict()) == {'feature_map.projection_matrix', 'qk_norm.query_weight',
                                           'qk_norm.key_weight'}


@pytest.mark.parametrize('E,r,dtype', [(64, 128, torch.bfloat16), (32, 16, torch.float32)])
def test_streams_graphs_and_repeats(E, r, dtype, sbl_lib):
    """The same bits twice, on another stream, and in two captured graphs replayed on new inputs (torch captures no
    backward pass while an eager graph of the same leaves lives: the steps keep none)."""
    from fly_b200 import ops
    q, k, v, dout, W = inputs(2, 400, 400, 2, E, E, r, dtype)
    xs = [x.requires_grad_() for x in (q, k, v)]

    def step():
        out = ops.sblocal_attention(*xs, W, 100)
        grads = torch.autograd.grad(out, xs, dout)
        return (out.detach(), *grads)

    first = [x.detach().clone() for x in step()]
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(second):
        held2 = step()
    with torch.no_grad():
        q.copy_(q.flip(1))
    graph.replay()
    second.replay()
    torch.cuda.synchronize()
    fresh = step()
    assert all(torch.equal(a, b) for a, b in zip(held, fresh))
    assert all(torch.equal(a, b) for a, b in zip(held2, fresh))
    assert not torch.equal(held[0], first[0])


def test_outputs_have_guarded_borders(sbl_lib):
    """Gradients written into strided views leave what lies between their rows as it was."""
    import ctypes

    from fly_b200 import _cabi, ops
    for E, D, r, dtype in ((64, 64, 128, torch.bfloat16), (21, 17, 13, torch.float32)):
        q, k, v, dout, W = inputs(2, 150, 150, 2, E, D, r, dtype)
        prob = ops.Problem(q, k, v, W, 40)
        ws = torch.empty(prob.workspace_bytes, dtype=torch.uint8, device='cuda')
        out, stats = prob.forward_train(ws)
        want = prob.backward(dout, stats)
        full = [torch.full((2, 152, 3, x.shape[-1] + 8), 7.0, device='cuda', dtype=dtype) for x in want]
        views = [f[:, 1:151, :2, :x.shape[-1]] for f, x in zip(full, want)]
        g = _cabi.SblGrads()
        g.dout, g.do_stride_b, g.do_stride_t, g.do_stride_h = dout.data_ptr(), *dout.stride()[:3]
        g.row_stats = stats.data_ptr()
        g.dq, g.dq_stride_b, g.dq_stride_t, g.dq_stride_h = views[0].data_ptr(), *views[0].stride()[:3]
        g.dk, g.dk_stride_b, g.dk_stride_s, g.dk_stride_h = views[1].data_ptr(), *views[1].stride()[:3]
        g.dv, g.dv_stride_b, g.dv_stride_s, g.dv_stride_h = views[2].data_ptr(), *views[2].stride()[:3]
        n = prob.backward_workspace_bytes()
        # the workspace ends inside a larger buffer: the bytes behind it stay
        room = torch.full((n + 4096,), 85, dtype=torch.uint8, device='cuda')
        rc = sbl_lib.sbl_backward(ctypes.byref(prob.params), ctypes.byref(g), room.data_ptr(), n,
                                  torch.cuda.current_stream().cuda_stream)
        _cabi.check(rc)
        torch.cuda.synchronize()
        assert (room[n:] == 85).all()
        for f, view, x in zip(full, views, want):
            assert torch.equal(view, x)
            view.fill_(7.0)
            assert (f == 7.0).all()
