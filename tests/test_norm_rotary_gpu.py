"""Norm and rotation of query and key heads (`ops.qk_norm_rotary`, `QKNormRotary`) against the definition in 64 bits.

Tolerances, relative to the largest value of a row's definition:
  bf16 results are one rounding of an fp32 value: half a step, 2^-8, plus the fp32 error;
  fp32: the sum over E <= 512 entries in partial sums of at most 16 terms and 5 shuffle steps, a reciprocal root, an
    angle reduced in fp64 and rounded once, and five products: under 32 roundings of 2^-24 = 2e-6;
  weight gradients: sums over R rows in fp32.  Partial sums of at most 32 rows per lane and a tree behind them: 48
    roundings of 2^-24 of the sum of magnitudes, which is the scale they are compared on.
"""
import pytest
import torch

from oracle.training_oracle import norm_rotary

pytestmark = pytest.mark.gpu

FP32 = 2e-6
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def make(B, T, S, Hq, Hk, E, dtype, wdtype=torch.float32, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    q, k = n(B, T, Hq, E).to(dtype), n(B, S, Hk, E).to(dtype)
    wq, wk = (1 + 0.2 * n(E)).to(wdtype), (1 + 0.2 * n(E)).to(wdtype)
    return q, k, wq, wk, n(B, T, Hq, E).to(dtype), n(B, S, Hk, E).to(dtype)


def check_side(y, dx, dw, x, w, dy, tol_extra=0.0, **kw):
    xd = x.detach().double().requires_grad_()
    wd = None if w is None else w.detach().double().requires_grad_()
    ref = norm_rotary(xd, wd, **kw)
    leaves = [xd] + ([wd] if wd is not None else [])
    grads = torch.autograd.grad(ref, leaves, dy.double())
    step = HALF_STEP[x.dtype]

    def close(got, want, extra=0.0):
        scale = want.abs().amax(-1, keepdim=True).clamp_min(1e-30)
        assert torch.isfinite(got).all()
        err = ((got.double() - want).abs() / scale).max()
        assert err <= step + FP32 + extra, f'{float(err):.3e}'

    close(y, ref.detach(), tol_extra)
    # a row's gradient is a difference of two vectors of the size of dy * w / rms
    rms = x.double().square().mean(-1, keepdim=True).add(1e-6).sqrt()
    size = (dy.double().abs().amax(-1, keepdim=True) * 2 / rms)
    err = ((dx.double() - grads[0]).abs() / torch.maximum(size, grads[0].abs())).max()
    assert err <= step + FP32 + tol_extra, f'{float(err):.3e}'
    if w is not None:
        unit = x.double() / rms
        size = (dy.double().abs().amax(-1, keepdim=True) * 2 * unit.abs()).sum((0, 1, 2))
        err = ((dw.double() - grads[1]).abs() / size).max()
        assert err <= HALF_STEP[w.dtype] + 48 * 2.0 ** -24 + tol_extra, f'{float(err):.3e}'


CASES = [
    # B, T, S, Hq, Hk, E, rotary, dtype
    (2, 5, 5, 4, 4, 64, 64, torch.bfloat16),
    (1, 1, 1, 1, 1, 64, 64, torch.bfloat16),        # one token
    (8, 1, 1, 16, 2, 128, 128, torch.bfloat16),     # decode, shared key heads
    (2, 33, 17, 3, 5, 128, 64, torch.float32),      # lengths and heads differ, part of the head turned
    (3, 129, 129, 7, 1, 96, 32, torch.bfloat16),    # 12 of 16 lanes hold a row
    (2, 31, 31, 5, 2, 256, 256, torch.float32),
    (2, 31, 31, 5, 2, 32, 0, torch.float32),        # nothing turned
    (1, 700, 700, 2, 2, 8, 8, torch.bfloat16),
    (2, 31, 31, 3, 3, 24, 24, torch.bfloat16),      # halves of 12: entry by entry
    (2, 19, 23, 3, 2, 21, 14, torch.float32),       # odd head dim
    (1, 9, 9, 2, 2, 1, 0, torch.float32),
    (2, 7, 7, 3, 3, 510, 510, torch.bfloat16),
    (1, 4100, 4100, 16, 16, 64, 64, torch.bfloat16),  # more tokens than warps
]


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(str(x) for x in c[:7]) + str(c[7])[6:])
def test_values_and_gradients(case, interleaved, sbl_lib):
    from fly_b200 import ops
    B, T, S, Hq, Hk, E, rotary, dtype = case
    q, k, wq, wk, dq, dk = make(B, T, S, Hq, Hk, E, dtype)
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    y = ops.qk_norm_rotary(q, k, wq, wk, pos0=3, rotary_dim=rotary, interleaved=interleaved, theta=500.0)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    kw = dict(pos0=3, rotary=rotary, interleaved=interleaved, theta=500.0)
    check_side(y[0], grads[0], grads[2], q, wq, dq, **kw)
    check_side(y[1], grads[1], grads[3], k, wk, dk, **kw)
    with torch.no_grad():
        z = ops.qk_norm_rotary(q, k, wq, wk, pos0=3, rotary_dim=rotary, interleaved=interleaved, theta=500.0)
    assert torch.equal(z[0], y[0]) and torch.equal(z[1], y[1])


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('E', [64, 20])
def test_far_negative_and_repeated_positions(E, interleaved, sbl_lib):
    """Angles of positions up to 2^40: the fp64 product is off by 2^-53 of it, 2^-13 turns at the fastest pair."""
    from fly_b200 import ops
    q, k, wq, wk, dq, dk = make(3, 11, 11, 4, 2, E, torch.float32)
    pos = torch.randint(-(1 << 24), 1 << 24, (3, 11), device='cuda')
    pos[0, :4] = pos[0, 0]
    for p, extra in ((pos, 1e-8 * 2 ** 1), (pos + (1 << 40), 2 * 3.2 * 2.0 ** (40 - 53))):
        leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]
        y = ops.qk_norm_rotary(*leaves, positions=p, interleaved=interleaved)
        g = torch.autograd.grad(y, leaves, (dq, dk))
        check_side(y[0], g[0], g[2], q, wq, dq, extra, positions=p, interleaved=interleaved)
        check_side(y[1], g[1], g[3], k, wk, dk, extra, positions=p, interleaved=interleaved)
    # (T,) positions are shared by the batch; the keys' may differ from the queries'
    a = ops.qk_norm_rotary(q, k, wq, wk, positions=pos[1], key_positions=pos, interleaved=interleaved)
    b = ops.qk_norm_rotary(q, k, wq, wk, positions=pos[1].expand(3, 11), key_positions=pos, interleaved=interleaved)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize('wdtype', [torch.float32, torch.bfloat16, None])
def test_views_weights_and_broadcast(wdtype, sbl_lib):
    """Heads out of a packed projection, an expanded output gradient, weights of either type or none."""
    from fly_b200 import ops
    g = torch.Generator(device='cuda').manual_seed(5)
    for H, E in ((4, 64), (3, 20)):
        packed = torch.randn(2, 37, 3 * H * E, generator=g, device='cuda').bfloat16()
        q, k, _ = packed.view(2, 37, 3, H, E).unbind(2)
        assert not q.is_contiguous()
        wq = wk = None
        if wdtype is not None:
            wq, wk = ((1 + 0.2 * torch.randn(E, generator=g, device='cuda')).to(wdtype).requires_grad_() for _ in 'ab')
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        y = ops.qk_norm_rotary(q, k, wq, wk)
        dy = torch.randn(1, 1, 1, E, generator=g, device='cuda').bfloat16().expand(2, 37, H, E)
        leaves = [x for x in (q, k, wq, wk) if x is not None]
        grads = torch.autograd.grad(y, leaves, (dy, dy)) + (None, None)
        check_side(y[0], grads[0], grads[2], q, wq, dy)
        check_side(y[1], grads[1], grads[3], k, wk, dy)
        # a row stride that is no multiple of 16 bytes
        odd = torch.randn(2, 9, H, E + 1, generator=g, device='cuda').bfloat16()[..., 1:]
        a = ops.qk_norm_rotary(odd, odd, wq, wk)
        b = ops.qk_norm_rotary(odd.contiguous(), odd.contiguous(), wq, wk)
        assert (a[0].float() - b[0].float()).abs().max() <= 2 * 2.0 ** -8 * b[0].float().abs().max()


def test_zero_rows_and_no_rows(sbl_lib):
    from fly_b200 import ops
    q, k, wq, wk, dq, dk = make(2, 6, 6, 2, 2, 64, torch.bfloat16)
    q[1, 2] = 0
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    y = ops.qk_norm_rotary(q, k, wq, wk)
    g = torch.autograd.grad(y, leaves, (dq, dk))
    assert (y[0][1, 2] == 0).all() and all(torch.isfinite(x).all() for x in g)
    check_side(y[0], g[0], g[2], q, wq, dq)
    for shape in ((0, 5), (2, 0)):
        e = torch.empty(*shape, 2, 64, device='cuda', dtype=torch.bfloat16, requires_grad=True)
        y = ops.qk_norm_rotary(e, e, wq, wk)
        g = torch.autograd.grad(y, (e, wq, wk), y)
        assert y[0].shape == e.shape and (g[1] == 0).all() and (g[2] == 0).all()
    # keys without rows beside queries with some
    e = torch.empty(2, 0, 3, 64, device='cuda', dtype=torch.bfloat16)
    assert torch.equal(ops.qk_norm_rotary(q, e, wq, wk)[0], ops.qk_norm_rotary(q, k, wq, wk)[0])


def test_streams_graphs_and_repeats(sbl_lib):
    """The same bits on another stream, in a replayed graph that sees new inputs, and twice in a row."""
    from fly_b200 import ops
    q, k, wq, wk, dq, dk = make(2, 513, 513, 8, 8, 64, torch.bfloat16)
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]

    def step():
        y = ops.qk_norm_rotary(q, k, wq, wk)
        grads = torch.autograd.grad(y, leaves, (dq, dk))
        # no eager graph of the leaves may be alive when torch captures a backward pass of theirs
        return (*(x.detach() for x in y), *grads)

    first = [x.clone() for x in step()]
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        q.copy_(q.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))
    assert not torch.equal(held[0], first[0])
