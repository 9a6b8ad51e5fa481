"""Definitions, in 64 bits, of what is trained: SBLocal attention written out over all (query, key) pairs, and the
norm and rotation of heads.  Gradients come from torch autograd over these definitions, so they share nothing with
the kernels' formulas.  Test infrastructure only."""
import math

import torch


def sblocal_dense(q, k, v, W, w, tau=None, lengths=None):
    """out (B,T,H,D) of q (B,T,H,E), k (B,S,H,E), v (B,S,H,D), in float64: a key inside the window of a row weighs
    exp(tau q.k), any other real key phi(q).phi(k); rows are divided by the sum of their weights.  Rows without a
    real key give zero."""
    q, k, v = (x.double().transpose(1, 2) for x in (q, k, v))
    W = W.double()
    tau = tau or q.shape[-1] ** -0.5
    T, S = q.shape[2], k.shape[2]

    def features(x):
        u = math.sqrt(tau) * (x @ W.T)
        return torch.exp(torch.cat([u, -u], -1) - tau * (x * x).sum(-1, keepdim=True) / 2
                         - math.log(2 * W.shape[0]) / 2)

    i, s = torch.arange(T, device=q.device)[:, None], torch.arange(S, device=q.device)
    near = (s >= i - w // 2) & (s < i - w // 2 + w)
    real = torch.ones(q.shape[0], S, dtype=torch.bool, device=q.device)
    if lengths is not None:
        real = s < lengths[:, None]
    weight = torch.where(near, torch.exp(tau * (q @ k.transpose(2, 3))), features(q) @ features(k).transpose(2, 3))
    weight = weight * real[:, None, None]
    total = weight.sum(-1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    return ((weight / total) @ v).transpose(1, 2)


def sblocal_grads(q, k, v, dout, W, w, tau=None, lengths=None):
    """(out, dq, dk, dv) in float64."""
    xs = [x.detach().double().requires_grad_() for x in (q, k, v)]
    out = sblocal_dense(*xs, W, w, tau, lengths)
    return (out.detach(), *torch.autograd.grad(out, xs, dout.double()))


def norm_rotary(x, weight=None, positions=None, pos0=0, rotary=None, theta=10000.0, interleaved=False, eps=1e-6):
    """(B,T,H,E) -> float64: each head row over its root mean square, times `weight`, its pairs turned."""
    x = x.double()
    E, T = x.shape[-1], x.shape[1]
    z = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        z = z * weight.double()
    rotary = E if rotary is None else rotary
    if positions is None:
        positions = pos0 + torch.arange(T, device=x.device)
    angle = positions.double()[..., None, None] * theta ** (
        -torch.arange(0, rotary, 2, device=x.device, dtype=torch.float64) / max(rotary, 1))
    c, s = torch.cos(angle), torch.sin(angle)
    half = rotary // 2
    if interleaved:
        a, b = z[..., 0:rotary:2], z[..., 1:rotary:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = z[..., :half], z[..., half:rotary]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, z[..., rotary:]], -1)


def rel2(x, ref):
    """|x - ref| / |ref| in the 2-norm."""
    return float((x.double() - ref).norm() / ref.norm())
