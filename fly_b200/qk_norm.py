"""Learned root-mean-square norm of query and key heads with the rotation by position, as a layer in front of an
attention layer.

The bf16 attention kernels are accurate for logits of about unit scale (they never rescale an accumulator and their
low-rank estimate loses digits as norms grow): a norm in front bounds every query and key by its weight, whatever the
projections in front of it learn.  `init = dim_heads ** -0.25` gives heads with tau |q|^2 = 1 at the default
temperature, the scale the kernels are measured at; 1 is the usual start of such a norm.
No counterpart in the reference.
"""
import torch
import torch.nn as nn

from . import ops


class QKNormRotary(nn.Module):
    """forward(query (B,T,Hq,E), key (B,S,Hk,E), positions=None, key_positions=None) -> (query, key); see
    `ops.qk_norm_rotary` for the arguments.  rotary_dim=0: the norm alone."""

    def __init__(self, dim_heads, rotary_dim=None, theta=10000.0, interleaved=False, eps=1e-6, init=1.0, device=None,
                 dtype=None):
        super().__init__()
        rotary_dim = dim_heads - dim_heads % 2 if rotary_dim is None else rotary_dim
        if rotary_dim < 0 or rotary_dim > dim_heads or rotary_dim % 2:
            raise ValueError(f'rotary_dim must be even and in 0..{dim_heads}, got {rotary_dim}')
        self.rotary_dim, self.theta, self.interleaved, self.eps = rotary_dim, theta, interleaved, eps
        self.query_weight = nn.Parameter(torch.full((dim_heads,), float(init), device=device, dtype=dtype))
        self.key_weight = nn.Parameter(torch.full((dim_heads,), float(init), device=device, dtype=dtype))

    def forward(self, query, key, positions=None, key_positions=None):
        return ops.qk_norm_rotary(query, key, self.query_weight, self.key_weight, positions, key_positions,
                                  rotary_dim=self.rotary_dim, theta=self.theta, interleaved=self.interleaved,
                                  eps=self.eps)

    def extra_repr(self):
        return (f'{self.query_weight.numel()}, rotary_dim={self.rotary_dim}, theta={self.theta}, '
                f'interleaved={self.interleaved}, eps={self.eps}')
