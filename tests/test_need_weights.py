"""Gradients through `need_weights` are refused by the backward pass, not left out in silence."""
import pytest
import torch


class _Stub:
    """A problem without a device: an output and weights of the right shapes."""

    def __init__(self, query, key, value, *args, generic):
        assert generic
        self.out = torch.ones(*query.shape[:3], value.shape[3])
        self.weights = torch.ones(query.shape[0], query.shape[2], query.shape[1], key.shape[1])

    def workspace(self):
        return None

    def forward(self, workspace=None):
        return self.out

    def attention_weights(self, unnormalized=False, workspace=None):
        return (self.weights, self.weights + 1, self.weights + 2) if unnormalized else self.weights


def check(layer, q, k, v):
    for unnormalized in (False, True):
        out, attn = layer(q, k, v, need_weights=True, return_attn_unnormalized=unnormalized)
        assert isinstance(attn, tuple) == unnormalized
        for x in (out, *(attn if unnormalized else (attn,))):
            # beside another term that can be differentiated
            with pytest.raises(NotImplementedError, match='need_weights'):
                (x.sum() + q.sum() + k.sum() + v.sum()).backward()
        with torch.no_grad():
            out, attn = layer(q, k, v, need_weights=True)
        assert not out.requires_grad and not attn.requires_grad


def test_backward_through_weights_raises(monkeypatch):
    from fly_b200 import SBLocalAttention, ops
    monkeypatch.setattr(ops, 'Problem', _Stub)
    q, k, v = torch.randn(2, 5, 2, 8), torch.randn(2, 6, 2, 8), torch.randn(2, 6, 2, 4)
    for i in range(3):
        xs = [x.clone().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
        layer = SBLocalAttention(4, 8, 8)
        if i == 0:
            # only the norm in front of the layer learns
            layer.qk_norm = lambda a, b: (a * torch.ones(8, requires_grad=True), b)
            xs = [q.clone().requires_grad_(), k, v]
        check(layer, *xs)


@pytest.mark.gpu
def test_backward_through_weights_raises_on_the_device(sbl_lib):
    from fly_b200 import QKNormRotary, SBLocalAttention
    q, k, v = (torch.randn(2, 70, 2, 64, device='cuda') for _ in 'abc')
    layer = SBLocalAttention(16, 64, 64).cuda()
    layer.qk_norm = QKNormRotary(64).cuda()
    check(layer, q.requires_grad_(), k, v)
    out, attn = layer(q, k, v, need_weights=True)
    again, none = layer(q, k, v)
    # (fp32: the same kernels)
    assert none is None and torch.equal(out, again) and attn.shape == (2, 2, 70, 70)
