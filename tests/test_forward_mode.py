"""Forward-mode differentiation is refused: a result without its tangent would be wrong in silence.  The check comes
before the device is asked for, so it needs none."""
import pytest
import torch
from torch.autograd import forward_ad


def calls():
    from fly_b200 import QKNormRotary, SBLocalAttention, ops
    x, w = torch.randn(1, 5, 2, 8), torch.randn(8)
    W = torch.randn(4, 8)
    yield 'attention', lambda q, k, v: ops.sblocal_attention(q, k, v, W, 2), [x, x.clone(), x.clone()]
    yield 'norm', lambda q, k, a, b: ops.qk_norm_rotary(q, k, a, b), [x, x.clone(), w, w.clone()]
    norm = QKNormRotary(8)
    yield 'norm module', lambda q, k: norm(q, k), [x, x.clone()]
    layer = SBLocalAttention(2, 8, 8)
    yield 'layer', lambda q, k, v: layer(q, k, v)[0], [x, x.clone(), x.clone()]


@pytest.mark.parametrize('i', range(4))
def test_tangents_are_refused(i):
    _, f, args = list(calls())[i]
    for j in range(len(args)):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(x, torch.ones_like(x)) if n == j else x for n, x in enumerate(args)]
            with pytest.raises(NotImplementedError, match='forward-mode'):
                f(*dual)
            # no tangents among them: what a plain call gets, here that there is no device
            with pytest.raises(ValueError, match='CUDA'):
                f(*args)
        with pytest.raises(NotImplementedError, match='forward-mode'):
            torch.func.jvp(lambda x: f(*args[:j], x, *args[j + 1:]), (args[j],), (torch.ones_like(args[j]),))


@pytest.mark.gpu
def test_tangents_are_refused_on_the_device(sbl_lib):
    from fly_b200 import ops
    q, k, v = (torch.randn(1, 30, 2, 64, device='cuda') for _ in 'abc')
    W = torch.randn(32, 64, device='cuda')
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for grad in (False, True):
            k.requires_grad_(grad)
            with pytest.raises(NotImplementedError):
                ops.sblocal_attention(dual, k, v, W, 8)
            with pytest.raises(NotImplementedError):
                ops.qk_norm_rotary(dual, k)
            assert ops.sblocal_attention(q, k, v, W, 8).shape == q.shape
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda x: ops.qk_norm_rotary(x, k)[0], (q,), (torch.ones_like(q),))
