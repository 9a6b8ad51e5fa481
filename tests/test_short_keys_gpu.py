"""Output and gradients where query tiles of one key tile each follow one another: few keys, or short texts in a padded
batch.  Metric and tolerance as in test_training_gpu.py."""
import pytest
import torch

from oracle.training_oracle import rel2, sblocal_grads
from tests.test_training_gpu import BF16_TENSOR, check, grads_of, inputs

pytestmark = pytest.mark.gpu

# B, H, T, S, w, lengths (repeated over the batch)
CASES = [
    (21, 11, 177, 27, 214, None),
    (94, 2, 144, 74, 252, (56, 74, 34, 74, 57, 74)),
    (77, 2, 176, 16, 424, (6, 13, 16, 0, 16, 14)),
    (17, 14, 181, 15, 669, (2, 8, 0, 13, 5, 11)),
    (10, 18, 158, 17, 232, None),
    (32, 8, 512, 512, 128, (100, 90, 512, 128)),
    (64, 4, 700, 100, 2048, None),
    (40, 8, 400, 128, 500, (128, 128, 64)),
]


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c[:5])))
def test_few_keys(case, d, sbl_lib):
    from fly_b200 import ops
    B, H, T, S, w, lengths = case
    q, k, v, dout, W = inputs(B, T, S, H, d, d, 2 * d, torch.bfloat16, seed=3)
    if lengths:
        lengths = torch.tensor((lengths * B)[:B], device='cuda')
    ref = sblocal_grads(q, k, v, dout, W, w, None, lengths)
    first = ops.sblocal_forward(q, k, v, W, w, key_lengths=lengths)
    assert torch.isfinite(first).all() and rel2(first, ref[0]) <= BF16_TENSOR
    for _ in range(5):
        assert torch.equal(ops.sblocal_forward(q, k, v, W, w, key_lengths=lengths), first)
    got = grads_of(q, k, v, dout, W, w, None, lengths)
    assert torch.equal(got[0], first)
    check(got, ref, BF16_TENSOR)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(got, grads_of(q, k, v, dout, W, w, None, lengths)))
    ops.status_watch.poll(wait=True)
