"""Gradients on the tensor cores where a CTA gets tiles of few steps, or none, one after the other: few queries with more
keys, and batches whose lengths leave tiles empty.  Metric and tolerance as in test_training_gpu.py."""
import pytest
import torch

from oracle.training_oracle import sblocal_grads
from tests.test_training_gpu import BF16_TENSOR, check, grads_of, inputs

pytestmark = pytest.mark.gpu

# B, H, T, S, w, lengths (repeated over the batch)
CASES = [
    (200, 1, 128, 384, 64, None),                    # one-step tiles and tiles that nobody sees
    (64, 8, 64, 1000, 128, (700, 333, 128, 1000, 90)),
    (64, 1, 1, 1024, 256, None),
    (64, 12, 100, 100, 64, (100, 0, 0, 57)),         # batches without keys
    (200, 1, 256, 256, 1, (256, 100, 0)),
    (8, 40, 128, 128, 64, (128, 128, 0)),
    (16, 16, 100, 300, 256, (300, 150, 110, 300)),
]


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c[:5])))
def test_short_and_empty_tiles(case, d, sbl_lib):
    B, H, T, S, w, lengths = case
    q, k, v, dout, W = inputs(B, T, S, H, d, d, 2 * d, torch.bfloat16, seed=11)
    if lengths:
        lengths = torch.tensor((lengths * B)[:B], device='cuda')
    got = grads_of(q, k, v, dout, W, w, None, lengths)
    check(got, sblocal_grads(q, k, v, dout, W, w, None, lengths), BF16_TENSOR)
    # the same bits again: nothing depends on who was first
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, grads_of(q, k, v, dout, W, w, None, lengths)))
