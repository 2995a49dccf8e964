"""Token log probabilities and their gradient where a row's numbers leave the ordinary range."""
import math

import pytest
import torch

from nectarml_b200 import ops, train

from test_gpu_token_log_probs import DEV, DTYPES, logits

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("vocab", [1, 5, 40, 1500, 70001])
def test_gradient_of_rows_with_nan_or_infinity(vocab, entropy, dtype):
    """NaN in every element of such a row, as softmax has it, and in no other; so that a check for finite gradients sees it."""
    x = logits((5, vocab), dtype, 21)
    x[0, vocab // 2] = math.nan
    x[1, vocab // 3] = math.inf
    x[2] = math.nan
    x[3, vocab - 1] = -math.inf if vocab > 1 else 1.0
    t = torch.zeros(5, dtype=torch.int64, device=DEV)
    r = ops.token_log_probs(x, t)
    ones = torch.ones(5, device=DEV)
    d = ops.token_log_probs_backward(x, t, r.stats, r.entropy, ones, ones if entropy else None)
    ops.device_status()
    assert bool(d[:3].isnan().all()) and bool(d[3:].isfinite().all())
    into = x.clone()
    assert ops.token_log_probs_backward(into, t, r.stats, r.entropy, ones, ones if entropy else None, out=into)[:3].isnan().all()


def test_gradient_of_rows_with_nan_through_autograd():
    x = logits((3, 300), torch.float32, 22)
    x[1, 7] = math.nan
    x.requires_grad_(True)
    train.token_log_probs(x, torch.tensor([1, 2, 3], device=DEV)).log_probs.sum().backward()
    assert bool(x.grad[1].isnan().all()) and bool(x.grad[0::2].isfinite().all())
