"""Token log probabilities and their gradient where a row's numbers leave the ordinary range: NaN and infinities without an entropy
gradient, logits on both sides of the magnitude from which distances are taken from the maximum itself, sums under a far larger maximum."""
import math

import pytest
import torch

from nectarml_b200 import _lib, ops, train

from test_gpu_token_log_probs import DEV, DTYPES, U, chain, check_backward, check_forward, logits, plain, tokens

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


@pytest.mark.parametrize("vocab", [5, 777, 3000, 70001])
@pytest.mark.parametrize("around", [1e7, -1e7])
def test_logits_on_both_sides_of_far(around, vocab):
    """Maxima of 1e7 and more (or of -1e7 and less) are references of their own, smaller ones are rounded products: both in one row, as in one
    that a mask of -1e7 covers as a whole.  The gradient is good to what test_large_offsets derives."""
    x = around + logits((40, vocab), torch.float32, 23, spread=2.5) - (3.0 if around < 0 else -3.0) * torch.arange(
        -2, 3, device=DEV).repeat(8)[:, None]
    assert bool(((x.abs() >= 1e7).any(1) & (x.abs() < 1e7).any(1)).any())
    t = tokens((40,), vocab)
    r = check_forward(x, t, min(3, vocab))
    d, dh = logits((40,), torch.float32, 24), logits((40,), torch.float32, 25)
    lp, _, h, _ = plain(x, t)
    p = lp.exp()
    want = -d[:, None] * p * (t >= 0)[:, None] - dh[:, None] * p * torch.where(p > 0, lp + h[:, None], 0.0)
    want[torch.arange(40, device=DEV), t.clamp(min=0)] += torch.where(t >= 0, d, 0.0)
    got = ops.token_log_probs_backward(x, t, r.stats, r.entropy, d, dh).double()
    size = (d.abs().max() + dh.abs().max() * 16).item()
    assert bool(((got - want).abs() <= 2 * size * (8 + chain(vocab, torch.float32)) * U).all())


@pytest.mark.parametrize("vocab", [777, 70001])
def test_half_precision_logits_on_both_sides_of_far(vocab):
    """The same at fp16's lowest values, where maxima below -65000 are references of their own."""
    g = torch.Generator(device=DEV).manual_seed(26)
    x = (-65008 + 32 * torch.randint(-2, 3, (40, vocab), device=DEV, generator=g)).half()
    assert bool((x < -65000).any()) and bool((x >= -65000).any()) and bool(x.isfinite().all())
    t = tokens((40,), vocab)
    check_forward(x, t, 3)
    # every unit on one side: the maxima meet where lanes are merged
    y = torch.full((4, vocab), -65024.0, device=DEV).half()
    y[:, : vocab // 2] = -64992.0
    y[2:] = y[2:].flip(1)
    check_forward(y, t[:4].contiguous(), 3)
    check_backward(y, t[:4].contiguous(), False)


def test_large_sums_below_a_far_larger_maximum():
    """A thread's sums reach 5e8 before the largest logit comes; what is left of them is 0, not 0 times what times 1e30 is no finite number."""
    vocab = 400_000_000
    x = torch.full((1, vocab), 7.9, device=DEV)
    x.view(8, -1)[:, :8192] = 0.0         # (sums against 0: e^7.9 a logit)
    x[0, -1] = 3e38
    t = torch.tensor([vocab - 1], device=DEV)
    r = ops.token_log_probs(x, t)
    ops.device_status()
    assert float(r.log_probs) == 0.0 and float(r.entropy) == 0.0 and r.stats[0].tolist() == [x[0, -1].item(), 0.0]


@DTYPES
def test_training_loss_leaves_padding_out(dtype):
    """Rows with a negative label count neither in the loss, the entropy's part included, nor in the gradient."""
    x, t = logits((12, 300), dtype, 27), tokens((12,), 300)
    kept = t >= 0
    assert 0 < int(kept.sum()) < 12
    step = train.TrainStep(None, "token_log_probs", entropy_weight=0.5)
    value, grads = [], []
    for rows in (torch.ones_like(kept), kept):
        y = x[rows].clone().requires_grad_(True)
        value.append(step._loss(y, t[rows], 8))
        value[-1].backward()
        grads.append(y.grad)
    # (sums of the same numbers, among which the one has zeros, in whatever order: 12 roundings of a sum of 9 logs and entropies below 6 each)
    assert abs(float(value[0].detach().double() - value[1].detach().double())) <= 24 * U * 9 * (10 + 0.5 * 6) / 8
    assert not grads[0][~kept].any() and bool(grads[0][kept].any())
    # (the same rows, but 300 logits are no whole number of 32-byte units, so without the padded ones they start elsewhere in them and are summed in another
    # order: either side is good to what test_large_offsets derives, and rounded to its type)
    size, c = (1 + 0.5 * 16) / 8, chain(300, dtype)
    tol = 2 * 2 * size * (8 + c) * U + (2 * 2.0 ** -11 * grads[1].double().abs() + 2.0 ** -24 if dtype == torch.float16 else 0.0)
    assert bool(((grads[0][kept].double() - grads[1].double()).abs() <= tol).all())


def test_training_step_with_padding():
    """Of labels that are all padding nothing is learned, with an entropy term too; of some, as much as torch's loss and entropy over the others give."""
    n, classes = 8, 24
    x = torch.randn(n, 64, 64, 3, device=DEV).half()
    labels = torch.randint(0, classes, (n,), device=DEV)
    for padded in (range(n), (1, 4, 5)):
        t = labels.clone()
        t[list(padded)] = -1
        kept = t >= 0
        net = train.ResNet50(DEV, num_classes=classes, blocks=(1, 1, 1, 1), width=16)
        net.init(seed=3)
        step = train.TrainStep(net, "token_log_probs", loss_scale=8192.0, entropy_weight=0.3)
        value = float(step([(x, t)], global_count=n, optimize=False))
        ops.device_status()
        if not bool(kept.any()):
            assert value == 0 and not net.store.grad.any()
            continue
        with torch.no_grad():
            lp = net.forward(x).double().log_softmax(1)
        h = -(lp * lp.exp()).sum(1)
        want = -float((lp[kept, t[kept]] + 0.3 * h[kept]).sum()) / n
        assert abs(value - want) <= 1e-5 * abs(want) and bool(net.store.grad.any())


@DTYPES
def test_gradient_beside_the_logits(dtype):
    """Between the logits' rows, in the columns beside them, in place in a view; and refused where it would lie over other elements."""
    x = logits((6, 501), dtype, 28)
    t = tokens((6,), 501)
    room = torch.empty(12, 501, dtype=dtype, device=DEV)
    room[0::2] = x
    check_backward(room[0::2], t, True, out=room[1::2])
    assert torch.equal(room[0::2], x)
    wide = torch.empty(6, 1010, dtype=dtype, device=DEV)
    wide[:, :501] = x
    check_backward(wide[:, :501], t, True, out=wide[:, 501:1002])
    assert torch.equal(wide[:, :501], x)
    r = ops.token_log_probs(x, t)
    ones = torch.ones(6, device=DEV)
    for a, b in ((wide[:, :501], wide[:, 500:1001]), (wide[:, 1:502], wide[:, :501]), (wide[:5, :501], wide[1:, :501])):
        n = a.shape[0]
        with pytest.raises(_lib.NectarB200Error, match="status 1"):
            ops.token_log_probs_backward(a, t[:n], r.stats[:n], None, ones[:n], out=b)
    one = wide[:1, 3:504]
    one.copy_(x[:1])
    first = ops.token_log_probs(one, t[:1])
    got = ops.token_log_probs_backward(one, t[:1], first.stats, None, ones[:1], out=wide.view(-1)[3:504].view(1, 501))   # one row, in place, another pitch
    assert got.data_ptr() == one.data_ptr() and bool(got.isfinite().all())
