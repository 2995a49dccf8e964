"""Token log probabilities, entropy, alternatives and their gradient against a plain form in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32): a term e^d costs 2 u for the exponential and 2 |d| u for its argument, and |d| e^d <= 1/e,
so a term is good to 4 u of the largest; sums of one sign add u for each term behind one another (`chain`: a thread's share, then
16 for the merges); the statistics are rescaled at most once a term, another 4 u each in the worst case, which `chain` is widened
by.  Hence log s is off by at most (8 + chain) u + u log s, and the entropy log s - t / s by that and (|t| / s) (16 + 2 chain) u."""
import math

import pytest
import torch

from nectarml_b200 import ops, train

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def plain(x, targets, top=0):
    x = x.double()
    vocab = x.shape[-1]
    m = x.amax(-1, keepdim=True)
    dead = (m == -math.inf)
    d = torch.where(dead, -math.inf, x - m)
    e = d.exp()
    s = torch.where(dead, 1.0, e.sum(-1, keepdim=True))
    lp = d - s.log()
    h = (s.log() - torch.where(e == 0, 0.0, d * e).sum(-1, keepdim=True) / s)[..., 0]
    token = lp.gather(-1, targets.clamp(0, vocab - 1)[..., None])[..., 0]
    token = torch.where(targets < 0, 0.0, torch.where(targets >= vocab, math.nan, token))
    if not top:
        return lp, token, h, None
    order = x.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    return lp, token, h, order


def chain(vocab, dtype):
    per = 16 if dtype == torch.float16 else 8
    units = -(-vocab // per) + 1
    threads = 32 if units <= 128 else 128
    return 5 * per * -(-units // threads) + 16


def check_forward(x, targets, top):
    r = ops.token_log_probs(x, targets, top=top)
    ops.device_status()
    lp, token, h, order = plain(x, targets, top)
    c = chain(x.shape[-1], x.dtype)
    m = x.double().amax(-1)
    live = torch.isfinite(m)
    log_s = torch.where(live, lp.amax(-1).abs(), 0.0)
    tol = (8 + c) * U + 2 * U * log_s + 2 * U * torch.where(torch.isfinite(token), token.abs(), 0.0)
    same = torch.isfinite(token)
    assert torch.equal(same, torch.isfinite(r.log_probs)) and torch.equal(torch.isnan(token), torch.isnan(r.log_probs))
    assert bool(((r.log_probs.double() - token).abs() <= tol)[same].all())
    fine = torch.isfinite(h)
    assert torch.equal(fine, torch.isfinite(r.entropy))
    assert bool(((r.entropy.double() - h).abs() <= (8 + c) * U + 4 * U * log_s + h * (16 + 2 * c) * U)[fine].all())
    if top:
        assert torch.equal(r.top_indices, order)
        want = lp.gather(-1, order)
        assert torch.equal(torch.isfinite(want), torch.isfinite(r.top_log_probs))
        ok = torch.isfinite(want)
        assert bool(((r.top_log_probs.double() - want).abs() <= ((8 + c) * U + 2 * U * log_s)[..., None] + 2 * U * want.abs())[ok].all())
    else:
        assert r.top_indices is None and r.top_log_probs is None
    return r


def logits(shape, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(shape, device=DEV, generator=g)).to(dtype)


def tokens(shape, vocab, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000)
    t = torch.randint(0, vocab, shape, device=DEV, generator=g)
    t.view(-1)[1::5] = -100
    return t


DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])


@DTYPES
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 1, 0), (3, 2, 2), (5, 7, 7), (2, 16, 3), (4, 17, 17), (7, 31, 31), (3, 33, 32), (9, 255, 5), (300, 1000, 5), (5, 2047, 32), (4, 2049, 1),
    (6, 16383, 20), (6, 16385, 8), (1, 50021, 0), (40, 50021, 32), (1, 131072, 20), (150, 33001, 4)])
def test_sizes(rows, vocab, top, dtype):
    check_forward(logits((rows, vocab), dtype, vocab), tokens((rows,), vocab), top)


@pytest.mark.parametrize("offset", [1e3, 1e6, 9e6, 1.1e7, 1e8, 1e10, 1e15, 1e20, 1e29, 1e31, 1e38])
def test_large_offsets(offset):
    """Only distances count, however far the logits lie from 0: the gradient too."""
    g = torch.Generator(device=DEV).manual_seed(3)
    for sign in (1, -1):
        x = sign * offset * (1 + 1e-3 * torch.rand(40, 1, device=DEV, generator=g)) + logits((40, 777), torch.float32, 4)
        x[3, 5:] = -math.inf
        x[4, 5:] = torch.finfo(torch.float32).min
        t = tokens((40,), 777)
        t[3:5] = 2
        r = check_forward(x, t, 3)
        d, dh = logits((40,), torch.float32, 5), logits((40,), torch.float32, 6)
        lp, _, h, _ = plain(x, t)
        p = lp.exp()
        want = -d[:, None] * p * (t >= 0)[:, None] - dh[:, None] * p * torch.where(p > 0, lp + h[:, None], 0.0)
        want[torch.arange(40, device=DEV), t.clamp(min=0)] += torch.where(t >= 0, d, 0.0)
        got = ops.token_log_probs_backward(x, t, r.stats, r.entropy, d, dh).double()
        # y = log2 p is good to 2 u of x log2 e - M, whose size is that of M's rounding (up to 1 where it is not 0) and of y, and as log s is
        size = (d.abs().max() + dh.abs().max() * 16).item()
        assert bool(((got - want).abs() <= 2 * size * (8 + chain(777, torch.float32)) * U).all())


@DTYPES
@pytest.mark.parametrize("step", [0.01, 0.5, 7.9, 8.1, 60.0])
def test_rising_logits(step, dtype):
    """Every unit has a new maximum: the sums move seldom, always or by nearly as much as leaves them where they are."""
    v = torch.arange(2000, device=DEV, dtype=torch.float64) * step
    x = (v - v[-1] / 2).clamp(-60000, 60000).to(dtype)
    check_forward(torch.stack([x, x.flip(0), x.roll(1000)]), torch.tensor([1999, 1, 1000], device=DEV), 4)


@DTYPES
def test_ties(dtype):
    """Few values, many of each: alternatives by index, however many units share their maximum."""
    g = torch.Generator(device=DEV).manual_seed(8)
    for vocab in (1000, 2000, 5000, 40000):
        for values, top in ((1, 32), (3, 32), (40, 7), (40, 1)):
            x = torch.randint(0, values, (70, vocab), device=DEV, generator=g).to(dtype)
            got = ops.token_log_probs(x, tokens((70,), vocab), top=top).top_indices
            assert torch.equal(got, x.float().sort(dim=-1, descending=True, stable=True).indices[:, :top]), (vocab, values)


@DTYPES
def test_more_rows_than_blocks(dtype):
    check_forward(logits((10000, 257), dtype, 1), tokens((10000,), 257), 3)
    check_forward(logits((5000, 5001), dtype, 2), tokens((5000,), 5001), 2)


@DTYPES
def test_long_rows_of_few_blocks(dtype):
    """The longest vocabulary with alternatives, and one beyond it without."""
    longest = 2_000_000 if dtype == torch.float16 else 1_000_000
    check_forward(logits((2, longest), dtype, 3), tokens((2,), longest), 32)
    check_forward(logits((3, 2_200_003), dtype, 4), tokens((3,), 2_200_003), 0)


@DTYPES
def test_strided_rows_and_leading_dimensions(dtype):
    wide = logits((4, 6, 1203), dtype, 5)
    for x in (wide[..., 3:1000], wide[:, :, 1:], wide[1:3, :, 7:8], wide[0, 1::2, :]):
        check_forward(x, tokens(x.shape[:-1], x.shape[-1]), min(5, x.shape[-1]))
    one = logits((77,), dtype, 6)
    check_forward(one, torch.tensor(5, device=DEV), 3)
    with pytest.raises(AssertionError, match="one pitch"):
        ops.token_log_probs(wide[:, 1:4, :], tokens((4, 3), 1203))
    with pytest.raises(AssertionError, match="dense"):
        ops.token_log_probs(wide[..., ::2], tokens((4, 6), 602))


def test_no_rows():
    r = ops.token_log_probs(torch.zeros(0, 100, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), top=4)
    assert r.log_probs.shape == (0,) and r.stats.shape == (0, 2) and r.top_indices.shape == (0, 4)
    x = torch.zeros(0, 100, device=DEV)
    assert ops.token_log_probs_backward(x, torch.zeros(0, dtype=torch.int64, device=DEV), r.stats, None, r.log_probs).shape == x.shape


@DTYPES
@pytest.mark.parametrize("vocab", [40, 1500, 20011, 131072])
def test_masks(vocab, dtype):
    lowest = torch.finfo(dtype).min
    x = logits((12, vocab), dtype, 7)
    x[0] = -math.inf                      # nothing left
    x[1] = lowest                         # nothing but the lowest value: uniform
    x[2, : vocab // 2] = -math.inf
    x[3, vocab // 2:] = lowest
    x[4] = -math.inf
    x[4, vocab - 1] = 2.0                 # one token left
    x[5] = lowest
    x[5, 0] = -3.0
    x[6] = 1.25                           # all the same: ties by index
    x[7, 1::2] = -0.0
    x[7, ::2] = 0.0                       # one value
    x[8] = torch.finfo(dtype).max
    x[9, 3] = torch.finfo(dtype).max
    x[10] = -math.inf
    x[10, 2::3] = lowest                  # masked both ways, nothing else left
    x[11, vocab // 3:] = -math.inf
    x[11, : vocab // 4] = lowest
    t = torch.tensor([1, 2, vocab - 1, 0, vocab - 1, 0, 3, 4, 5, 3, -1, vocab], device=DEV)
    r = check_forward(x, t, min(20, vocab))
    for entropy in (False, True):
        check_backward(x, t.clamp(max=vocab - 1), entropy)
    assert r.log_probs[0] == -math.inf and r.entropy[0] == 0 and r.stats[0].tolist() == [-math.inf, 0.0]
    assert r.top_log_probs[0].eq(-math.inf).all() and r.top_indices[0].tolist() == list(range(min(20, vocab)))
    assert r.entropy[4] == 0 and r.log_probs[4] == 0
    check_forward(x, t, 0)


@DTYPES
@pytest.mark.parametrize("vocab", [40, 1500, 70001])
def test_nan_and_infinity(vocab, dtype):
    x = logits((4, vocab), dtype, 8)
    x[0, vocab // 2] = math.nan
    x[1, 3] = math.inf
    x[2] = math.nan
    t = torch.tensor([0, 0, 0, 0], device=DEV)
    r = ops.token_log_probs(x, t, top=5)
    for v in (r.log_probs, r.entropy, r.top_log_probs):
        assert v[:3].isnan().all() and v[3].isfinite().all()
    assert bool(((r.top_indices >= 0) & (r.top_indices < vocab)).all())
    d = ops.token_log_probs_backward(x, t, r.stats, r.entropy, torch.ones(4, device=DEV), torch.ones(4, device=DEV))
    assert d[2].isnan().all() and d[0, vocab // 2].isnan() and d[3].isfinite().all()


def check_backward(x, targets, entropy, out=None, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(77)
    vocab = x.shape[-1]
    lp, _, h, _ = plain(x, targets)
    dlp = scale * torch.randn(targets.shape, device=DEV, generator=g)
    dh = scale * torch.randn(targets.shape, device=DEV, generator=g) if entropy else None
    r = ops.token_log_probs(x, targets)
    got = ops.token_log_probs_backward(x, targets, r.stats, r.entropy, dlp, dh, out=out)
    ops.device_status()
    dead = (x == -math.inf).all(-1, keepdim=True)
    p = torch.where(dead, 0.0, lp.exp())
    gd = torch.where(targets < 0, 0.0, dlp.double())[..., None]
    hd = dh.double()[..., None] if entropy else torch.zeros_like(gd)
    hot = torch.zeros_like(p).scatter_(-1, targets.clamp(min=0)[..., None], 1.0)
    inner = torch.where(p > 0, lp + h[..., None], 0.0)
    want = torch.where(dead, 0.0, gd * (hot - p) - hd * p * inner)
    # p is off by the statistics' error and that of its argument; the bracket and the products by a few u each
    c = chain(vocab, x.dtype)
    m = x.double().amax(-1, keepdim=True)
    span = torch.where(torch.isfinite(lp), lp.abs(), 0.0)
    log_s = torch.where(dead, 0.0, lp.amax(-1, keepdim=True).abs())
    off_lp = (8 + c) * U + 4 * U * (span + log_s)
    off_h = (8 + c) * U + 4 * U * log_s + h[..., None] * (16 + 2 * c) * U
    size = p * (gd.abs() + hd.abs() * (span + h[..., None]))
    tol = size * (off_lp + 8 * U) + p * hd.abs() * (off_lp + off_h) + 2 * U * (gd * hot).abs()
    tol = tol + (2.0 ** -11 * want.abs() + 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -149)
    assert got.dtype == x.dtype and got.shape == x.shape
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))
    return got


@DTYPES
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 17), (5, 33), (256, 1000), (7, 2049), (3, 50021), (1, 131072), (1200, 1111)])
def test_gradient(rows, vocab, entropy, dtype):
    check_backward(logits((rows, vocab), dtype, vocab + 1), tokens((rows,), vocab), entropy, scale=100.0)


@DTYPES
def test_gradient_of_masked_rows(dtype):
    x = logits((6, 3001), dtype, 9)
    x[0] = -math.inf
    x[1, :3000] = -math.inf
    x[2, 5:] = torch.finfo(dtype).min
    x[3] = torch.finfo(dtype).min
    t = torch.tensor([4, 3000, 1, 2, -100, 0], device=DEV)
    for entropy in (False, True):
        d = check_backward(x, t, entropy)
        assert not d[0].any()


@DTYPES
def test_gradient_into_views(dtype):
    """A result whose rows start elsewhere than the logits', and one in the logits' own memory; what lies beside it stays."""
    x = logits((5, 1003), dtype, 10)
    t = tokens((5,), 1003)
    for lead in (0, 1, 5):
        room = torch.full((5, 1100), 7.0, dtype=dtype, device=DEV)
        check_backward(x, t, True, out=room[:, lead:lead + 1003])
        assert room[:, :lead].eq(7).all() and room[:, lead + 1003:].eq(7).all()
    want = check_backward(x, t, True)
    y = x.clone()
    r = ops.token_log_probs(y, t)
    g = torch.Generator(device=DEV).manual_seed(77)
    dlp, dh = torch.randn(5, device=DEV, generator=g), torch.randn(5, device=DEV, generator=g)
    got = ops.token_log_probs_backward(y, t, r.stats, r.entropy, dlp, dh, out=y)
    assert got.data_ptr() == y.data_ptr() and torch.equal(got, want)


def test_target_beyond_the_vocabulary():
    x, t = logits((2, 50), torch.float32, 11), torch.tensor([50, 3], device=DEV)
    r = ops.token_log_probs(x, t)
    assert r.log_probs[0].isnan() and r.log_probs[1].isfinite() and r.entropy.isfinite().all()
    assert ops.token_log_probs_backward(x, t, r.stats, None, torch.ones(2, device=DEV))[0].isnan().all()


def test_gradient_against_differences():
    x = logits((4, 37), torch.float32, 12).double()
    t = tokens((4,), 37)
    wl, wh = torch.randn(4, device=DEV), torch.randn(4, device=DEV)
    r = ops.token_log_probs(x.float(), t)
    d = ops.token_log_probs_backward(x.float(), t, r.stats, r.entropy, wl, wh)

    def value(z):
        _, token, h, _ = plain(z, t)
        return wl.double() * token + wh.double() * h
    x = x.float().double()
    for j in range(37):
        z = x.clone()
        z[:, j] += 1e-5
        w = x.clone()
        w[:, j] -= 1e-5
        # (central differences: h^2 / 6 times a third derivative below 50, and 64-bit rounding over h)
        assert torch.allclose(d[:, j].double(), (value(z) - value(w)) / 2e-5, rtol=1e-5, atol=1e-6)


def test_repeatable_on_other_streams_and_in_graphs():
    x = logits((64, 30011), torch.float16, 13)
    t = tokens((64,), 30011)
    dlp = torch.ones(64, device=DEV)
    want = ops.token_log_probs(x, t, top=9)
    grad = ops.token_log_probs_backward(x, t, want.stats, want.entropy, dlp, dlp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.token_log_probs(x, t, top=9)
        grad2 = ops.token_log_probs_backward(x, t, again.stats, again.entropy, dlp, dlp)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, again)) and torch.equal(grad, grad2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.token_log_probs(x, t, top=9)
        grad3 = ops.token_log_probs_backward(x, t, held.stats, held.entropy, dlp, dlp)
    x.copy_(logits((64, 30011), torch.float16, 14))
    graph.replay()
    new = ops.token_log_probs(x, t, top=9)
    assert all(torch.equal(a, b) for a, b in zip(new, held))
    assert torch.equal(grad3, ops.token_log_probs_backward(x, t, new.stats, new.entropy, dlp, dlp))
    ops.device_status()


def test_offsets_beyond_32_bits():
    """Rows whose elements lie more than 2^32 bytes and 2^31 elements into the tensor."""
    rows, vocab = 70000, 32768
    x = torch.empty(rows, vocab, dtype=torch.float16, device=DEV)
    last = logits((3, vocab), torch.float16, 15)
    x.fill_(0.5)
    x[-3:] = last
    t = tokens((rows,), vocab)
    r = ops.token_log_probs(x, t, top=2)
    small = ops.token_log_probs(last, t[-3:].contiguous(), top=2)
    for a, b in zip(r, small):
        assert torch.allclose(a[-3:].double(), b.double(), rtol=1e-5, atol=0)
    assert r.top_indices[:-3].eq(torch.arange(2, device=DEV)).all()
    d = ops.token_log_probs_backward(x, t, r.stats, None, torch.ones(rows, device=DEV), out=x)
    want = ops.token_log_probs_backward(last, t[-3:].contiguous(), r.stats[-3:].contiguous(), None, torch.ones(3, device=DEV))
    assert torch.equal(d[-3:], want)


@DTYPES
def test_autograd(dtype):
    """Gradients of shared, broadcast and unused outputs."""
    x = logits((6, 777), dtype, 16).requires_grad_(True)
    t = tokens((6,), 777)
    r = train.token_log_probs(x, t, top=4)
    assert not r.top_log_probs.requires_grad and not r.stats.requires_grad
    plainly = ops.token_log_probs(x.detach(), t, top=4)
    assert all(torch.equal(a, b) for a, b in zip(r, plainly))
    (2.0 * r.log_probs.sum() + r.log_probs.sum() - r.entropy.mean()).backward()
    ones = torch.ones(6, device=DEV)
    want = ops.token_log_probs_backward(x.detach(), t, plainly.stats, plainly.entropy, 3 * ones, -(1 / torch.full((6,), 6.0, device=DEV)))
    assert torch.equal(x.grad, want)
    for part in ("log_probs", "entropy"):
        x.grad = None
        getattr(train.token_log_probs(x, t), part).sum().backward()
        want = ops.token_log_probs_backward(x.detach(), t, plainly.stats, plainly.entropy, ones * (part == "log_probs"),
                                            ones if part == "entropy" else None)
        assert torch.equal(x.grad, want)
    weight = ones.clone().requires_grad_(True)
    g, = torch.autograd.grad((weight * train.token_log_probs(x, t).log_probs).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):   # (and not a second gradient that lacks a part)
        g.square().sum().backward()


def test_training_step_with_this_loss():
    """The classifier's step with the library's loss against the same step with torch's, and with an entropy term."""
    n, classes = 8, 24
    x = torch.randn(n, 64, 64, 3, device=DEV).half()
    labels = torch.randint(0, classes, (n,), device=DEV)
    grads = {}
    for loss, weight in (("cross_entropy", 0.0), ("token_log_probs", 0.0), ("token_log_probs", 0.1)):
        net = train.ResNet50(DEV, num_classes=classes, blocks=(1, 1, 1, 1), width=16)
        net.init(seed=3)
        step = train.TrainStep(net, loss, loss_scale=8192.0, entropy_weight=weight)
        value = step([(x, labels)], global_count=n, optimize=False)
        ops.device_status()
        grads[loss, weight] = (float(value), net.store.grad.double().clone(), net)
    (a, ga, _), (b, gb, _), (c, gc, net) = grads.values()
    # (the logits' gradients are half precision: they differ by single roundings of 2^-11, which every layer behind passes on)
    assert abs(a - b) <= 1e-5 * abs(a) and float((ga - gb).norm()) <= 2.0 ** -8 * float(ga.norm())
    with torch.no_grad():
        out = net.forward(x).double()
    h = -(out.log_softmax(1) * out.softmax(1)).sum()
    assert abs(c - (b - 0.1 * float(h) / n)) <= 1e-5 * abs(c) and float((gc - gb).norm()) > 0.01 * float(gb.norm())
