"""Orthogonalised matrices and the optimizer step on them against the iteration in 64 bits.

Tolerances (Frobenius norm of the difference over that of the result).  A step takes A, P = b I + c A and U = a I + P A through storage of
w bits, each off by half a step, u = 2^-w.  Near singular values of 1, where the result's norm is, U = 0.70 and P A = -2.74, so U is off by
(2 x 2.74 + 0.70) u = 8.9 u of itself where roundings all point one way; an error there shrinks by |p'(1)| = 0.72 a step, which
sums to 3.6 over any number of steps: 32 u.  With fp16 storage ("f16", u = 2^-12): 7.9e-3.  With two halves ("3xf16", u = 2^-23) and the
product of the low halves left out, another 2^-22: 1.2e-5.  To that comes X's own storage, 2^-23 in either mode, which grows by a a step
in directions that hold nothing else: 2^-23 a^5 = 5.8e-5 of |X_0| = 1, while the result's norm is at least 0.6 sqrt(number of
directions); spread over a matrix of 4 or more such directions 5e-5 in all."""
import math

import pytest
import torch

from nectarml_b200 import _lib, ops, train

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
COEF = ops.ORTHOGONALIZE_COEFFICIENTS
TOL = {"3xf16": 7e-5, "f16": 8e-3}
HALF = 2.0 ** -11


def plain(g, steps=5, coefficients=COEF, eps=1e-7):
    x = g.double()
    turn = x.shape[-2] > x.shape[-1]
    x = x.mT if turn else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for k in range(steps):
        a, b, c = coefficients[k] if hasattr(coefficients[0], "__len__") else coefficients
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if turn else x


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def gradient(rows, cols, dtype=torch.float32, seed=0, n=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    shape = (rows, cols) if n is None else (n, rows, cols)
    rank = min(rows, cols, 24)
    a = torch.randn(*shape[:-1], rank, device=DEV, generator=g)
    b = torch.randn(*shape[:-2], rank, cols, device=DEV, generator=g)
    return (0.02 * (a @ b / math.sqrt(rank) + 0.3 * torch.randn(shape, device=DEV, generator=g))).to(dtype)


MODES = pytest.mark.parametrize("mode", ["3xf16", "f16"])
SIZES = [(1, 1), (1, 7), (7, 1), (2, 3), (16, 16), (64, 147), (65, 64), (64, 64), (127, 129), (128, 128), (129, 300), (1, 1000), (200, 1000), (1000, 200), (256, 513),
         (513, 257), (640, 641), (192, 2304), (2304, 192), (66, 8000), (190, 5000), (3000, 321), (449, 1025)]


@MODES
@pytest.mark.parametrize("rows,cols", SIZES)
def test_sizes(rows, cols, mode):
    g = gradient(rows, cols, seed=rows + cols)
    y = ops.orthogonalize(g, math=mode)
    ops.device_status()
    assert y.shape == g.shape and y.dtype == torch.float32
    assert off(y, plain(g)) <= TOL[mode]


@pytest.mark.parametrize("rows,cols", [(3, 5), (100, 60), (300, 700), (1024, 1024)])
def test_half_precision(rows, cols):
    g = gradient(rows, cols, torch.float16, seed=rows)
    y = ops.orthogonalize(g)
    assert y.dtype == torch.float16 and off(y, plain(g)) <= TOL["3xf16"] + HALF
    assert torch.equal(y, ops.orthogonalize(g, math="3xf16"))
    fast = ops.orthogonalize(g, math="f16")
    assert fast.dtype == torch.float16 and off(fast, plain(g)) <= TOL["f16"] + HALF
    wide = ops.orthogonalize(g, math="3xf16", out_dtype=torch.float32)
    assert wide.dtype == torch.float32 and off(wide, plain(g)) <= TOL["3xf16"]
    half = ops.orthogonalize(g.float(), out_dtype=torch.float16)
    assert half.dtype == torch.float16 and off(half, plain(g)) <= TOL["3xf16"] + HALF


@MODES
@pytest.mark.parametrize("shapes", [[(1601, 1700)], [(2000, 1537)], [(1550, 2600)], [(1100, 1100), (700, 2000), (65, 300), (1, 5), (900, 640)],
                                    [(384, 1024)] * 15 + [(129, 4000), (300, 257)]], ids=str)
def test_many_tiles(shapes, mode):
    """Two blocks to a tile: an odd and an even number of block rows, one alone, ragged ends, beside matrices of one block row."""
    gs = [gradient(r, c, seed=r + k) for k, (r, c) in enumerate(shapes)]
    ys = ops.orthogonalize(gs, math=mode)
    ops.device_status()
    for g, y in zip(gs, ys):
        assert off(y, plain(g)) <= TOL[mode], g.shape
    assert all(torch.equal(a, b) for a, b in zip(ys, ops.orthogonalize(gs, math=mode)))


def test_many_tiles_in_graphs_on_streams_and_few_sms():
    """Two graphs with workspaces of their own, replayed side by side; any number of SMs; a NaN stays in its matrix."""
    gs = [gradient(r, c, seed=r) for r, c in ((1600, 1800), (1700, 1601))]
    want = [ops.orthogonalize(g) for g in gs]
    streams, spaces = [torch.cuda.Stream() for _ in gs], [ops.Workspace() for _ in gs]
    ins, outs, graphs = [torch.zeros_like(g) for g in gs], [torch.zeros_like(g) for g in gs], []
    for x, y, ws, stream in zip(ins, outs, spaces, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.orthogonalize(x, out=y, ws=ws)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            ops.orthogonalize(x, out=y, ws=ws)
    for x, g in zip(ins, gs):
        x.copy_(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    ops.device_status()
    assert all(torch.equal(y, w) for y, w in zip(outs, want))
    try:
        for sms in (1, 2, 3, 37):
            ops.set_sm_limit(sms)
            assert off(ops.orthogonalize(gs[0]), plain(gs[0])) <= TOL["3xf16"], sms
    finally:
        ops.set_sm_limit(0)
    group = [gradient(512, 2048, seed=k) for k in range(9)]
    group[4][3, 5] = math.nan
    ys = ops.orthogonalize(group)
    assert bool(ys[4].isnan().all())
    assert all(off(ys[k], plain(group[k])) <= TOL["3xf16"] for k in range(9) if k != 4)


@MODES
def test_singular_values_and_vectors(mode):
    """What the operator is for: singular values near 1, the same singular vectors."""
    g = gradient(96, 250, seed=5)
    y = ops.orthogonalize(g, math=mode).double()
    u, s, v = torch.linalg.svd(g.double(), full_matrices=False)
    d = u.T @ y @ v.T
    assert bool(((d.diagonal() > 0.6) & (d.diagonal() < 1.3)).all())
    assert float((d - torch.diag(d.diagonal())).norm()) <= 2 * TOL[mode] * float(y.norm())


@MODES
def test_groups(mode):
    """Many matrices through the same launches, more than go in at once."""
    shapes = [(1 + 37 * k % 300, 1 + 61 * k % 500) for k in range(140)]
    gs = [gradient(r, c, seed=k) for k, (r, c) in enumerate(shapes)]
    ys = ops.orthogonalize(gs, math=mode)
    ops.device_status()
    assert len(ys) == len(gs)
    for g, y in zip(gs, ys):
        assert off(y, plain(g)) <= TOL[mode], g.shape
    assert all(torch.equal(a, b) for a, b in zip(ys, ops.orthogonalize(gs, math=mode)))


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (15, 16), (16, 17), (17, 1000), (64, 64), (64, 147), (64, 1536), (1537, 64), (48, 10000), (33, 20001)])
def test_small_matrices_are_rounded_once(rows, cols):
    """Groups of matrices with a short side up to 64 are computed in double: off by a rounding of fp32 storage, in either mode; 2^-45 a^10 of what
    double leaves is far below that."""
    g = [gradient(rows, cols, seed=cols), gradient(64, 300, seed=1), torch.outer(torch.randn(rows, device=DEV), torch.randn(cols, device=DEV))]
    for mode in ("3xf16", "f16"):
        for x, y in zip(g, ops.orthogonalize(g, math=mode)):
            assert off(y, plain(x)) <= 2.0 ** -24, mode
    many = [gradient(1 + k % 64, 1 + 37 * k % 300, seed=k) for k in range(150)]
    ys = ops.orthogonalize(many)
    assert all(off(y, plain(x)) <= 2.0 ** -24 for x, y in zip(many, ys))
    assert torch.equal(ops.orthogonalize(many[100]), ys[100])
    half = [x.half() for x in g]
    for x, y in zip(half, ops.orthogonalize(half)):
        assert y.dtype == torch.float16 and off(y, plain(x)) <= HALF


@MODES
def test_batches(mode):
    g = gradient(70, 150, seed=6, n=5)
    y = ops.orthogonalize(g, math=mode)
    for k in range(5):
        assert off(y[k], plain(g[k])) <= TOL[mode]
    both = ops.orthogonalize([g, g[0].T.contiguous()], math=mode)
    assert off(both[0], plain(g)) <= TOL[mode] and off(both[1], plain(g[0].T)) <= TOL[mode]
    same = ops.orthogonalize(g[:1].expand(3, 70, 150), math=mode)   # one matrix, read three times
    assert off(same[0], plain(g[0])) <= TOL[mode] and all(torch.equal(same[k], same[0]) for k in range(3))
    out = torch.empty(1, 70, 150, device=DEV).expand(3, 70, 150)
    with pytest.raises(AssertionError, match="places of their own"):
        ops.orthogonalize(g[:3], out=out)


@MODES
def test_views(mode):
    big = gradient(400, 700, seed=7)
    for g in (big.T, big[:, 1:302], big[3:200], big[5:133, 7:264].T, big[:, 9:10], big[17:18, 3:], big[:1].T, big[:2, :3], big[:, 4:5].T):
        want = plain(g)
        y = ops.orthogonalize(g, math=mode)
        assert off(y, want) <= TOL[mode], (g.shape, g.stride())
        room = torch.full((g.shape[0] + 2, g.shape[1] + 3), 9.0, device=DEV)
        into = room[1:-1, 2:-1]
        assert ops.orthogonalize(g, math=mode, out=into) is not None and torch.equal(into, y)
        room[1:-1, 2:-1] = 9.0
        assert room.eq(9.0).all()
        turned = torch.empty(g.shape[1], g.shape[0], device=DEV).T
        ops.orthogonalize(g, math=mode, out=turned)
        assert torch.equal(turned, y)
    with pytest.raises(AssertionError, match="dense dimension"):
        ops.orthogonalize(big[:, ::2])
    with pytest.raises(AssertionError, match="matrices"):
        ops.orthogonalize(big[0])


def test_in_place():
    g = gradient(130, 260, seed=8)
    want = ops.orthogonalize(g)
    assert torch.equal(ops.orthogonalize(g, out=g), want) and torch.equal(g, want)


@MODES
def test_zeros_nan_infinity_and_range(mode):
    zero, nan, inf = torch.zeros(100, 140, device=DEV), gradient(100, 140), gradient(140, 100)
    nan[99, 139] = math.nan
    inf[0, 0] = math.inf
    tiny, huge = gradient(100, 140, seed=9) * 1e-30, gradient(100, 140, seed=9) * 1e30
    one = torch.zeros(100, 140, device=DEV)
    one[3, 5] = 7.0
    for eps in (0.0, 1e-7):
        y = ops.orthogonalize([zero, nan, inf, huge, one], math=mode, eps=eps)
        assert not y[0].any() and y[1].isnan().all() and y[2].isnan().all()
        assert off(y[3], plain(huge, eps=eps)) <= TOL[mode]
        want = plain(one, eps=eps)
        assert off(y[4], want) <= TOL[mode] and int((y[4] != 0).sum()) == 1
    assert off(ops.orthogonalize(tiny, math=mode, eps=0.0), plain(tiny, eps=0.0)) <= TOL[mode]
    y, want = ops.orthogonalize(tiny, math=mode), plain(tiny)   # far below eps: small, but right
    assert float(want.norm()) < 1e-10 and float(y.norm()) < 1e-10
    ops.device_status()


@MODES
def test_coefficients(mode):
    g = gradient(80, 200, seed=10)
    rows = ((3.9, -4.0, 1.2), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375))
    for steps, c in ((1, COEF), (2, COEF), (3, rows), (1, (1.0, 0.0, 0.0)), (3, (1.5, -0.5, 0.0)), (12, (2.0, -1.5, 0.5))):
        y = ops.orthogonalize(g, steps=steps, coefficients=c, math=mode)
        assert off(y, plain(g, steps, c)) <= TOL[mode], (steps, c)
    with pytest.raises(_lib.NectarB200Error, match="status 4"):
        ops.orthogonalize(g, coefficients=(9.0, 5.0, 5.0))


@MODES
def test_repeatable_on_other_streams_in_graphs_and_on_fewer_sms(mode):
    gs = [gradient(300, 500, seed=11), gradient(520, 130, seed=12)]
    want = ops.orthogonalize(gs, math=mode)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    assert same(ops.orthogonalize(gs, math=mode), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ws = ops.Workspace()
    with torch.cuda.stream(side):
        again = ops.orthogonalize(gs, math=mode, ws=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert same(again, want)
    ops.set_sm_limit(5)
    try:
        few = ops.orthogonalize(gs, math=mode)   # (in other tiles, so in another order of sums)
    finally:
        ops.set_sm_limit(0)
    assert all(off(y, plain(g)) <= TOL[mode] for y, g in zip(few, gs))
    graph, own = torch.cuda.CUDAGraph(), ops.Workspace()
    own.get(1 << 26, DEV)
    with torch.cuda.graph(graph):
        held = ops.orthogonalize(gs, math=mode, ws=own)
    for g in gs:
        g.mul_(-0.5).add_(0.01)
    graph.replay()
    assert same(held, ops.orthogonalize(gs, math=mode))
    ops.device_status()


def test_large_matrices():
    for rows, cols in ((2048, 1100), (4100, 2050)):
        g = gradient(rows, cols, seed=13)
        want = plain(g)
        assert off(ops.orthogonalize(g), want) <= TOL["3xf16"]
        assert off(ops.orthogonalize(g, math="f16"), want) <= TOL["f16"]


# ------------------------------------------------------------------ the optimizer step --
def model(shapes, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda s: 0.05 * torch.randn(s, device=DEV, generator=g)
    return [mk(s) for s in shapes], [64.0 * mk(s) for s in shapes], [mk(s) for s in shapes]


def plain_step(p, g, v, lr, momentum, nesterov, decay, inv, scaling):
    p, g, v = p.double(), g.double() * inv, v.double()
    v = momentum * v + g
    u = g + momentum * v if nesterov else v
    if p.dim() > 1:
        rows, cols = p.shape[0], p.numel() // p.shape[0]
        s = {"spectral": math.sqrt(max(1.0, rows / cols)), "rms": 0.2 * math.sqrt(max(rows, cols)), None: 1.0}[scaling]
        u = s * plain(u.reshape(rows, cols)).reshape(p.shape)
    return p * (1 - lr * decay) - lr * u, v, lr * u


SHAPES = [(64, 3, 7, 7), (64,), (130, 70), (70,), (1, 9), (9, 1), (257, 300), (5,), (32, 16, 4, 4)]


@pytest.mark.parametrize("nesterov,scaling,mode", [(True, "spectral", "3xf16"), (False, "rms", "3xf16"), (True, None, "f16")])
def test_muon_step(nesterov, scaling, mode):
    params, grads, momenta = model(SHAPES)
    halves = [None if k % 3 == 2 else p.half() for k, p in enumerate(params)]
    lr, mom, decay, inv = 0.03, 0.9, 0.1, 1 / 64
    want = [plain_step(p, g, v, lr, mom, nesterov, decay, inv, scaling) for p, g, v in zip(params, grads, momenta)]
    ops.muon_step(params, grads, momenta, halves, lr=lr, momentum=mom, nesterov=nesterov, weight_decay=decay, inv_scale=inv, scaling=scaling, math=mode)
    ops.device_status()
    for p, v, h, (wp, wv, wu) in zip(params, momenta, halves, want):
        tol = TOL[mode] * float(wu.norm()) + 2.0 ** -22 * float(wp.norm())
        assert float((p.double() - wp).norm()) <= tol, p.shape
        assert float((v.double() - wv).norm()) <= 2.0 ** -22 * float(wv.norm())
        if h is not None:
            assert torch.equal(h, p.half())


@pytest.mark.parametrize("shapes", [[(1601, 1700), (33,)], [(2000, 1537)], [(1700, 1600), (1600, 1700)], [(384, 1024)] * 8 + [(1030, 390)] * 9], ids=str)
def test_muon_step_of_many_tiles(shapes):
    """Pairs of blocks: parameters whose rows are aligned and not, along and across memory, an odd number of block rows."""
    params, grads, momenta = model(shapes)
    halves = [p.half() for p in params]
    want = [plain_step(p, g, v, 0.03, 0.9, True, 0.1, 1.0, "spectral") for p, g, v in zip(params, grads, momenta)]
    ops.muon_step(params, grads, momenta, halves, lr=0.03, momentum=0.9, weight_decay=0.1)
    ops.device_status()
    for p, v, h, (wp, wv, wu) in zip(params, momenta, halves, want):
        assert float((p.double() - wp).norm()) <= TOL["3xf16"] * float(wu.norm()) + 2.0 ** -22 * float(wp.norm()), p.shape
        assert float((v.double() - wv).norm()) <= 2.0 ** -22 * float(wv.norm())
        assert torch.equal(h, p.half())


def test_muon_step_of_small_parameters():
    """The same where all matrices have a short side up to 64."""
    shapes = [(64, 3, 7, 7), (64,), (13, 70), (500, 64), (1, 9), (9, 1), (64, 64)]
    params, grads, momenta = model(shapes, 7)
    halves = [p.half() for p in params]
    want = [plain_step(p, g, v, 0.03, 0.9, True, 0.1, 1 / 64, "spectral") for p, g, v in zip(params, grads, momenta)]
    kept = [t.clone() for t in params + momenta + halves]
    found = torch.ones(1, dtype=torch.int32, device=DEV)
    step = lambda: ops.muon_step(params, grads, momenta, halves, lr=0.03, momentum=0.9, weight_decay=0.1, inv_scale=1 / 64, found_inf=found)
    step()
    assert all(torch.equal(a, b) for a, b in zip(params + momenta + halves, kept))
    found.zero_()
    step()
    ops.device_status()
    for p, v, h, (wp, wv, wu) in zip(params, momenta, halves, want):
        # (the momentum is fp32: its rounding, 2 x 2^-24, grows with the update's small directions like the tolerances above)
        assert float((p.double() - wp).norm()) <= TOL["3xf16"] * float(wu.norm()) + 2.0 ** -22 * float(wp.norm()), p.shape
        assert float((v.double() - wv).norm()) <= 2.0 ** -22 * float(wv.norm()) and torch.equal(h, p.half())


def test_muon_step_leaves_everything_where_a_gradient_overflowed():
    params, grads, momenta = model(SHAPES, 1)
    halves = [p.half() for p in params]
    kept = [t.clone() for t in params + momenta + halves]
    found = torch.ones(1, dtype=torch.int32, device=DEV)
    grads[0][0, 0, 0, 0] = math.inf
    ops.muon_step(params, grads, momenta, halves, lr=0.1, found_inf=found)
    assert all(torch.equal(a, b) for a, b in zip(params + momenta + halves, kept))
    found.zero_()
    grads[0][0, 0, 0, 0] = 0.0
    ops.muon_step(params, grads, momenta, halves, lr=0.1, found_inf=found)
    assert not any(torch.equal(a, b) for a, b in zip(params + momenta + halves, kept))
    ops.device_status()


def test_muon_step_over_many_parameters():
    shapes = [s for k in range(140) for s in ((8 + k, 40), (8 + k,))]
    params, grads, momenta = model(shapes, 2)
    want = [plain_step(p, g, v, 0.02, 0.95, True, 0.0, 1.0, "spectral") for p, g, v in zip(params, grads, momenta)]
    ops.muon_step(params, grads, momenta, lr=0.02)
    for p, (wp, _, wu) in zip(params, want):
        assert float((p.double() - wp).norm()) <= TOL["3xf16"] * float(wu.norm()) + 2.0 ** -22 * float(wp.norm()), p.shape
    ops.muon_step([], [], [], lr=0.02)
    with pytest.raises(_lib.NectarB200Error, match="status 1"):
        ops.muon_step([params[0], params[0]], [grads[0], grads[0]], [momenta[0], momenta[0]], lr=0.02)


@pytest.mark.parametrize("optimizer", ["sgd", "muon"])
def test_training_steps(optimizer):
    """Two optimisation steps of the classifier with the library's loss: forward, backward, finiteness check and update, against the
    updates computed from the same gradients."""
    n, classes = 8, 24
    net = train.ResNet50(DEV, num_classes=classes, blocks=(1, 1, 1, 1), width=16)
    net.init(seed=3)
    s = net.store
    step = train.TrainStep(net, "token_log_probs", lr=0.02, momentum=0.9, weight_decay=1e-2, loss_scale=1024.0, entropy_weight=0.01, optimizer=optimizer)
    x = torch.randn(n, 64, 64, 3, device=DEV).half()
    labels = torch.randint(0, classes, (n,), device=DEV)
    for _ in range(2):
        before, vel = s.p32.clone(), s.vel.clone()
        step([(x, labels)], global_count=n)
        ops.device_status()
        assert int(s.found_inf) == 0
        for i, shape in enumerate(s.shapes):
            part = slice(s.offsets[i], s.offsets[i] + math.prod(shape))
            p, g, v = before[part].view(shape), s.g32(i), vel[part].view(shape)
            if optimizer == "muon":
                want, wv, wu = plain_step(p, g, v, 0.02, 0.9, True, 1e-2, 1 / 1024, "spectral")
            else:
                wv = 0.9 * v.double() + g.double() / 1024 + 1e-2 * p.double()
                want, wu = p.double() - 0.02 * wv, 0.02 * wv
            tol = (TOL["3xf16"] if optimizer == "muon" else 2.0 ** -21) * float(wu.norm()) + 2.0 ** -22 * float(want.norm())
            assert float((s.w32(i).double() - want).norm()) <= tol, (i, shape)
            assert torch.equal(s.w16(i), s.w32(i).half())
    net.store.grad[5] = math.inf
    kept = s.p32.clone()
    step.optimizer_step()
    assert int(s.found_inf) == 1 and torch.equal(s.p32, kept)
