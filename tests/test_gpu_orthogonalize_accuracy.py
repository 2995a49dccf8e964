"""How exact orthogonalised matrices are beside the same steps in fp32, for chains of any length and steps of any polynomial.

The tolerance.  Two halves hold a number to 2^-22, and a product leaves another 2^-22 for that of the low halves: 3 x 2^-22 in all, where fp32 rounds both factors
by 2^-24.  That is 12 of its roundings to 2, so six times the error that the plain fp32 steps show on the same matrix; truncating accumulators
(7e-5 over K = 8192, some 2e-6 in fp32) would not pass."""
import math

import pytest
import torch

from nectarml_b200 import _lib, ops, train

from test_gpu_orthogonalize import COEF, DEV, MODES, TOL, gradient, model, off, plain, plain_step

pytestmark = pytest.mark.gpu


def in_fp32(g, steps=5, coefficients=COEF, eps=1e-7):
    assert not torch.backends.cuda.matmul.allow_tf32
    x = g.float()
    turn = x.shape[-2] > x.shape[-1]
    x = x.mT if turn else x
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + eps).float()
    for k in range(steps):
        a, b, c = coefficients[k] if hasattr(coefficients[0], "__len__") else coefficients
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if turn else x


def check(g, y, steps=5, coefficients=COEF, mode="3xf16", one_way=0.0):
    want = plain(g, steps, coefficients)
    assert off(y, want) <= (6 * off(in_fp32(g, steps, coefficients), want) + one_way if mode == "3xf16" else TOL["f16"]), (g.shape, steps, off(y, want))


@pytest.mark.parametrize("shapes", [[(300, 400)], [(256, 513)], [(300, 700)], [(400, 5000)], [(1024, 1024)], [(2048, 8192)], [(8192, 2048)], [(1600, 1700)], [(1100, 1700)],
                                    [(512, 2048)] * 9, [(500, 900), (200, 2000), (384, 384)] * 3], ids=lambda s: str(s[:4]))
@pytest.mark.parametrize("kind", ["random", "strong directions"])
def test_as_exact_as_fp32(shapes, kind):
    gen = torch.Generator(device=DEV).manual_seed(3)
    gs = [gradient(r, c, seed=k) if kind != "random" else torch.randn(r, c, device=DEV, generator=gen) for k, (r, c) in enumerate(shapes)]
    for g, y in zip(gs, ops.orthogonalize(gs)):
        check(g, y)
    ops.device_status()


ROWS = ((3.9, -4.0, 1.2), (2.0, -1.5, 0.5), (3.4445, -4.7750, 2.0315), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0), (2.5, -2.0, 0.6), (1.2, -0.3, 0.05), (2.0, -1.5, 0.5))


MILD = ((3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.2, -0.3, 0.05), (1.1, -0.1, 0.01))


def largest(steps, coefficients, margin):
    """The largest singular value that a start of at most 1 may reach, each step's by `margin` more."""
    most = reach = margin
    for k in range(steps):
        a, b, c = coefficients[k] if hasattr(coefficients[0], "__len__") else coefficients
        x = torch.linspace(0, min(reach, 1e3), 4001, dtype=torch.float64)
        reach = float((a * x + b * x ** 3 + c * x ** 5).abs().max()) * margin
        most = max(most, reach)
    return most


@MODES
@pytest.mark.parametrize("shapes", [[(300, 700)], [(700, 256), (128, 300)], [(512, 1500)] * 8, [(1601, 2500), (300, 2000)]], ids=str)
def test_polynomials_and_chains(shapes, mode):
    """Chains of every length (what ends one is how much its steps amplify an error): of one to eight steps with coefficients of their own, of twelve, sixteen and
    nineteen equal ones, two at a time and more, so that each pair of buffers takes its turns.

    Beside six times fp32's error: a step multiplies X, or a chain's Q, by U, whose diagonal is a and what little the steps add; it is stored to 2^-22, so is the
    product, and that of the low halves is left out, 3 x 2^-22 of the result.  Where X stays small, U's diagonal is the same number in every
    step and every direction, so these roundings all point one way and add up: 3 x 2^-22 a step.  (The fp32 steps multiply X by a itself.)"""
    gs = [gradient(r, c, seed=70 + k) for k, (r, c) in enumerate(shapes)]
    calls = [(n, ROWS[:n]) for n in range(1, 9)] + [(12, (2.0, -1.5, 0.5)), (16, (1.5, -0.5, 0.0)), (19, (1.2, -0.3, 0.05)), (2, COEF), (3, COEF), (4, COEF), (7, (1.05, 0.02, 0.0)),
                                                    (3, (6.0, -9.0, 4.0)), (4, ((1.0, 0.0, 0.0),) * 4), (5, ((-1.0, 0.0, 0.0),) * 5)]
    calls += [(n, MILD[:n]) for n in range(2, 9)]
    taken = 0
    for steps, c in calls:
        if largest(steps, c, 1.01) > 64:   # (refused where a singular value could grow beyond 64, by bounds that hold between the points where they are taken)
            if largest(steps, c, 1.0) > 64:
                with pytest.raises(_lib.NectarB200Error, match="status 4"):
                    ops.orthogonalize(gs, steps=steps, coefficients=c, math=mode)
            continue
        taken += 1
        ys = ops.orthogonalize(gs, steps=steps, coefficients=c, math=mode)
        ops.device_status()
        for g, y in zip(gs, ys):
            check(g, y, steps, c, mode, steps * 3 * 2.0 ** -22)
    assert taken == 18


def test_optimizer_step_in_graphs():
    """Captured with a workspace of its own, on a side stream, replayed with other gradients, beside eager steps of another workspace; skipped where
    the device says so."""
    shapes = [(130, 70), (70,), (300, 700), (64, 3, 7, 7), (64,), (20000,)]
    params, grads, momenta = model(shapes, 5)
    halves = [p.half() for p in params]
    found = torch.zeros(1, dtype=torch.int32, device=DEV)
    ws, eager_ws, stream, graph = ops.Workspace(), ops.Workspace(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    step = lambda p, g, v, h, w: ops.muon_step(p, g, v, h, lr=0.03, momentum=0.9, weight_decay=0.1, found_inf=found, ws=w)
    state = [t.clone() for t in params + momenta + halves]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(params, grads, momenta, halves, ws)   # (the workspace is there when the capture begins)
    torch.cuda.synchronize()
    for t, s in zip(params + momenta + halves, state):
        t.copy_(s)
    with torch.cuda.graph(graph, stream=stream):
        step(params, grads, momenta, halves, ws)
    other = [[t.clone() for t in part] for part in (params, grads, momenta, halves)]
    for k in range(4):
        for g, o in zip(grads, other[1]):
            g.copy_(torch.randn_like(g) * (k + 1))
            o.copy_(g)
        found.fill_(int(k == 2))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        step(*other, eager_ws)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params + momenta + halves, other[0] + other[2] + other[3])), k
    want = [plain_step(p, g, v, 0.03, 0.9, True, 0.1, 1.0, "spectral") for p, g, v in zip(params, grads, momenta)]
    graph.replay()
    torch.cuda.synchronize()
    ops.device_status()
    for p, (wp, _, wu) in zip(params, want):
        assert float((p.double() - wp).norm()) <= TOL["3xf16"] * float(wu.norm()) + 2.0 ** -22 * float(wp.norm()), p.shape


def test_captured_training_update():
    """ParamStore's own step in a graph: the finiteness check, the update and a workspace that nothing else grows."""
    net = train.ResNet50(DEV, num_classes=24, blocks=(1, 1, 1, 1), width=16)
    net.init(seed=3)
    step, s = train.TrainStep(net, "token_log_probs", lr=0.02, loss_scale=1024.0, optimizer="muon"), net.store
    s.grad.normal_()
    start = [t.clone() for t in (s.p32, s.vel, s.p16)]
    step.optimizer_step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (s.p32, s.vel, s.p16)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.optimizer_step()
    for bad in (False, True):
        for t, v in zip((s.p32, s.vel, s.p16), start):
            t.copy_(v)
        if bad:
            s.grad[7] = math.inf
        graph.replay()
        torch.cuda.synchronize()
        assert int(s.found_inf) == int(bad)
        assert all(torch.equal(t, v) for t, v in zip((s.p32, s.vel, s.p16), start if bad else want))
    ops.device_status()
