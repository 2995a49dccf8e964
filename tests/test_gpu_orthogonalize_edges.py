"""Orthogonalised matrices at the edges of their range: many steps on matrices that have not full rank, norms far below eps,
results over matrices, long vectors."""
import math

import pytest
import torch

from nectarml_b200 import _lib, ops

from test_gpu_orthogonalize import COEF, DEV, MODES, TOL, gradient, off, plain

pytestmark = pytest.mark.gpu

POLAR = (2.0, -1.5, 0.5)   # p(1) = 1, p'(1) = 0: singular values end at 1, from above 1.0018 at most


def without_full_rank(rows, cols, kind, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device=DEV, generator=g, dtype=torch.float64)
    if kind == "duplicated rows":
        a = mk(rows, cols)
        a[rows - rows // 2:] = a[: rows // 2]
    else:
        rank = min(rows, cols, int(kind.split()[1]))
        a = mk(rows, rank) @ mk(rank, cols)
    return a.float()


KINDS = pytest.mark.parametrize("kind", ["duplicated rows", "rank 1", "rank 8"])


def check_steps(g, y, steps, coefficients, mode, largest):
    """Everything finite and bounded as the polynomial is (what rounding leaves of the missing directions grows with the steps and may end as one of the
    directions); with a polynomial that converges, the directions that the matrix has are the polar factor's.  A step is off by 8.9 u of
    itself (u = 2^-12, or with two halves 2^-23 and as much again for the product of the low halves), and over the steps that adds up at most."""
    y = y.double()
    assert bool(y.isfinite().all())
    u = 2.0 ** -12 if mode == "f16" else 2.0 ** -22
    assert float(torch.linalg.matrix_norm(y, 2)) <= largest * (1 + steps * 8.9 * u)
    if coefficients == POLAR:
        left, s, right = torch.linalg.svd(g.double(), full_matrices=False)
        n = int((s > 0.05 * s[0]).sum())
        d = left[:, :n].T @ y @ right[:n].T
        assert float((d - torch.eye(n, device=DEV)).norm()) <= steps * 8.9 * u * math.sqrt(n) * 2


@MODES
@KINDS
@pytest.mark.parametrize("rows,cols", [(64, 147), (147, 64), (20, 33)])
def test_many_steps_on_small_matrices(rows, cols, kind, mode):
    """In one chain as long as that is exact (its result is off by a rounding, and by 2^-53 times the sums' 147 terms and what directions
    that are not there take from one step to the next, 3.45^9); in several beyond."""
    g = without_full_rank(rows, cols, kind)
    for steps in (1, 5, 9):
        assert off(ops.orthogonalize(g, steps=steps, math=mode), plain(g, steps)) <= 2.0 ** -24 + 147 * 2.0 ** -53 * 3.4445 ** 9, steps
    for steps in (10, 12, 16, 20, 32):
        check_steps(g, ops.orthogonalize(g, steps=steps, math=mode), steps, COEF, mode, 1.21)
    for steps in (15, 17, 20, 32):
        check_steps(g, ops.orthogonalize(g, steps=steps, coefficients=POLAR, math=mode), steps, POLAR, mode, 1.0018)
    steep = ((60.0, 0.0, 0.0), (0.015, 0.0, 0.0), (50.0, 0.0, 0.0), (0.015, 0.0, 0.0), (60.0, 0.0, 0.0))   # two chains of steps that scale: X is rounded twice
    y = ops.orthogonalize(g * 1e-3, steps=5, coefficients=steep, eps=float(torch.tensor(float(g.norm()) * 100)), math=mode)
    assert off(y, plain(g * 1e-3, 5, steep, float(torch.tensor(float(g.norm()) * 100)))) <= 2.0 ** -22
    half = g.half()
    for steps in (5, 12):
        y = ops.orthogonalize(half, steps=steps, coefficients=POLAR, math=mode)
        assert y.dtype == torch.float16 and off(y, ops.orthogonalize(half.float(), steps=steps, coefficients=POLAR, math=mode)) <= 2.0 ** -11 + 2.0 ** -24
    many = [without_full_rank(1 + k % 64, 1 + 7 * k, kind, k) for k in range(20)]
    for x, y in zip(many, ops.orthogonalize(many, steps=25, coefficients=POLAR, math=mode)):
        check_steps(x, y, 25, POLAR, mode, 1.0018)
    ops.device_status()


@KINDS
def test_many_steps_of_the_optimizer_on_small_matrices(kind):
    shapes = [(64, 147), (33, 20), (50,), (48, 4, 3, 3)]
    grads = [without_full_rank(s[0], math.prod(s[1:]), kind, 1).reshape(s) if len(s) > 1 else torch.ones(s, device=DEV) for s in shapes]
    for steps in (12, 20, 32):
        params, momenta = [torch.zeros(s, device=DEV) for s in shapes], [torch.zeros(s, device=DEV) for s in shapes]
        ops.muon_step(params, grads, momenta, lr=1.0, momentum=0.0, nesterov=False, scaling=None, steps=steps, coefficients=POLAR)
        for p, g in zip(params, grads):
            if p.dim() > 1:
                check_steps(g.reshape(g.shape[0], -1), -p.reshape(p.shape[0], -1), steps, POLAR, "3xf16", 1.0018)
    ops.device_status()


@MODES
@pytest.mark.parametrize("rows,cols", [(20, 40), (64, 2000), (300, 200)])
def test_results_over_other_matrices(rows, cols, mode):
    """Every matrix of a call is read before a result is written: two that trade places, one that is read in place and elsewhere."""
    a, b = gradient(rows, cols, seed=31), gradient(rows, cols, seed=32)
    want = plain(a), plain(b)
    x, y = a.clone(), b.clone()
    ops.orthogonalize([x, y], out=[y, x], math=mode)
    assert off(y, want[0]) <= TOL[mode] and off(x, want[1]) <= TOL[mode]
    if rows <= 64:   # (formed elsewhere, and taken to their places as they are)
        assert all(torch.equal(p, q) for p, q in zip((y, x), ops.orthogonalize([a, b], math=mode)))
    x, y = a.clone(), torch.empty_like(a)
    ops.orthogonalize([x, x], out=[x, y], math=mode)
    assert off(x, want[0]) <= TOL[mode] and torch.equal(x, y)
    for steps in (1, 2, 20):
        x, y = a.half(), b.half()
        u, v = x.clone(), y.clone()
        ops.orthogonalize([u, v], out=[v, u], math=mode, steps=steps, coefficients=POLAR)
        for got, z in ((v, x), (u, y)):   # (a rounding to fp16 more than in its own place)
            assert off(got, plain(z, steps, POLAR)) <= TOL[mode] + 2 * 2.0 ** -11
    ops.device_status()


def test_results_in_one_buffer():
    """Side by side in the rows of one buffer, and refused where they meet."""
    a, b = gradient(90, 70, seed=33), gradient(90, 50, seed=34)
    room = torch.full((90, 130), 5.0, device=DEV)
    ops.orthogonalize([a, b], out=[room[:, 3:73], room[:, 73:123]])
    assert off(room[:, 3:73], plain(a)) <= TOL["3xf16"] and off(room[:, 73:123], plain(b)) <= TOL["3xf16"]
    assert room[:, :3].eq(5).all() and room[:, 123:].eq(5).all()
    kept = room.clone()
    batch = torch.empty(3 * 90 * 70, device=DEV)
    for mats, outs in (([a, b], [room[:, 3:73], room[:, 72:122]]), ([a[:40], a[:40].clone()], [room[:40, :70], room[39:79, :70]])):
        with pytest.raises(_lib.NectarB200Error, match="status 1"):
            ops.orthogonalize(mats, out=outs)
    with pytest.raises(_lib.NectarB200Error, match="status 1"):   # a batch whose results lie half a matrix apart
        ops.orthogonalize(torch.stack([a, a]), out=batch.as_strided((2, 90, 70), (90 * 35, 70, 1)))
    with pytest.raises(_lib.NectarB200Error, match="status 1"):
        ops.orthogonalize(room[:89, :70], out=room[1:, :70])
    assert torch.equal(room, kept)


def test_results_given_as_any_sequence():
    """A list, a tuple, the matrices of one tensor, or what is run through once."""
    gs = [gradient(30 + k, 50, seed=40 + k) for k in range(2)] + [gradient(30, 50, seed=42)]
    want = ops.orthogonalize(gs)
    mk = lambda: [torch.empty_like(g) for g in gs]
    for wrap in (list, tuple, iter, lambda o: (x for x in o)):
        outs = mk()
        got = ops.orthogonalize(gs, out=wrap(outs))
        assert all(y.data_ptr() == o.data_ptr() and torch.equal(o, w) for y, o, w in zip(got, outs, want))
    same = [gs[2], gs[2].neg()]
    out = torch.zeros(2, 30, 50, device=DEV)
    got = ops.orthogonalize(same, out=out)
    assert torch.equal(out[0], want[2]) and torch.equal(out[1], -want[2]) and got[1].data_ptr() == out[1].data_ptr()
    got = ops.orthogonalize(torch.stack(same), out=out)   # (a batch with its batch)
    assert got is out or got.data_ptr() == out.data_ptr()
    with pytest.raises(AssertionError, match="one tensor for each"):
        ops.orthogonalize(gs, out=iter(mk()[:2]))
    with pytest.raises(TypeError):
        ops.orthogonalize(gs, out=3)


@pytest.mark.parametrize("n", [16383, 16384, 16385, 2_100_003])
def test_long_vectors(n):
    """Vectors of any length, beside short ones: 2^-22 is four roundings of fp32."""
    g = torch.Generator(device=DEV).manual_seed(n)
    mk = lambda: [torch.randn(k, device=DEV, generator=g) for k in (n, 5, n, 1)]
    params, grads, momenta = mk(), mk(), mk()
    halves = [p.half() for p in params]
    want = []
    for p, q, v in zip(params, grads, momenta):
        v = 0.9 * v.double() + q.double()
        want.append((p.double() * (1 - 0.02 * 0.1) - 0.02 * (q.double() + 0.9 * v), v))
    ops.muon_step(params, grads, momenta, halves, lr=0.02, momentum=0.9, weight_decay=0.1)
    ops.device_status()
    for p, v, h, (wp, wv) in zip(params, momenta, halves, want):
        assert bool(((p.double() - wp).abs() <= 2.0 ** -22 * (1 + wp.abs())).all())
        assert bool(((v.double() - wv).abs() <= 2.0 ** -22 * (4 + wv.abs())).all()) and torch.equal(h, p.half())


def test_the_longest_vector():
    """2^31 - 1 values: an index that goes on by a block's threads must not pass 2^31 (25 GB; powers of two, so exact)."""
    n = 2 ** 31 - 1
    p, q, v = (torch.full((n,), value, device=DEV) for value in (1.0, 0.5, 0.25))
    ops.muon_step([p], [q], [v], lr=0.5, momentum=0.5, nesterov=False)
    ops.device_status()
    for part in (slice(0, 100000), slice(2 ** 30 - 100, 2 ** 30 + 100), slice(n - 100000, n)):
        assert bool((v[part] == 0.625).all()) and bool((p[part] == 1 - 0.3125).all())
    assert float(p.min()) == float(p.max()) == 0.6875


@MODES
@pytest.mark.parametrize("shapes", [[(200, 300)], [(300, 700), (90, 80)], [(700, 300)], [(512, 1100)] * 2 + [(1601, 1700)], [(40, 90), (64, 64)]], ids=str)
def test_norms_below_eps(shapes, mode):
    """X starts at |G| / (|G| + eps), however small: fp32 keeps such numbers as well as any.  While X is small a step multiplies it by a, rounded once in U, and
    rounds it once: with two halves 2^-22 each and as much for the product of the low ones, in five steps 15 x 2^-22 = 3.6e-6 beyond what
    the module's tolerance holds for norms of 1."""
    gs = [gradient(r, c, seed=50 + r) for r, c in shapes]
    for ratio in (0.3, 0.03, 1e-3, 1e-5, 1e-8, 1e-15):
        eps = float(torch.tensor(float(gs[0].norm()) * (1 / ratio - 1)))
        ys = ops.orthogonalize(gs, eps=eps, math=mode)
        for g, y in zip(gs, ys):
            want = plain(g, eps=eps)
            assert off(y, want) <= (3.6e-6 if mode == "3xf16" and ratio <= 1e-3 else TOL[mode]), (ratio, g.shape)
            assert off(ops.orthogonalize(g * 2.0 ** -60, eps=eps * 2.0 ** -60, math=mode), want) <= TOL[mode], (ratio, g.shape)   # (only their ratio counts)
    for steps, c in ((1, COEF), (3, ((3.9, -4.0, 1.2), (0.3, -0.1, 0.0), (2.0, -1.5, 0.5))), (20, POLAR)):
        for g in gs:
            eps = float(torch.tensor(float(g.norm()) * 1e5))
            assert off(ops.orthogonalize(g, steps=steps, coefficients=c, eps=eps, math=mode), plain(g, steps, c, eps)) <= TOL[mode], steps
    ops.device_status()


def test_optimizer_step_with_norms_below_eps():
    shapes = [(130, 70), (300, 700), (64, 3, 7, 7)]
    grads = [1e-13 * gradient(s[0], math.prod(s[1:]), seed=60 + k).reshape(s) for k, s in enumerate(shapes)]
    params, momenta = [torch.zeros(s, device=DEV) for s in shapes], [torch.zeros(s, device=DEV) for s in shapes]
    ops.muon_step(params, grads, momenta, lr=1.0, momentum=0.0, scaling=None)
    for p, g in zip(params, grads):
        assert off(-p.reshape(p.shape[0], -1), plain(g.reshape(p.shape[0], -1))) <= 3.6e-6
