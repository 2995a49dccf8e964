"""What the orthogonalisation and the optimizer step on it refuse before anything reaches a GPU, and the size of their workspace."""
import ctypes as C

import pytest
import torch

from nectarml_b200 import _lib, ops, train

P, INVALID, WORKSPACE, UNSUPPORTED = 4096, 1, 2, 4
COEF = (3.4445, -4.7750, 2.0315)


@pytest.fixture(autouse=True)
def _built(lib):
    pass


def _need(lib, shapes, math=_lib.NML_MATH_3XF16, steps=5):
    m = (_lib.Matrix * len(shapes))(*[_lib.Matrix(P, P, r, c, c, 1, c, 1) for r, c in shapes])
    n = C.c_size_t()
    return lib.nml_orthogonalize_workspace_size(m, len(shapes), math, steps, C.byref(n)), n.value


def test_workspace_size(lib):
    assert _need(lib, []) == (0, 0)
    block, tables = 65536, 65536
    rc, one = _need(lib, [(128, 256)])          # two iterates of two blocks, three symmetric matrices of one
    assert rc == 0 and 7 * block <= one <= 7 * block + tables
    assert _need(lib, [(256, 128)])[1] == one   # turned wide
    assert _need(lib, [(128, 256)], _lib.NML_MATH_F16)[1] == one + 5 * block   # a block of the identity for each step
    chained = _need(lib, [(256, 512)])[1]       # two iterates of eight blocks, seven symmetric matrices of three
    assert 37 * block <= chained <= 37 * block + tables
    assert _need(lib, [(256, 512)], steps=1)[1] == chained - 12 * block
    group = _need(lib, [(128, 256)] * 64)[1]
    assert group >= 64 * 7 * block and _need(lib, [(128, 256)] * 1000)[1] == group   # one group at a time
    assert _need(lib, [(1, (1 << 24) + 1)])[0] == INVALID
    for bad in ([(0, 4)], [(4, 0)], [(-1, 4)], [(1 << 30, 1 << 30)]):
        assert _need(lib, bad)[0] == INVALID
    for steps in (0, 33, -1):
        assert _need(lib, [(4, 4)], steps=steps)[0] == INVALID
    assert _need(lib, [(4, 4)], math=_lib.NML_MATH_3XTF32)[0] == INVALID


def _call(lib, inp=P, out=P, rows=4, cols=6, in_row=6, in_col=1, out_row=6, out_col=1, in_dtype=0, out_dtype=0, math=_lib.NML_MATH_3XF16,
          steps=5, coef=COEF * 5, eps=1e-7, ws=None, ws_bytes=0):
    m = _lib.Matrix(inp, out, rows, cols, in_row, in_col, out_row, out_col)
    c = None if coef is None else (C.c_double * len(coef))(*coef)
    return lib.nml_orthogonalize(C.byref(m), 1, in_dtype, out_dtype, math, steps, c, eps, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(inp=None), dict(out=None), dict(inp=P + 2), dict(out=P + 1, out_dtype=1), dict(in_dtype=2), dict(out_dtype=-1), dict(coef=None),
    dict(eps=-1.0), dict(eps=float("nan")), dict(in_row=5), dict(in_col=2), dict(in_row=1, in_col=3), dict(out_row=5), dict(out_row=12, out_col=2),
    dict(out_row=0)], ids=str)
def test_orthogonalize_arguments(lib, bad):
    assert _call(lib, **bad) == INVALID


def test_coefficients_that_diverge(lib):
    assert _call(lib, coef=(9.0, 5.0, 5.0) * 5) == UNSUPPORTED
    assert _call(lib, coef=(float("nan"), 0.0, 0.0) * 5) == UNSUPPORTED
    assert _call(lib, coef=(2e3, 0.0, 0.0), steps=1) == UNSUPPORTED


def test_missing_workspace(lib):
    assert _call(lib) == WORKSPACE and _call(lib, ws=P, ws_bytes=1000) == WORKSPACE


def _muon(lib, params, steps=5, coef=COEF * 5, eps=1e-7, found=None):
    p = (_lib.MuonParam * len(params))(*[_lib.MuonParam(*v) for v in params])
    c = None if coef is None else (C.c_double * len(coef))(*coef)
    return lib.nml_muon_step(p, len(params), _lib.NML_MATH_3XF16, steps, c, eps, 0.1, 0.9, 1, 0.0, 1.0, found, None, 0, None)


def test_muon_arguments(lib):
    good = (0x10000, 0x20000, 0x30000, 0x40000, 8, 8, 1.0)
    assert _muon(lib, [good]) == WORKSPACE        # (that is: nothing else is wrong with it)
    for at, value in ((0, None), (1, None), (2, None), (0, 0x10002), (1, 0x20001), (2, 0x30002), (3, 0x40001), (4, -1), (5, 0), (5, -2)):
        assert _muon(lib, [good[:at] + (value,) + good[at + 1:]]) == INVALID, (at, value)
    assert _muon(lib, [good], coef=None) == INVALID and _muon(lib, [good], eps=-1.0) == INVALID and _muon(lib, [good], found=2) == INVALID
    assert _muon(lib, [good], coef=(9.0, 5.0, 5.0) * 5) == UNSUPPORTED


def test_muon_refuses_a_parameter_listed_twice(lib):
    good = (0x10000, 0x20000, 0x30000, 0x40000, 8, 8, 1.0)
    assert _muon(lib, [good, good]) == INVALID
    beside = (0x10100, 0x21000, 0x31000, 0x41000, 8, 8, 1.0)     # the next 256 bytes: apart
    assert _muon(lib, [good, beside]) == WORKSPACE
    assert _muon(lib, [good, (0x100fc,) + beside[1:]]) == INVALID  # one element of the first
    assert _muon(lib, [good, beside[:2] + (0x30000,) + beside[3:]]) == INVALID   # momentum shared
    assert _muon(lib, [good, beside[:3] + (0x40000,) + beside[4:]]) == INVALID   # half copy shared
    assert _muon(lib, [(0x10000, 0x20000, 0x10000, None, 0, 8, 1.0)]) == INVALID  # momentum is the parameter


def test_muon_refuses_gradients_among_what_it_writes(lib):
    good = (0x10000, 0x20000, 0x30000, 0x40000, 8, 8, 1.0)
    beside = (0x10100, 0x20000, 0x31000, 0x41000, 8, 8, 1.0)
    assert _muon(lib, [good, beside]) == WORKSPACE                 # one gradient for two parameters
    for at in (0x10000, 0x100fc, 0x0ff04, 0x30000, 0x4007c, 0x310fc):
        assert _muon(lib, [good, beside[:1] + (at,) + beside[2:]]) == INVALID, hex(at)
    for at in (0x0ff00, 0x10200, 0x40080):                         # ends where one begins, begins where one ends
        assert _muon(lib, [good, beside[:1] + (at,) + beside[2:]]) == WORKSPACE, hex(at)


def test_results_in_places_of_their_own(lib):
    def call(*m):
        c = (C.c_double * 15)(*(COEF * 5))
        return lib.nml_orthogonalize((_lib.Matrix * len(m))(*m), len(m), 0, 0, _lib.NML_MATH_3XF16, 5, c, 1e-7, None, 0, None)
    a = _lib.Matrix(P, P, 4, 4, 4, 1, 4, 1)
    assert call(a) == WORKSPACE
    assert call(a, _lib.Matrix(P, 2 * P, 4, 4, 4, 1, 4, 1)) == WORKSPACE       # one matrix twice, two results
    assert call(a, _lib.Matrix(2 * P, P, 4, 4, 4, 1, 4, 1)) == INVALID
    assert call(_lib.Matrix(P, P, 4, 4, 4, 1, 1, 4)) == INVALID                # in place, turned
    assert _call(lib, out_dtype=1) == INVALID                                  # in place, of another type


def test_every_store_has_a_workspace_of_its_own():
    """A captured step's stays where it is when another net's step needs a larger one."""
    assert train.ParamStore("cpu")._muon_ws is not train.ParamStore("cpu")._muon_ws


def test_tensor_level_refusals():
    e = _lib.NectarB200Error
    x = torch.zeros(4, 6)
    with pytest.raises(e, match="CUDA device"):
        ops.orthogonalize(x)
    with pytest.raises(e, match="float32 and float16"):
        ops.orthogonalize(x.double())
    with pytest.raises(e, match="math"):
        ops.orthogonalize(x, math="tf32")
    for c in ((1.0, 2.0), ((1.0, 2.0, 3.0),) * 4, ((1.0, 2.0),) * 5):
        with pytest.raises(e, match="coefficients"):
            ops.orthogonalize(x, coefficients=c)
    assert ops.orthogonalize([]) == []
    with pytest.raises(e, match="math"):
        ops.muon_step([x], [x], [x], lr=0.1, math="f64")
    with pytest.raises(e, match="scaling"):
        ops.muon_step([x], [x], [x], lr=0.1, scaling="none")
    with pytest.raises(AssertionError, match="one gradient"):
        ops.muon_step([x], [], [x], lr=0.1)
    with pytest.raises(AssertionError, match="float32"):
        ops.muon_step([x.half()], [x], [x], lr=0.1)
    with pytest.raises(e, match="CUDA device"):
        ops.muon_step([x], [x], [x], lr=0.1)
    with pytest.raises(ValueError, match="optimizer"):
        train.TrainStep(None, "l1", optimizer="adam")
