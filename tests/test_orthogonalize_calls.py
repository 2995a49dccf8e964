"""Calls of the orthogonalisation as the C ABI and the tensor-level entry points take them: what has to be true before anything reaches a GPU."""
import ctypes as C

import pytest
import torch

from nectarml_b200 import _lib, ops

P = 4096


@pytest.fixture(autouse=True)
def _built(lib):
    pass


def test_workspace_of_small_matrices(lib):
    """Partial products and results in double, and room for X in fp32, whatever the length: not for tiles of 128 rows."""
    def need(shapes, steps):
        m = (_lib.Matrix * len(shapes))(*[_lib.Matrix(P, P, r, c, c, 1, c, 1) for r, c in shapes])
        n = C.c_size_t()
        assert lib.nml_orthogonalize_workspace_size(m, len(shapes), _lib.NML_MATH_3XF16, steps, C.byref(n)) == 0
        return n.value
    one, tables = 64 * 64 * 8, 65536
    for rows, cols in ((64, 147), (147, 64), (1, 1 << 24), (1 << 20, 3), (64, 1 << 20)):
        for steps in (1, 5, 32):
            x = 4 * rows * cols
            assert x <= need([(rows, cols)], steps) <= x + 25 * one + tables, (rows, cols)
            assert 3 * x <= need([(rows, cols)] * 3, steps) <= 3 * x + 75 * one + tables


INVALID, WORKSPACE = 1, 2


def _call(lib, matrices, in_dtype=0, out_dtype=0):
    c = (C.c_double * 15)(*((3.4445, -4.7750, 2.0315) * 5))
    m = (_lib.Matrix * len(matrices))(*[_lib.Matrix(*v) for v in matrices])
    return lib.nml_orthogonalize(m, len(m), in_dtype, out_dtype, _lib.NML_MATH_3XF16, 5, c, 1e-7, None, 0, None)


def _rows(inp, out, rows, cols, in_pitch=None, out_pitch=None):
    return inp, out, rows, cols, in_pitch or cols, 1, out_pitch or cols, 1


def _columns(inp, out, rows, cols, pitch=None):   # the result lies turned
    return inp, out, rows, cols, cols, 1, 1, pitch or rows


A, B, OUT = 0x100000, 0x200000, 0x300000


@pytest.mark.parametrize("first,second,want", [
    # (the missing workspace is the next refusal: these calls are taken)
    (_rows(A, OUT, 8, 8), _rows(B, OUT + 256, 8, 8), WORKSPACE),                                  # one behind the other
    (_rows(A, OUT, 8, 8), _rows(B, OUT + 252, 8, 8), INVALID),                                    # one element of the first
    (_rows(A, OUT, 8, 8), _rows(B, OUT + 224, 8, 8), INVALID),                                    # its last row
    (_rows(A, OUT, 8, 8, out_pitch=20), _rows(B, OUT + 32, 8, 12, out_pitch=20), WORKSPACE),      # columns of one buffer
    (_rows(A, OUT, 8, 8, out_pitch=20), _rows(B, OUT + 32, 8, 13, out_pitch=20), INVALID),        # the next row's first
    (_rows(A, OUT, 8, 8, out_pitch=20), _rows(B, OUT + 28, 8, 12, out_pitch=20), INVALID),
    (_rows(A, OUT, 8, 8, out_pitch=20), _rows(B, OUT + 32 + 560, 8, 13, out_pitch=20), WORKSPACE),  # only the last row of the first is in front of it
    (_rows(A, OUT, 8, 8, out_pitch=20), _rows(B, OUT + 32 + 480, 8, 13, out_pitch=20), INVALID),
    (_rows(A, OUT, 8, 8, out_pitch=40), _rows(B, OUT + 80, 8, 8, out_pitch=40), WORKSPACE),       # every other row
    (_rows(A, OUT, 8, 8, out_pitch=16), _rows(B, OUT + 32, 4, 8, out_pitch=32), WORKSPACE),       # pitches of their own
    (_rows(A, OUT, 8, 8, out_pitch=16), _rows(B, OUT + 32, 4, 8, out_pitch=31), INVALID),
    (_rows(A, OUT, 8, 8, out_pitch=16), _rows(B, OUT + 32, 1, 8), WORKSPACE),                     # a row between two
    (_rows(A, OUT, 8, 8, out_pitch=16), _rows(B, OUT + 36, 1, 8), INVALID),
    (_rows(A, OUT, 8, 8, out_pitch=16), _rows(B, OUT + 32 + 448, 1, 800), WORKSPACE),             # one long row behind the last
    (_columns(A, OUT, 8, 8, 20), _columns(B, OUT + 32, 12, 8, 20), WORKSPACE),                    # the same, turned
    (_columns(A, OUT, 8, 8, 20), _columns(B, OUT + 32, 13, 8, 20), INVALID),
    (_rows(A, OUT, 8, 8, out_pitch=20), _columns(B, OUT + 32, 12, 8, 20), WORKSPACE),
    (_rows(A, OUT, 8, 8, out_pitch=20), _columns(B, OUT + 28, 12, 8, 20), INVALID),
    (_rows(A, OUT, 8, 8), _rows(B, OUT, 8, 8), INVALID),
    # a result and its own matrix
    (_rows(A, A, 8, 8), _rows(B, B, 8, 8), WORKSPACE),
    (_rows(A, A + 32, 8, 8), _rows(B, OUT, 8, 8), INVALID),
    (_rows(A, A + 4, 8, 8), _rows(B, OUT, 8, 8), INVALID),
    (_rows(A, A + 32, 8, 8, 16, 16), _rows(B, OUT, 8, 8), WORKSPACE),
    # a result and another matrix: read before it is written
    (_rows(A, A, 8, 8), _rows(A, OUT, 8, 8), WORKSPACE),
    (_rows(A, B, 8, 8), _rows(B, A, 8, 8), WORKSPACE),
])
def test_results_that_overlap(lib, first, second, want):
    assert _call(lib, [first, second]) == want and _call(lib, [second, first]) == want
    many = [_rows(0x10000000 + 0x1000 * k, 0x20000000 + 0x1000 * k, 8, 8) for k in range(70)]
    crossed = any(x[0] in (A, B) and y[1] == x[0] and x is not y for x, y in ((first, second), (second, first)))
    # (groups of 64 run in turn, so a result over another group's matrix would be there when that one is read)
    assert _call(lib, [first] + many + [second]) == (INVALID if crossed else want)


def test_overlaps_count_bytes(lib):
    """fp16 results of fp32 matrices, and the other way round."""
    a, b = _rows(A, OUT, 8, 8), _rows(B, OUT + 128, 8, 8)
    assert _call(lib, [a, b], 0, 1) == WORKSPACE and _call(lib, [a, b], 0, 0) == INVALID
    assert _call(lib, [_rows(A, A + 128, 8, 8)], 1, 0) == WORKSPACE and _call(lib, [_rows(A, A + 128, 8, 8)], 0, 1) == INVALID


def test_overlaps_against_sets_of_bytes(lib):
    """Any two results in one buffer, whatever their places, sizes and pitches, against the bytes that they hold."""
    import random
    rng = random.Random(5)
    met = set()
    for _ in range(3000):
        two, held = [], []
        pitch = rng.randint(1, 12)
        for k in range(2):
            rows, cols = rng.randint(1, 6), rng.randint(1, 6)
            step = max(pitch if rng.random() < 0.6 else 0, rng.randint(1, 12) if rng.random() < 0.5 else 0)
            at, turned = rng.randint(0, 40), rng.random() < 0.5
            runs, length = (cols, rows) if turned else (rows, cols)
            step = max(step, length)
            strides = (1, step) if turned else (step, 1)
            two.append((A + 0x10000 * k, OUT + 4 * at, rows, cols, cols, 1) + strides)
            held.append({at + i * step + j for i in range(runs) for j in range(length)})
        want = INVALID if held[0] & held[1] else WORKSPACE
        assert _call(lib, two) == want, two
        met.add(want)
    assert met == {INVALID, WORKSPACE}


def test_one_input_many_times(lib):
    """A matrix that is read as often as one likes costs no more than the others."""
    assert _call(lib, [_rows(A, OUT + 0x1000 * k, 8, 8) for k in range(20000)]) == WORKSPACE


def test_results_have_to_match_in_number():
    x = torch.zeros(4, 6)
    for outs in ([], [x, x], iter([]), torch.zeros(2, 4, 6)):
        with pytest.raises(AssertionError, match="one tensor for each"):
            ops.orthogonalize([x], out=outs)
    with pytest.raises(TypeError, match="sequence"):
        ops.orthogonalize([x], out=3)
