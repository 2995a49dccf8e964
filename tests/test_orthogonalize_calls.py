"""Calls of the orthogonalisation as the C ABI and the tensor-level entry points take them: what has to be true before anything reaches a GPU."""
import ctypes as C

import pytest

from nectarml_b200 import _lib

P = 4096


@pytest.fixture(autouse=True)
def _built(lib):
    pass


def test_workspace_of_small_matrices_has_room_for_either_way(lib):
    """Many steps are taken one by one on tiles, as those of larger matrices are; the coefficients, which decide, come with the call."""
    def need(shapes, steps):
        m = (_lib.Matrix * len(shapes))(*[_lib.Matrix(P, P, r, c, c, 1, c, 1) for r, c in shapes])
        n = C.c_size_t()
        assert lib.nml_orthogonalize_workspace_size(m, len(shapes), _lib.NML_MATH_3XF16, steps, C.byref(n)) == 0
        return n.value
    block, tables, partial = 65536, 65536, 64 * 64 * 8
    for steps in (2, 5, 32):   # two iterates of two blocks, three symmetric matrices of one
        assert need([(64, 147)], steps) >= 7 * block and need([(147, 64)] * 3, steps) >= 21 * block
    assert need([(64, 147)], 1) <= 4 * partial + tables   # (one step is always exact in double: three partial products and a result)
