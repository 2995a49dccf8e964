"""Where the gradient of token log probabilities may be written."""
import pytest

from nectarml_b200 import _lib

X, OUT, T, STATS, H, D, DH, INVALID = 0x100000, 0x200000, 0x300000, 0x310000, 0x320000, 0x330000, 0x340000, 1


@pytest.fixture(autouse=True)
def _built(lib):
    pass


# (pointers are never read: every call is refused on the host; calls that are taken are in the GPU's tests)
@pytest.mark.parametrize("bad", [
    dict(out=X + 4), dict(out=X - 4), dict(out=X + 400), dict(out=X - 1196), dict(out=X, d_pitch=101), dict(out=X + 404, pitch=101, d_pitch=101),
    dict(out=X + 40, pitch=109, d_pitch=109), dict(out=X + 36 + 436, pitch=209, d_pitch=209), dict(out=T - 4), dict(out=STATS - 1596), dict(out=D + 12), dict(out=DH + 12), dict(out=H + 12), dict(out=STATS + 28),
    dict(out=T + 28)], ids=str)
def test_results_over_what_is_read(lib, bad):
    a = dict(dict(out=OUT, pitch=100, d_pitch=100), **bad)
    assert lib.nml_token_log_probs_backward(X, 0, 4, 100, a["pitch"], T, STATS, H, D, DH, a["out"], a["d_pitch"], None) == INVALID
