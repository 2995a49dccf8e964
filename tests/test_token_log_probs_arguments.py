"""What the token log-probability calls refuse before anything reaches a GPU: through the tensor-level entry points, which raise, and
through the C ABI, which returns a status."""
import pytest
import torch

from nectarml_b200 import _lib, ops


@pytest.fixture(autouse=True)
def _built(lib):
    pass


def test_tensors_in_the_wrong_place_or_type():
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(_lib.NectarB200Error, match="CUDA device"):
        ops.token_log_probs(x, t)
    with pytest.raises(_lib.NectarB200Error, match="float32 and float16"):
        ops.token_log_probs(x.double(), t)
    with pytest.raises(TypeError, match="logits"):
        ops.token_log_probs(None, t)
    with pytest.raises(_lib.NectarB200Error, match="CUDA device"):
        ops.token_log_probs_backward(x, t, torch.zeros(3, 2), None, torch.zeros(3))


# (pointers are never read: every call is refused on the host)
P, INVALID, UNSUPPORTED = 4096, _lib.NML_OK + 1, 4


def _forward(lib, logits=P, dtype=0, rows=4, vocab=100, pitch=100, targets=P, top=0, lp=P, h=P, stats=P, top_lp=P, top_i=P):
    return lib.nml_token_log_probs(logits, dtype, rows, vocab, pitch, targets, top, lp, h, stats, top_lp, top_i, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(targets=None), dict(lp=None), dict(h=None), dict(stats=None), dict(dtype=2), dict(dtype=-1), dict(rows=0),
    dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(pitch=99), dict(top=-1), dict(top=101), dict(top=3, top_lp=None),
    dict(top=3, top_i=None), dict(logits=P + 2), dict(logits=P + 1, dtype=1), dict(targets=P + 4), dict(lp=P + 2), dict(stats=P + 1),
    dict(top=3, top_i=P + 4)], ids=str)
def test_forward_arguments(lib, bad):
    assert _forward(lib, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(top=33), dict(top=1, vocab=1_100_000, pitch=1_100_000), dict(top=1, vocab=2_100_000, pitch=2_100_000, dtype=1)], ids=str)
def test_forward_beyond_what_the_kernels_cover(lib, bad):
    assert _forward(lib, **bad) == UNSUPPORTED


def _backward(lib, logits=P, dtype=0, rows=4, vocab=100, pitch=100, targets=P, stats=P, h=P, dlp=P, dh=P, out=P, d_pitch=100):
    return lib.nml_token_log_probs_backward(logits, dtype, rows, vocab, pitch, targets, stats, h, dlp, dh, out, d_pitch, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(targets=None), dict(stats=None), dict(dlp=None), dict(out=None), dict(h=None), dict(dtype=3), dict(rows=0),
    dict(vocab=0), dict(pitch=99), dict(d_pitch=99), dict(out=P + 2), dict(targets=P + 4), dict(dlp=P + 2), dict(dh=P + 3), dict(d_pitch=101)], ids=str)
def test_backward_arguments(lib, bad):
    assert _backward(lib, **bad) == INVALID
