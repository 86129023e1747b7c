"""What the token-by-token operators refuse, before any launch: shapes, types and devices (no GPU needed)."""
import ctypes

import pytest
import torch

from worldattention_amd import _lib
from worldattention_amd import hsa as W

FAKE = 1 << 20


def _rope(**kw):
    a = dict(q=torch.zeros(2, 5, 4, 64), positions=torch.zeros(5, 2, dtype=torch.int64),
             inv_freq=torch.ones(24, dtype=torch.float64), sections=(16, 8), k=torch.zeros(2, 5, 2, 64))
    a.update(kw)
    return W.rope_axes(a["q"], a["positions"], a["inv_freq"], a["sections"], k=a["k"])


@pytest.mark.parametrize("bad,match", [
    (dict(q=torch.zeros(5, 4, 64)), r"\[B, L, H, D\]"), (dict(k=torch.zeros(2, 4, 2, 64)), "k must hold"),
    (dict(k=torch.zeros(2, 5, 2, 64).bfloat16()), "k must hold"), (dict(sections=(16, 9)), "inv_freq must be"),
    (dict(sections=(32, 8)), "do not fit"), (dict(sections=()), "sections"), (dict(sections=(24, -1)), "sections"),
    (dict(sections=(8, 4, 4, 4, 4)), "sections"), (dict(positions=torch.zeros(5, 3, dtype=torch.int64)), "positions must be"),
    (dict(positions=torch.zeros(3, 5, 2, dtype=torch.int64)), "positions must be"),
    (dict(inv_freq=torch.ones(24, dtype=torch.float64, requires_grad=True)), "no gradient")])
def test_rope_axes_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        _rope(**bad)


def test_rope_axes_refuses_types_and_cpu_tensors():
    with pytest.raises(TypeError, match="int32 or int64"):
        _rope(positions=torch.zeros(5, 2))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        _rope()
    with pytest.raises(ValueError, match="axes 1, 2 or 3"):
        W.axis_frequencies(128, axes=4)
    inv, sections = W.axis_frequencies(128)
    assert sections == (22, 21, 21) and inv.shape == (64,) and inv.dtype == torch.float64


def test_rope_axes_entry_point_refuses():
    lib = _lib.lib()
    assert lib.wa_rope_axes(None, None) == _lib.WA_ERR_ARG
    a = _lib.RopeAxesArgs()
    a.q = a.q_out = a.positions = a.inv_freq = FAKE
    a.B, a.L, a.Hq, a.D, a.n_axes, a.dtype = 1, 4, 2, 64, 1, _lib.WA_BF16
    a.sections[0] = 33
    assert lib.wa_rope_axes(ctypes.byref(a), None) == _lib.WA_ERR_ARG and b"do not fit" in lib.wa_last_error()
    a.sections[0], a.n_axes = 16, 5
    assert lib.wa_rope_axes(ctypes.byref(a), None) == _lib.WA_ERR_ARG and b"axes" in lib.wa_last_error()
    a.n_axes, a.dtype = 1, 7
    assert lib.wa_rope_axes(ctypes.byref(a), None) == _lib.WA_ERR_ARG and b"dtype" in lib.wa_last_error()
    a.dtype, a.q_out = _lib.WA_BF16, None
    assert lib.wa_rope_axes(ctypes.byref(a), None) == _lib.WA_ERR_ARG and b"null" in lib.wa_last_error()
    a.q_out, a.L = FAKE, 0
    assert lib.wa_rope_axes(ctypes.byref(a), None) == _lib.WA_OK  # nothing to rotate
