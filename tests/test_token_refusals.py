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


def _decay(step=False, **kw):
    a = dict(q=torch.zeros(2, 5, 4, 64), k=torch.zeros(2, 5, 4, 64), v=torch.zeros(2, 5, 4, 32),
             log_decay=torch.zeros(4), state=torch.zeros(2, 4, 64, 32), lengths=None)
    a.update(kw)
    if step:
        return W.decay_linear_step(a["q"], a["k"], a["v"], a["log_decay"], a["state"])
    return W.decay_linear_attention(a["q"], a["k"], a["v"], a["log_decay"], initial_state=a["state"], lengths=a["lengths"])


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("bad,match", [
    (dict(k=torch.zeros(2, 4, 4, 64)), "must be"), (dict(v=torch.zeros(2, 5, 3, 32)), "must be"),
    (dict(q=torch.zeros(2, 5, 4, 64).bfloat16()), "one dtype"), (dict(log_decay=torch.zeros(3)), "log_decay"),
    (dict(log_decay=torch.zeros(4).double()), "log_decay"), (dict(state=torch.zeros(2, 4, 32, 64)), "state must be"),
    (dict(state=torch.zeros(2, 4, 64, 32).bfloat16()), "state must be")])
def test_decay_refuses(step, bad, match):
    with pytest.raises(ValueError, match=match):
        _decay(step, **bad)


def test_decay_refuses_sizes_lengths_gradients_and_cpu_tensors():
    with pytest.raises(ValueError, match="at most 128"):
        _decay(q=torch.zeros(2, 5, 4, 160), k=torch.zeros(2, 5, 4, 160), state=None)
    for bad in (torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="lengths"):
            _decay(lengths=bad)
    with pytest.raises(ValueError, match="takes no gradient"):
        _decay(True, q=torch.zeros(2, 5, 4, 64, requires_grad=True))
    with pytest.raises(ValueError, match="contiguous"):
        _decay(True, state=torch.zeros(2, 4, 32, 64).transpose(-1, -2))
    with pytest.raises(ValueError, match="memory of its own"):
        _decay(True, state=torch.zeros(1, 4, 64, 32).expand(2, -1, -1, -1))
    for step in (False, True):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            _decay(step)


def test_decay_entry_points_refuse():
    lib = _lib.lib()
    for fn in (lib.wa_decay_fwd, lib.wa_decay_bwd, lib.wa_decay_step):
        assert fn(None, None) == _lib.WA_ERR_ARG
    assert lib.wa_decay_segments(1, 0, 4) == 0 and lib.wa_decay_segments(1, 1, 1) == 1
    f = _lib.DecayFwdArgs()
    f.q = f.k = f.v = f.o = f.log_decay = f.states = FAKE
    f.B, f.L, f.H, f.D, f.dtype = 1, 4, 2, 96, _lib.WA_BF16
    assert lib.wa_decay_fwd(ctypes.byref(f), None) == _lib.WA_ERR_ARG and b"head dim" in lib.wa_last_error()
    f.D, f.q = 64, FAKE + 2
    assert lib.wa_decay_fwd(ctypes.byref(f), None) == _lib.WA_ERR_ARG and b"aligned" in lib.wa_last_error()
    f.q, f.L = FAKE, 0
    assert lib.wa_decay_fwd(ctypes.byref(f), None) == _lib.WA_ERR_ARG and b"nothing" in lib.wa_last_error()
    b = _lib.DecayBwdArgs()
    b.B, b.L, b.H, b.D, b.dtype = 1, 4, 2, 64, _lib.WA_F32
    assert lib.wa_decay_bwd(ctypes.byref(b), None) == _lib.WA_ERR_ARG and b"null" in lib.wa_last_error()
    s = _lib.DecayStepArgs()
    s.B, s.L, s.H, s.D, s.Dv, s.dtype = 1, 1, 2, 300, 64, _lib.WA_F32
    assert lib.wa_decay_step(ctypes.byref(s), None) == _lib.WA_ERR_ARG and b"1 .. 256" in lib.wa_last_error()
