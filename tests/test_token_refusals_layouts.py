"""Layouts that the token-by-token entry points refuse, before any launch (no GPU needed)."""
import ctypes

import pytest

from worldattention_amd import _lib

FAKE = 1 << 20


def _decay_args(cls, dtype, st):
    a = cls()
    a.B, a.L, a.H, a.D, a.dtype = 1, 4, 2, 64, dtype
    names = [n for n, _ in cls._fields_]
    for n, kind in cls._fields_:
        if kind is ctypes.c_void_p and n not in ("lengths", "initial", "dfinal", "derivs", "dinitial", "dlog_decay"):
            setattr(a, n, FAKE)
        if n.endswith("_st") and n in names:
            setattr(a, n, st)
    return a


@pytest.mark.parametrize("fn,cls,read,written", [
    ("wa_decay_fwd", _lib.DecayFwdArgs, ("q_st", "k_st", "v_st"), ("o_st",)),
    ("wa_decay_bwd", _lib.DecayBwdArgs, ("q_st", "k_st", "v_st", "d_st"), ("dq_st", "dk_st", "dv_st"))])
@pytest.mark.parametrize("dtype", [_lib.WA_BF16, _lib.WA_F32])
def test_decay_refuses_tokens_that_share_memory(fn, cls, read, written, dtype):
    """bf16 tiles end by a byte range, which would hold parts of the rows behind the last one; outputs would race."""
    for field in (*read, *written) if dtype == _lib.WA_BF16 else written:
        for st in (0, 8, 56):
            a = _decay_args(cls, dtype, 64)
            setattr(a, field, st)
            assert getattr(_lib.lib(), fn)(ctypes.byref(a), None) == _lib.WA_ERR_ARG, (field, st)
            assert b"overlapping" in _lib.lib().wa_last_error()
