"""Layouts that the token-by-token entry points refuse, before any launch (no GPU needed)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from worldattention_amd import _lib
from worldattention_amd import hsa as W

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


def _state(b, h, sb, sh):
    return torch.zeros(4096).as_strided((b, h, 4, 8), (sb, sh, 8, 1))


def _step(state):
    b, h = state.shape[:2]
    x = [torch.zeros(b, 1, h, d) for d in (4, 4, 8)]
    return W.decay_linear_step(*x, torch.zeros(h), state)


@pytest.mark.parametrize("b,h,sb,sh", [(2, 1, 31, 32), (1, 2, 64, 16), (2, 3, 64, 32), (2, 2, 32, 32), (3, 2, 32, 64), (2, 2, 70, 100),
                                       (2, 2, 0, 32), (4, 1, 1, 0), (3, 3, 33, 49)])
def test_decay_step_refuses_states_that_share_memory(b, h, sb, sh):
    """Two workgroups would update the same elements."""
    with pytest.raises(ValueError, match="memory of its own"):
        _step(_state(b, h, sb, sh))


@pytest.mark.parametrize("b,h,sb,sh", [(2, 3, 96, 32), (2, 3, 32, 64), (1, 1, 0, 0), (1, 3, 0, 32), (3, 1, 40, 7), (2, 3, 48, 32 + 64), (2, 2, 40, 72),
                                       (2, 3, 100, 66)])
def test_decay_step_takes_states_apart(b, h, sb, sh):
    """Past the layouts' check, to the one for a GPU."""
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        _step(_state(b, h, sb, sh))


def test_decay_step_entry_point_refuses_one_state_for_two():
    a = _lib.DecayStepArgs()
    a.q = a.k = a.v = a.o = a.log_decay = a.state = FAKE
    a.B, a.L, a.H, a.D, a.Dv, a.dtype = 2, 1, 3, 64, 64, _lib.WA_F32
    for sb, sh in ((0, 4096), (4096, 0), (4096, 4096)):
        a.st_sb, a.st_sh = sb, sh
        assert _lib.lib().wa_decay_step(ctypes.byref(a), None) == _lib.WA_ERR_ARG and b"share memory" in _lib.lib().wa_last_error()


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-50, -1e-46, 7e-46])
def test_selected_attention_refuses_a_scale_of_zero_in_fp32(scale):
    """The library reads 0 as the default, so a scale that rounds to 0 would have been taken for D ** -0.5."""
    q, k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 64, 2, 64, dtype=torch.bfloat16)
    index, num = torch.zeros(1, 1, 2, 1, dtype=torch.int32), torch.ones(1, 1, 2, dtype=torch.int32)
    cache = {"k": k, "v": k, "k_block_sums": torch.zeros(1, 2, 1, 64), "k_block_sums_block_size": 64}
    with pytest.raises(ValueError, match="scale"):
        W.selected_attention(q, k, k, index, num, 64, block_size=64, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        W.attend_selected(q, cache, 64, topk=2, scale=scale)
    with pytest.raises(RuntimeError, match="ROCm GPU"):     # the smallest that fp32 holds
        W.selected_attention(q, k, k, index, num, 64, block_size=64, scale=2.0 ** -149)


def _calls():
    """Each operator on CPU tensors, by the argument that a tangent rides on."""
    def f(*shape):
        return torch.zeros(*shape)

    def b(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16)

    pos, inv = torch.zeros(5, 1, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    x, state, g = f(1, 5, 2, 64), f(1, 2, 64, 64), f(2)
    index, num = torch.zeros(1, 1, 2, 1, dtype=torch.int32), torch.ones(1, 1, 2, dtype=torch.int32)
    kv, sums = b(1, 64, 2, 64), f(1, 2, 1, 64)
    cache = {"k": kv, "v": kv, "k_block_sums": sums, "k_block_sums_block_size": 64}
    yield "rope_axes", x, lambda t: W.rope_axes(t, pos, inv, (32,))
    yield "rope_axes k", x, lambda t: W.rope_axes(x, pos, inv, (32,), k=t)
    yield "rope_axes inv_freq", inv, lambda t: W.rope_axes(x, pos, t, (32,))
    yield "decay v", x, lambda t: W.decay_linear_attention(x, x, t, g)
    yield "decay log_decay", g, lambda t: W.decay_linear_attention(x, x, x, t)
    yield "decay initial_state", state, lambda t: W.decay_linear_attention(x, x, x, g, initial_state=t)
    yield "step q", x, lambda t: W.decay_linear_step(t, x, x, g, state)
    yield "step state", state, lambda t: W.decay_linear_step(x, x, x, g, t)
    yield "select q", b(1, 1, 2, 64), lambda t: W.select_key_blocks(t, sums, 64, block_size=64, topk=2)
    yield "selected_attention v", kv, lambda t: W.selected_attention(b(1, 1, 2, 64), kv, t, index, num, 64, block_size=64)
    yield "attend_selected sums", sums, lambda t: W.attend_selected(b(1, 1, 2, 64), dict(cache, k_block_sums=t), 64, topk=2)


@pytest.mark.parametrize("name,t,call", list(_calls()), ids=[c[0] for c in _calls()])
def test_tangents_are_refused(name, t, call):
    """A dual tensor would lose its tangent: the kernels read the primal values alone."""
    with forward_ad.dual_level():
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled), pytest.raises(ValueError, match="forward-mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            with torch.set_grad_enabled(enabled), pytest.raises(RuntimeError, match="ROCm GPU"):
                call(t)
