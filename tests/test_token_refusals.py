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
    assert lib.wa_decay_segments(1, 0, 4, 0) == 0 and lib.wa_decay_segments(1, 1, 1, 1) == 1
    f = _lib.DecayFwdArgs()
    f.q = f.k = f.v = f.o = f.log_decay = f.states = FAKE
    f.B, f.L, f.H, f.D, f.dtype = 1, 4, 2, 96, _lib.WA_BF16
    assert lib.wa_decay_fwd(ctypes.byref(f), None) == _lib.WA_ERR_ARG and b"head dim" in lib.wa_last_error()
    f.D, f.q = 64, FAKE + 2
    assert lib.wa_decay_fwd(ctypes.byref(f), None) == _lib.WA_ERR_ARG and b"aligned" in lib.wa_last_error()
    f.q, f.o_st = FAKE, 3
    assert lib.wa_decay_fwd(ctypes.byref(f), None) == _lib.WA_ERR_ARG and b"aligned" in lib.wa_last_error()
    f.o_st, f.L = 0, 0
    assert lib.wa_decay_fwd(ctypes.byref(f), None) == _lib.WA_ERR_ARG and b"nothing" in lib.wa_last_error()
    b = _lib.DecayBwdArgs()
    b.B, b.L, b.H, b.D, b.dtype = 1, 4, 2, 64, _lib.WA_F32
    assert lib.wa_decay_bwd(ctypes.byref(b), None) == _lib.WA_ERR_ARG and b"null" in lib.wa_last_error()
    b.q = b.k = b.v = b.dout = b.dk = b.dv = b.log_decay = b.states = b.workspace = FAKE
    b.dq = FAKE + 4
    assert lib.wa_decay_bwd(ctypes.byref(b), None) == _lib.WA_ERR_ARG and b"aligned" in lib.wa_last_error()
    s = _lib.DecayStepArgs()
    s.B, s.L, s.H, s.D, s.Dv, s.dtype = 1, 1, 2, 300, 64, _lib.WA_F32
    assert lib.wa_decay_step(ctypes.byref(s), None) == _lib.WA_ERR_ARG and b"1 .. 256" in lib.wa_last_error()


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _selected(which, **kw):
    a = dict(q=_bf(2, 3, 8, 64), k=_bf(2, 200, 2, 64), v=_bf(2, 200, 2, 64), sums=torch.zeros(2, 2, 4, 64), kv_len=200,
             block_size=64, topk=4, sink=1, local=1, index=torch.zeros(2, 3, 2, 4, dtype=torch.int32),
             num=torch.zeros(2, 3, 2, dtype=torch.int32), scale=None)
    a.update(kw)
    if which == "select":
        return W.select_key_blocks(a["q"], a["sums"], a["kv_len"], block_size=a["block_size"], topk=a["topk"],
                                   sink_blocks=a["sink"], local_blocks=a["local"])
    if which == "attend":
        return W.selected_attention(a["q"], a["k"], a["v"], a["index"], a["num"], a["kv_len"], block_size=a["block_size"],
                                    scale=a["scale"])
    cache = {"k": a["k"], "v": a["v"], "k_block_sums": a["sums"], "k_block_sums_block_size": a["block_size"]}
    return W.attend_selected(a["q"], cache, a["kv_len"], topk=a["topk"], sink_blocks=a["sink"], local_blocks=a["local"],
                             scale=a["scale"])


@pytest.mark.parametrize("which,bad,match", [(w, b, m) for ws, b, m in [
    ("select attend both", dict(q=_bf(3, 3, 8, 64)), "q must be"), ("select attend both", dict(q=_bf(2, 3, 7, 64)), "do not share"),
    ("select attend both", dict(q=torch.zeros(2, 3, 8, 64)), "bf16"), ("select attend both", dict(block_size=32), "block_size"),
    ("select attend both", dict(kv_len=torch.zeros(2, dtype=torch.int64)), "kv_len"),
    ("select attend both", dict(kv_len=torch.zeros(3, dtype=torch.int32)), "kv_len"),
    ("select both", dict(topk=1), "must hold"), ("select both", dict(local=0), "must hold"), ("select both", dict(sink=-1), "must hold"),
    ("select both", dict(topk=32769), "at most"), ("select both", dict(sums=torch.zeros(2, 2, 4, 64).double()), "fp32"),
    ("select both", dict(sums=torch.zeros(2, 2, 64, 4).transpose(-1, -2)), "contiguous"), ("both", dict(sums=torch.zeros(2, 2, 5, 64)), "k_block_sums"),
    ("select", dict(sums=torch.zeros(2, 2, 0, 64)), "blocks"), ("select", dict(q=_bf(2, 3, 8, 96), sums=torch.zeros(2, 2, 4, 96)), "64 or 128"),
    ("attend both", dict(v=_bf(2, 200, 1, 64)), "matching"), ("attend both", dict(k=_bf(2, 200, 2, 64).float()), "bf16"),
    ("attend both", dict(k=_bf(2, 200, 64, 2).transpose(2, 3)), "in place"), ("attend both", dict(scale=0.0), "scale"),
    ("attend", dict(index=torch.zeros(2, 3, 1, 4, dtype=torch.int32)), "index / num"), ("attend", dict(num=torch.zeros(2, 3, 2)), "int32"),
    ("attend", dict(index=torch.zeros(2, 3, 2, 0, dtype=torch.int32)), "ids a row")] for w in ws.split()])
def test_selected_attention_refuses(which, bad, match):
    with pytest.raises(ValueError, match=match):
        _selected(which, **bad)


def test_selected_attention_refuses_gradients_missing_sums_and_cpu_tensors():
    for which in ("select", "attend", "both"):
        with pytest.raises(ValueError, match="takes no gradient"):
            _selected(which, q=_bf(2, 3, 8, 64).requires_grad_(True))
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            _selected(which)
    with pytest.raises(ValueError, match="keeps no k_block_sums"):
        W.attend_selected(_bf(1, 1, 2, 64), {"k": _bf(1, 9, 2, 64), "v": _bf(1, 9, 2, 64)}, 9, topk=2)


def test_selected_entry_points_refuse():
    lib = _lib.lib()
    assert lib.wa_select_blocks(None, None) == _lib.WA_ERR_ARG and lib.wa_selected_attn(None, None) == _lib.WA_ERR_ARG
    a = _lib.SelectBlocksArgs()
    a.q = a.k_sums = a.index = a.num = a.workspace = FAKE
    a.B, a.n, a.H, a.Hk, a.D, a.block_size, a.n_blocks, a.topk, a.sink_blocks, a.local_blocks = 1, 1, 4, 3, 64, 64, 4, 4, 1, 1
    for field, bad, match in (("Hk", 3, b"heads"), ("D", 80, b"head dim"), ("block_size", 16, b"block size"), ("topk", 0, b"topk"),
                              ("n_blocks", 40000, b"blocks"), ("cap", 257, b"do not hold"), ("local_blocks", 4, b"local"),
                              ("q", FAKE + 2, b"misaligned"), ("index", None, b"null")):
        a.Hk = 2
        keep = getattr(a, field)
        setattr(a, field, bad)
        assert lib.wa_select_blocks(ctypes.byref(a), None) == _lib.WA_ERR_ARG and match in lib.wa_last_error(), field
        setattr(a, field, keep)
    a.n, a.workspace = 17, None                              # more queries than one launch scores
    assert lib.wa_select_blocks_workspace_bytes(1, 17, 2, 4) > 0
    assert lib.wa_select_blocks(ctypes.byref(a), None) == _lib.WA_ERR_ARG and b"null" in lib.wa_last_error()
    s = _lib.SelectedAttnArgs()
    s.q = s.k = s.v = s.o = s.index = s.num = FAKE
    s.B, s.n, s.cap, s.H, s.Hk, s.D, s.block_size, s.topk = 1, 1, 4096, 4, 2, 64, 64, 64
    assert lib.wa_selected_attn_workspace_bytes(1, 1, 4, 2, 64, 64, 64) > 0
    assert lib.wa_selected_attn(ctypes.byref(s), None) == _lib.WA_ERR_ARG and b"workspace" in lib.wa_last_error()
    s.k_st = 3
    assert lib.wa_selected_attn(ctypes.byref(s), None) == _lib.WA_ERR_ARG and b"aligned" in lib.wa_last_error()
