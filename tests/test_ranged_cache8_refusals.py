"""What ranged attention and the 8-bit cache refuse, before any launch (no GPU needed)."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from worldattention_amd import _lib
from worldattention_amd import hsa as W

FAKE = 1 << 20
I32 = torch.int32


def zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


# ---------------------------------------------------------------------------------------------
# key_ranges
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes", [(-1, 4, 4), (1, -1, 4), (1, 4, -1), (1.5, 4, 4), (True, 4, 4), (1, (1 << 30) + 1, 4), (1, 4, (1 << 30) + 1)])
def test_key_ranges_refuses_sizes(sizes):
    with pytest.raises(ValueError):
        W.key_ranges(*sizes)


@pytest.mark.parametrize("rules", [
    dict(chunk=0), dict(chunk=2.5), dict(chunk=4, causal=False), dict(window=0), dict(window=-3), dict(sink=-1), dict(prefix=-1),
    dict(documents=zeros(3, dtype=I32), lengths=zeros(2, dtype=I32)),
    dict(prefix=zeros(3, dtype=I32)), dict(prefix=zeros(2, dtype=torch.int64)),
    dict(kv_len=zeros(2, dtype=torch.int64)), dict(kv_len=zeros(1, dtype=I32)),
    dict(lengths=zeros(2, dtype=torch.int64)), dict(lengths=zeros(2, 1, dtype=I32)),
    dict(documents=zeros(1, dtype=I32)), dict(documents=zeros(3, dtype=torch.int64)), dict(documents=zeros(3, 4, dtype=I32)),
    dict(documents=zeros(1, 2, 4, dtype=I32)),
    dict(given=zeros(2, 8, 2, dtype=I32)), dict(given=zeros(2, 7, 4, dtype=I32)), dict(given=zeros(3, 8, 4, dtype=I32)),
    dict(given=zeros(2, 8, 4, dtype=torch.int64)), dict(given=zeros(8, 4, dtype=I32)),
])
def test_key_ranges_refuses_rules(rules):
    with pytest.raises(ValueError):
        W.key_ranges(2, 8, 8, **rules)


@pytest.mark.parametrize("where", [dict(kv_len=zeros(2, dtype=I32)), dict(prefix=zeros(2, dtype=I32)), dict(lengths=zeros(2, dtype=I32)),
                                   dict(documents=zeros(4, dtype=I32)), dict(given=zeros(1, 8, 4, dtype=I32)), dict(device="cpu")])
def test_key_ranges_has_no_cpu_path(where):
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        W.key_ranges(2, 8, 8, **where)


# ---------------------------------------------------------------------------------------------
# ranged_attention
# ---------------------------------------------------------------------------------------------
def ranges(b=2, n=8, m=8):
    return W.KeyRanges(zeros(b, n, 4, dtype=I32), zeros(b, -(-n // 64), 12, dtype=I32),
                       zeros(b, -(-n // 128) - (-m // 128) + 1, dtype=I32), n, m)


def attention(q=(2, 8, 4, 64), k=(2, 8, 2, 64), v=None, dtypes=(torch.bfloat16,) * 3, r=None, **options):
    q, k, v = (zeros(*s, dtype=t) for s, t in zip((q, k, v or k), dtypes))
    return W.ranged_attention(q, k, v, r or ranges(), **options)


@pytest.mark.parametrize("case", [
    dict(q=(8, 4, 64)), dict(k=(8, 2, 64)), dict(k=(1, 8, 2, 64)), dict(k=(2, 8, 2, 128)), dict(v=(2, 8, 1, 64)), dict(v=(2, 9, 2, 64)),
    dict(k=(2, 8, 3, 64)), dict(k=(2, 8, 8, 64)), dict(k=(2, 8, 0, 64)), dict(q=(2, 8, 4, 192), k=(2, 8, 2, 192)),
    dict(dtypes=(torch.float32,) * 3), dict(dtypes=(torch.float16,) * 3), dict(dtypes=(torch.bfloat16, torch.bfloat16, torch.float32)),
    dict(q=(2, 9, 4, 64)), dict(k=(2, 9, 2, 64)), dict(r=ranges(3)), dict(r=ranges(2, 8, 9)),
])
def test_ranged_attention_refuses_shapes_and_types(case):
    with pytest.raises(ValueError):
        attention(**case)


@pytest.mark.parametrize("field,bad", [
    ("rows", zeros(2, 8, 3, dtype=I32)), ("rows", zeros(2, 8, 4, dtype=torch.int64)), ("rows", zeros(2, 4, 8, dtype=I32).transpose(1, 2)),
    ("tiles", zeros(1, 1, 12, dtype=I32)), ("tiles", zeros(2, 2, 12, dtype=I32)), ("order", zeros(2, 2, dtype=I32)),
    ("order", zeros(1, 3, dtype=I32)), ("order", zeros(2, 3)),
])
def test_ranged_attention_refuses_other_ranges(field, bad):
    with pytest.raises(ValueError):
        attention(r=ranges()._replace(**{field: bad}))


SCORES = [dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e-60), dict(scale=1e39),
          dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf), dict(cap=1e-7), dict(cap=2e6), dict(cap=5.0, scale=1e31),
          dict(slopes=torch.zeros(3)), dict(slopes=torch.zeros(4, dtype=torch.float64)), dict(slopes=torch.zeros(4, 1))]


@pytest.mark.parametrize("options", SCORES)
def test_ranged_attention_refuses_scores(options):
    with pytest.raises(ValueError):
        attention(**options)


def test_ranged_attention_has_no_cpu_path_and_no_forward_mode():
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        attention()
    with forward_ad.dual_level():
        q = forward_ad.make_dual(zeros(2, 8, 4, 64), zeros(2, 8, 4, 64))
        k = zeros(2, 8, 2, 64)
        with pytest.raises(ValueError, match="forward-mode"):
            W.ranged_attention(q, k, k, ranges())


# ---------------------------------------------------------------------------------------------
# The 8-bit cache
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("args,options", [
    ((2, 64, 1, 96), {}), ((2, 64, 1, 256), {}), ((0, 64, 1, 64), {}), ((2, 0, 1, 64), {}), ((2, 64, 0, 64), {}), ((2, 64.5, 1, 64), {}),
    ((2, 64, 1, 64), dict(block_size=32)), ((2, 64, 1, 64), dict(block_size=256)), ((2, 64, 1, 64), dict(dtype=torch.uint8)),
    ((2, 64, 1, 64), dict(dtype=torch.bfloat16)), ((2, 64, 1, 64), dict(dtype=torch.float8_e5m2)),
])
def test_new_cache_refuses(args, options):
    with pytest.raises(ValueError):
        W.new_cache_8bit(*args, device="cpu", **options)


def cache(b=2, cap=200, hk=2, d=64, **options):
    return W.new_cache_8bit(b, cap, hk, d, device="cpu", **options)


def broken():
    def with_(name, make):
        c = cache()
        c[name] = make(c[name])
        return c

    for name in ("k", "v", "k_scale", "v_scale", "k_block_sums_block_size"):
        c = cache()
        del c[name]
        yield f"no {name}", c
    yield "codes", with_("k", lambda t: t.view(torch.uint8))
    yield "bf16", with_("k", lambda t: t.to(torch.bfloat16))
    yield "two codes", with_("v", lambda t: t.view(torch.uint8).view(torch.float8_e4m3fn))
    yield "shape", with_("v", lambda t: t[:, :100])
    yield "dim", {**cache(), "k": torch.zeros(2, 200, 2, 32, dtype=torch.int8), "v": torch.zeros(2, 200, 2, 32, dtype=torch.int8)}
    yield "blocks", with_("k_scale", lambda t: t[..., :2])
    yield "scale type", with_("v_scale", lambda t: t.double())
    yield "scale heads", with_("v_scale", lambda t: torch.zeros(2, 1, 4))
    yield "sums", with_("k_block_sums", lambda t: t[..., :32])
    yield "sums type", with_("k_block_sums", lambda t: t.bfloat16())
    yield "block size", {**cache(), "k_block_sums_block_size": 48}
    yield "other block size", {**cache(), "k_block_sums_block_size": 128}
    yield "strided codes", with_("k", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    yield "strided scales", with_("k_scale", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    yield "address", with_("k", lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype)[1:].view(t.shape))


@pytest.mark.parametrize("c", [pytest.param(c, id=name.replace(" ", "_")) for name, c in broken()])
def test_operators_refuse_other_caches(c):
    new, q = zeros(2, 1, 2, 64), zeros(2, 1, 4, 64)
    for call in (lambda: W.kv_append_8bit(c, new, new, 0), lambda: W.kv_read_8bit(c, 0, 4), lambda: W.attend_8bit(q, c, 10)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("k,v,start,lengths", [
    ((2, 3, 2, 64), (2, 4, 2, 64), 0, None), ((1, 3, 2, 64), None, 0, None), ((2, 3, 1, 64), None, 0, None), ((2, 3, 2, 128), None, 0, None),
    ((2, 2, 64), None, 0, None), ((2, 201, 2, 64), None, 0, None), ((2, 3, 2, 64), None, 198, None), ((2, 3, 2, 64), None, -1, None),
    ((2, 3, 2, 64), None, zeros(3, dtype=I32), None), ((2, 3, 2, 64), None, zeros(2, dtype=torch.int64), None),
    ((2, 3, 2, 64), None, 0, zeros(3, dtype=I32)), ((2, 3, 2, 64), None, 0, zeros(2, dtype=torch.int64)),
])
def test_append_refuses(k, v, start, lengths):
    with pytest.raises(ValueError):
        W.kv_append_8bit(cache(), zeros(*k), zeros(*(v or k)), start, lengths=lengths)


def test_append_refuses_types_gradients_and_cpu():
    new = zeros(2, 1, 2, 64)
    with pytest.raises(ValueError):
        W.kv_append_8bit(cache(), new, new.float(), 0)
    with pytest.raises(ValueError, match="no gradient"):
        W.kv_append_8bit(cache(), new.clone().requires_grad_(), new, 0)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        W.kv_append_8bit(cache(), new, new, 0)


@pytest.mark.parametrize("start,n,options", [(0, -1, {}), (0, 1.5, {}), (zeros(3, dtype=I32), 1, {}), (zeros(2, dtype=torch.int64), 1, {}),
                                             (0, 4, dict(dtype=torch.float16)), (0, 4, dict(dtype=torch.int8))])
def test_read_refuses(start, n, options):
    with pytest.raises(ValueError):
        W.kv_read_8bit(cache(), start, n, **options)


@pytest.mark.parametrize("far", [1 << 63, (1 << 64) + 5, -(1 << 64)])
def test_numbers_that_64_bits_do_not_hold(far):
    for call in (lambda: W.kv_read_8bit(cache(), far, 4), lambda: W.attend_8bit(zeros(2, 1, 4, 64), cache(), far),
                 lambda: W.kv_append_8bit(cache(), zeros(2, 1, 2, 64), zeros(2, 1, 2, 64), far), lambda: W.key_ranges(1, 4, 4, kv_len=far),
                 lambda: W.key_ranges(1, 4, 4, prefix=abs(far)), lambda: W.key_ranges(1, 4, 4, window=abs(far)),
                 lambda: W.attend_8bit(zeros(2, 1, 4, 64), cache(), 9, window=abs(far))):
        with pytest.raises(ValueError):
            call()


def lists(b=2, n=1, hk=2, topk=3, dtype=I32):
    return W.BlockSelection(torch.zeros(b, n, hk, topk, dtype=dtype), torch.zeros(b, n, hk, dtype=dtype))


@pytest.mark.parametrize("options", SCORES + [
    dict(window=0), dict(window=-1), dict(window=1.5), dict(sink=4), dict(sink=-1, window=4), dict(chosen=lists(), window=8),
    dict(chosen=lists(), sink=1), dict(chosen=lists(b=1)), dict(chosen=lists(n=2)), dict(chosen=lists(hk=4)), dict(chosen=lists(topk=0)),
    dict(chosen=lists(dtype=torch.int64)), dict(chosen=lists(topk=_lib.SELECT_MAX_BLOCKS + 1)),
    dict(kv_len=zeros(1, dtype=I32)), dict(kv_len=zeros(2, dtype=torch.int64)),
])
def test_attend_refuses_options(options):
    options = dict(options)
    with pytest.raises(ValueError):
        W.attend_8bit(zeros(2, 1, 4, 64), cache(), options.pop("kv_len", 10), **options)


@pytest.mark.parametrize("q", [zeros(1, 4, 64), zeros(1, 1, 4, 64), zeros(2, 1, 4, 128), zeros(2, 1, 3, 64), zeros(2, 1, 1, 64), zeros(2, 1, 0, 64),
                               zeros(2, 1, 4, 64, dtype=torch.float32)], ids=lambda t: f"{tuple(t.shape)}")
def test_attend_refuses_queries(q):
    with pytest.raises(ValueError):
        W.attend_8bit(q, cache(), 10)


def test_attend_and_read_refuse_gradients_and_cpu():
    q = zeros(2, 1, 4, 64)
    with pytest.raises(ValueError, match="no gradient"):
        W.attend_8bit(q.clone().requires_grad_(), cache(), 10)
    with pytest.raises(ValueError, match="no gradient"):
        W.attend_8bit(q, cache(), 10, slopes=torch.zeros(4, requires_grad=True))
    for call in (lambda: W.attend_8bit(q, cache(), 10), lambda: W.kv_read_8bit(cache(), 0, 4), lambda: W.attend_selected(q, cache(), 10, topk=2)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_attend_selected_checks_an_8bit_cache():
    c = cache()
    c["v_scale"] = c["v_scale"][..., :1]
    with pytest.raises(ValueError):
        W.attend_selected(zeros(2, 1, 4, 64), c, 10, topk=2)


# ---------------------------------------------------------------------------------------------
# The C entries: every refusal below is an error code, and nothing is launched.
# ---------------------------------------------------------------------------------------------
def _filled(cls, sizes, optional=()):
    a = cls()
    for name, kind in cls._fields_:
        if kind is ctypes.c_void_p and name not in optional:
            setattr(a, name, FAKE)
        elif name.endswith(("_sb", "_st", "_sh")):
            setattr(a, name, 64)
    for name, x in sizes.items():
        setattr(a, name, x)
    return a


def _refused(fn, a):
    assert getattr(_lib.lib(), fn)(ctypes.byref(a), None) == _lib.WA_ERR_ARG
    assert _lib.lib().wa_last_error()


ATTENTION = dict(B=1, H=2, Hk=1, Lq=8, Lk=8, D=64, scale=0.125, cap=0.0, ranges_sb=0)
BAD_ATTENTION = [dict(D=96), dict(B=0), dict(Lq=0), dict(Lk=0), dict(Hk=0), dict(H=1, Hk=2), dict(H=3, Hk=2), dict(Lq=(1 << 30) + 1),
                 dict(q=None), dict(k=None), dict(v=None), dict(rows=None), dict(tiles=None), dict(order=None), dict(rows=FAKE + 8),
                 dict(q=FAKE + 8), dict(k=FAKE + 2), dict(q_sb=4), dict(v_sh=12), dict(k_st=-64), dict(k_st=(1 << 23) + 8),
                 dict(v_st=(1 << 23) + 8), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(cap=-1.0),
                 dict(cap=math.nan), dict(cap=1e-7), dict(cap=1e7), dict(cap=1.0, scale=1e31)]


@pytest.mark.parametrize("bad", BAD_ATTENTION + [dict(o=None), dict(lse=None), dict(o_st=4), dict(workspace=None, Lk=1 << 20)])
def test_c_ranged_fwd_refuses(bad):
    _refused("wa_ranged_fwd", _filled(_lib.RangedFwdArgs, {**ATTENTION, **bad}))


@pytest.mark.parametrize("bad", BAD_ATTENTION + [dict(o=None), dict(dout=None), dict(lse=None), dict(dq=None), dict(dk=None), dict(dv=None),
                                                 dict(workspace=None), dict(dq=FAKE + 8), dict(q_st=(1 << 23) + 8), dict(d_st=-64),
                                                 dict(d_sh=4), dict(slopes=None), dict(workspace=FAKE + 8)])
def test_c_ranged_bwd_refuses(bad):
    _refused("wa_ranged_bwd", _filled(_lib.RangedBwdArgs, {**ATTENTION, **bad}))


@pytest.mark.parametrize("bad", [dict(B=0), dict(Lq=0), dict(Lk=-1), dict(Lq=(1 << 30) + 1), dict(Lk=(1 << 30) + 1), dict(rows=None),
                                 dict(tiles=None), dict(order=None), dict(rows=FAKE + 4), dict(chunk=0), dict(window=-1), dict(sink=-1),
                                 dict(prefix=None, prefix_all=-1), dict(n_borders=1)])
def test_c_key_ranges_refuses(bad):
    sizes = dict(B=1, Lq=8, Lk=8, chunk=1, window=0, sink=0, prefix_all=0, n_borders=2, documents_sb=0)
    _refused("wa_key_ranges", _filled(_lib.KeyRangesArgs, {**sizes, **bad}, optional=("given",)))


BAD_CACHE = [dict(D=96), dict(block_size=32), dict(code=7), dict(B=0), dict(Hk=0), dict(cap=0), dict(cap=(1 << 30) + 1), dict(k=None),
             dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=FAKE + 8), dict(v=FAKE + 1)]


def _cache8(**bad):
    return _filled(_lib.Cache8, {**dict(B=1, cap=128, Hk=1, D=64, block_size=64, code=_lib.WA_CODE_INT8), **bad})


ENTRIES = {
    "wa_kv8_append": (_lib.Kv8AppendArgs, dict(dtype=_lib.WA_BF16, n=2, start_all=0), ("start",)),
    "wa_kv8_read": (_lib.Kv8ReadArgs, dict(dtype=_lib.WA_BF16, n=2, last=0, window=0, sink=0), ()),
    "wa_kv8_attend": (_lib.Kv8AttendArgs, dict(n=1, H=2, topk=0, window=0, sink=0, scale=0.125, cap=0.0), ("index", "num")),
}


@pytest.mark.parametrize("bad", BAD_CACHE)
@pytest.mark.parametrize("fn", ENTRIES)
def test_c_cache_entries_refuse_caches(fn, bad):
    cls, sizes, optional = ENTRIES[fn]
    _refused(fn, _filled(cls, {**sizes, "cache": _cache8(**bad)}, optional))


@pytest.mark.parametrize("fn,bad", [
    ("wa_kv8_append", dict(n=-1)), ("wa_kv8_append", dict(n=129)), ("wa_kv8_append", dict(start_all=-1)), ("wa_kv8_append", dict(start_all=127)),
    ("wa_kv8_append", dict(dtype=9)), ("wa_kv8_append", dict(k=None)), ("wa_kv8_append", dict(v=FAKE + 8)), ("wa_kv8_append", dict(k_st=4)),
    ("wa_kv8_read", dict(n=-1)), ("wa_kv8_read", dict(last=-1)), ("wa_kv8_read", dict(window=-1)), ("wa_kv8_read", dict(sink=-1)),
    ("wa_kv8_read", dict(dtype=9)), ("wa_kv8_read", dict(k_out=None)), ("wa_kv8_read", dict(v_out=FAKE + 4)),
    ("wa_kv8_attend", dict(n=0)), ("wa_kv8_attend", dict(H=0)), ("wa_kv8_attend", dict(window=-1)), ("wa_kv8_attend", dict(sink=-1)),
    ("wa_kv8_attend", dict(q=None)), ("wa_kv8_attend", dict(o=None)), ("wa_kv8_attend", dict(lse=None)), ("wa_kv8_attend", dict(q=FAKE + 8)),
    ("wa_kv8_attend", dict(o_sh=4)), ("wa_kv8_attend", dict(scale=math.nan)), ("wa_kv8_attend", dict(cap=1e-7)),
    ("wa_kv8_attend", dict(index=FAKE, topk=2)), ("wa_kv8_attend", dict(index=FAKE, num=FAKE, topk=0)),
    ("wa_kv8_attend", dict(index=FAKE, num=FAKE, topk=_lib.SELECT_MAX_BLOCKS + 1)), ("wa_kv8_attend", dict(index=FAKE, num=FAKE, topk=2, window=4)),
])
def test_c_cache_entries_refuse(fn, bad):
    cls, sizes, optional = ENTRIES[fn]
    _refused(fn, _filled(cls, {**sizes, "cache": _cache8(), **bad}, optional))


BIG = 1 << 40


@pytest.mark.parametrize("fn,cls,sizes,optional", [
    ("wa_ranged_fwd", _lib.RangedFwdArgs, {**ATTENTION, "B": BIG, "H": BIG}, ()),
    ("wa_ranged_fwd", _lib.RangedFwdArgs, {**ATTENTION, "B": 1 << 20, "Lq": 1 << 30}, ()),
    ("wa_ranged_bwd", _lib.RangedBwdArgs, {**ATTENTION, "B": BIG, "H": BIG}, ()),
    ("wa_ranged_bwd", _lib.RangedBwdArgs, {**ATTENTION, "B": 1 << 20, "Lk": 1 << 30}, ()),
    ("wa_key_ranges", _lib.KeyRangesArgs, dict(B=BIG, Lq=BIG >> 12, Lk=8, chunk=1, n_borders=2), ("given",)),
    ("wa_key_ranges", _lib.KeyRangesArgs, dict(B=1 << 62, Lq=1 << 30, Lk=8, chunk=1, n_borders=2), ("given",)),
    ("wa_kv8_append", _lib.Kv8AppendArgs, dict(dtype=_lib.WA_BF16, n=2, cache=_cache8(B=1 << 30, Hk=65536)), ("start",)),
    ("wa_kv8_append", _lib.Kv8AppendArgs, dict(dtype=_lib.WA_BF16, n=1 << 30, cache=_cache8(B=1 << 20, cap=1 << 30)), ()),
    ("wa_kv8_read", _lib.Kv8ReadArgs, dict(dtype=_lib.WA_BF16, n=1 << 30, cache=_cache8(Hk=32768)), ()),
    ("wa_kv8_read", _lib.Kv8ReadArgs, dict(dtype=_lib.WA_BF16, n=2, cache=_cache8(B=65536)), ()),
    ("wa_kv8_attend", _lib.Kv8AttendArgs, dict(n=1 << 24, H=65536, cache=_cache8(B=1 << 24, Hk=65536)), ("index", "num")),
    ("wa_kv8_attend", _lib.Kv8AttendArgs, dict(n=1 << 24, H=65536, topk=4, cache=_cache8(B=1 << 24)), ()),
    ("wa_kv8_attend", _lib.Kv8AttendArgs, dict(n=1 << 20, H=64, cache=_cache8(B=1 << 20)), ("index", "num")),
])
def test_c_entries_refuse_sizes_that_no_grid_holds(fn, cls, sizes, optional):
    _refused(fn, _filled(cls, {**({"scale": 0.1} if "attend" in fn else {}), **sizes}, optional))


@pytest.mark.parametrize("fn", ["wa_key_ranges", "wa_ranged_fwd", "wa_ranged_bwd", "wa_kv8_append", "wa_kv8_read", "wa_kv8_attend"])
def test_c_entries_refuse_null(fn):
    assert getattr(_lib.lib(), fn)(None, None) == _lib.WA_ERR_ARG


@pytest.mark.parametrize("x", [2.5, -0.5, math.inf, -math.inf, math.nan, True])
def test_numbers_that_are_not_whole(x):
    """Places and lengths are not cut off to whole numbers, and rules that are not numbers of tokens are no other errors."""
    c, kv = cache(), zeros(2, 3, 2, 64)
    for call in (lambda: W.key_ranges(2, 8, 8, kv_len=x), lambda: W.kv_append_8bit(c, kv, kv, x), lambda: W.kv_read_8bit(c, x, 3),
                 lambda: W.kv_read_8bit(c, 0, x), lambda: W.attend_8bit(zeros(2, 1, 4, 64), c, x), lambda: W.key_ranges(2, 8, 8, window=x),
                 lambda: W.key_ranges(2, 8, 8, prefix=x), lambda: W.key_ranges(x, 8, 8), lambda: W.new_cache_8bit(2, x, 2, 64, device="cpu")):
        with pytest.raises(ValueError, match="whole number"):
            call()


@pytest.mark.parametrize("start_all", [(1 << 63) - 1, (1 << 63) - 2, 1 << 62])
def test_c_append_refuses_places_whose_end_64_bits_do_not_hold(start_all):
    cls, sizes, optional = ENTRIES["wa_kv8_append"]
    _refused("wa_kv8_append", _filled(cls, {**sizes, "cache": _cache8(), "start_all": start_all}, optional))
