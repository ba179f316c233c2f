"""What omni_rotary, OmniPagedCache, omni_cache_append and omni_cache_attention refuse, and what the C entry points return
for it. Nothing here needs a GPU: every check comes before the device is touched."""
import ctypes
import math

import pytest
import torch

import omni_attention_b200 as omni
from omni_attention_b200 import OmniAttnError, ops

f16, f32, i32 = torch.float16, torch.float32, torch.int32


def cache(pages=4, heads=2, page=16, D=64, B=2, per=2, dtype=f16):
    return omni.OmniPagedCache.allocate(pages, heads, page, D, B, per, dtype, device="cpu")


def t(*shape, dtype=f16):
    return torch.zeros(*shape, dtype=dtype)


def refused(match, fn, *a, error=OmniAttnError, **kw):
    with pytest.raises(error, match=match):
        fn(*a, **kw)


def test_rotary_object():
    make = omni.OmniRotary
    refused("layout", make, torch.ones(4, dtype=torch.float64), "both")
    refused("float64", make, torch.ones(4))
    refused("float64", make, torch.ones(2, 2, dtype=torch.float64))
    refused("finite", make, torch.ones(4, dtype=torch.float64), "half", float("nan"))
    for bad in (0, 1, 7, -2):
        refused("rotary_dim", make.from_base, bad)
    for bad in (1.0, 0.0, float("inf")):
        refused("base", make.from_base, 64, bad)
    refused("type", make.from_base, 64, scaling={"type": "other", "factor": 2})
    refused("does not know", make.from_base, 64, scaling={"type": "linear", "factor": 2, "base": 1})
    refused("factor", make.from_base, 64, scaling={"type": "linear", "factor": 0.5})
    refused("factor", make.from_base, 64, scaling={"type": "ntk"})
    refused("above 2", make.from_base, 2, scaling={"type": "ntk", "factor": 2})
    refused("original_length", make.from_base, 64, scaling={"type": "yarn", "factor": 2})
    r = make.from_base(64, scaling={"type": "linear", "factor": 4})
    assert torch.allclose(r.inv_freq * 4, make.from_base(64).inv_freq) and r.rotary_dim == 64 and r.factor == 1.0
    y = make.from_base(64, scaling={"type": "yarn", "factor": 8, "original_length": 4096})
    plain = make.from_base(64).inv_freq
    assert torch.equal(y.inv_freq[0], plain[0]) and torch.allclose(y.inv_freq[-1] * 8, plain[-1]) and y.factor > 1
    n = make.from_base(64, scaling={"type": "ntk", "factor": 8})
    assert torch.allclose(n.inv_freq[-1] * 8, plain[-1]) and n.inv_freq[0] == plain[0]


@pytest.mark.parametrize("rotary_dim,length", [(64, 4096), (128, 32768), (64, 131072), (16, 32768), (4, 4096), (32, 300000)])
def test_yarn_frequencies(rotary_dim, length):
    """Every pair by how often it turns in the trained length. A pair between the two borders is mixed: the ramp ends where a pair
    would turn beta_slow times, not at the last pair there is."""
    base, s, fast, slow = 10000.0, 8.0, 32.0, 1.0
    got = omni.OmniRotary.from_base(rotary_dim, base, scaling={"type": "yarn", "factor": s, "original_length": length}).inv_freq
    pair_of = lambda turns: rotary_dim / 2 * math.log(length / (2 * math.pi * turns), base)
    lo, hi = max(math.floor(pair_of(fast)), 0), math.ceil(pair_of(slow))
    assert hi < rotary_dim
    for p in range(rotary_dim // 2):
        plain = base ** (-2 * p / rotary_dim)
        turns = length * plain / (2 * math.pi)
        stretched = min(max((p - lo) / (hi - lo), 0.0), 1.0)
        assert math.isclose(float(got[p]), plain * (1 - stretched) + plain / s * stretched, rel_tol=1e-12), p
        # by the definition's own words, wherever the whole-numbered borders leave room
        if turns > fast and p <= lo:
            assert math.isclose(float(got[p]), plain, rel_tol=1e-12)
        if slow < turns < fast and lo < p:
            assert plain / s < float(got[p]) < plain


def test_rotary_call():
    f, r = omni.omni_rotary, omni.OmniRotary.from_base(64)
    q, k = t(2, 4, 3, 64), t(2, 2, 3, 64)
    refused("neither", f, q, k)
    refused("OmniRotary", f, q, k, torch.ones(32))
    refused("needs q or k", f, None, None, r)
    refused(r"\[B, H, N, D\]", f, t(4, 3, 64), None, r)
    refused("head_dim=48", f, t(1, 1, 3, 48), None, r, error=ValueError)
    refused("dtype", f, t(1, 1, 3, 64, dtype=torch.float64), None, r)
    refused("dtype", f, t(1, 1, 3, 64, dtype=torch.int16), None, r)
    refused("empty", f, t(1, 0, 3, 64), None, r)
    refused("empty", f, t(0, 1, 3, 64), None, r)
    for bad in (t(2, 2, 4, 64), t(1, 2, 3, 64), t(2, 2, 3, 32), t(2, 2, 3, 64, dtype=f32)):
        refused("share", f, q, bad, r)
    refused("larger", f, t(1, 1, 3, 32), None, r)
    for p in (torch.zeros(3), torch.zeros(4, dtype=i32), torch.zeros(3, 3, dtype=i32), torch.zeros(2, 3, 1, dtype=i32), torch.zeros((), dtype=i32)):
        refused("positions", f, q, k, r, p)
    refused("q_weight", f, q, k, r, None, t(32))
    refused("q_weight", f, q, k, r, None, t(2, 64))
    refused("k_weight", f, q, k, r, None, None, t(4, 64))
    refused("q_weight", f, q, k, r, None, t(64, dtype=torch.bfloat16))
    refused("one form", f, q, k, r, None, t(64), t(2, 64))
    refused("one form", f, q, k, r, None, t(64), t(64, dtype=f32))
    refused("without", f, None, k, r, None, t(64))
    refused("eps", f, q, k, r, None, t(64), None, -1.0)
    refused("eps", f, q, k, r, None, t(64), None, float("nan"))
    refused("CUDA", f, q, k, r)


def test_cache_object():
    make = omni.OmniPagedCache
    kp, vp, table, n = t(4, 2, 16, 64), t(4, 2, 16, 64), torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32)
    assert make(kp, vp, table, n).page_size == 16
    refused("one shape", make, kp, t(4, 2, 16, 32), table, n)
    refused("one shape", make, kp, vp.bfloat16(), table, n)
    refused("one shape", make, kp[0], vp[0], table, n)
    refused("dtype", make, kp.float(), vp.float(), table, n)
    refused("contiguous", make, kp.transpose(1, 2), vp.transpose(1, 2), table, n)
    for size in (8, 17, 48, 2048):
        refused("page_size", make, t(1, 1, size, 64), t(1, 1, size, 64), table, n)
    refused("head_dim", make, t(4, 2, 16, 96), t(4, 2, 16, 96), table, n, error=ValueError)
    refused("page_table", make, kp, vp, table.long(), n)
    refused("page_table", make, kp, vp, table[0], n)
    refused("lengths", make, kp, vp, table, n.long())
    refused("lengths", make, kp, vp, table, torch.zeros(3, dtype=i32))
    c = cache()
    assert int(c.page_table.max()) == -1 and not c.lengths.any()
    other = c.layer_like(t(9, 2, 16, 64), t(9, 2, 16, 64))
    assert other.page_table is c.page_table and other.lengths is c.lengths


def test_append_call():
    f, r, c = omni.omni_cache_append, omni.OmniRotary.from_base(64), cache()
    q, k = t(2, 4, 3, 64), t(2, 2, 3, 64)
    refused("CUDA", f, c, k, k, q, r)
    refused("share shape", f, c, k, t(2, 2, 4, 64))
    refused("share shape", f, c, k, k.bfloat16())
    refused("dtype", f, c, k.float(), k.float())
    refused("share", f, c, k, k, t(2, 4, 2, 64), r)
    refused("heads", f, c, t(2, 4, 3, 64), t(2, 4, 3, 64))
    refused("head_dim", f, c, t(2, 2, 3, 32), t(2, 2, 3, 32))
    refused("dtype", f, c, k.bfloat16(), k.bfloat16())
    refused("page_table", f, c, t(3, 2, 3, 64), t(3, 2, 3, 64))
    for bad in (torch.zeros(3, dtype=i32), torch.zeros(2), torch.zeros(2, dtype=torch.int64), torch.zeros(4, dtype=i32)[::2]):
        refused("counts", f, c, k, k, counts=bad)
    refused("positions", f, c, k, k, q, r, torch.zeros(4, dtype=i32))
    refused("q_weight without q", f, c, k, k, q_weight=t(64))
    refused("no backward", f, c, k.requires_grad_(), k)
    with torch.no_grad():
        refused("CUDA", f, c, k, k)
    broken = cache()
    broken.page_table = torch.zeros(2, 4, dtype=i32)[:, ::2]
    refused("page_table", f, broken, t(2, 2, 3, 64), t(2, 2, 3, 64))


def test_attention_call():
    f, c = omni.omni_cache_attention, cache()
    q = t(2, 4, 3, 64)
    refused("CUDA", f, q, c)
    refused("divide", f, t(2, 3, 3, 64), c)
    refused("dtype", f, q.float(), c)
    refused("dtype", f, q.bfloat16(), c)
    refused("head_dim", f, t(2, 4, 3, 128), c)
    refused("page_table", f, t(1, 4, 3, 64), c)
    refused("empty", f, t(2, 4, 0, 64), c)
    refused("counts", f, q, c, counts=torch.zeros(2, 1, dtype=i32))
    for bad in (torch.zeros(2, dtype=i32), torch.zeros(2, 4, dtype=i32), torch.zeros(2, 3), torch.zeros(3, 2, dtype=i32).t()):
        refused("limits", f, q, c, limits=bad)
    for bad in (-1, 33):
        refused("shared_prefix", f, q, c, shared_prefix=bad)
    refused("finite", f, q, c, scale=float("nan"))
    refused("negative", f, q, c, scale=-1.0)
    refused("finite", f, q, c, softcap=float("inf"))
    refused("no backward", f, q.requires_grad_(), c)


@pytest.mark.parametrize("value", [0.0, 1e-60, 1e60, float("inf")])
def test_numbers_that_32_bits_do_not_hold(value):
    c, q = cache(), t(2, 4, 3, 64)
    refused("scale", omni.omni_cache_attention, q, c, scale=value)     # 0 must not turn into the default
    if value > 1:
        refused("finite", omni.omni_cache_attention, q, c, softcap=value)
        refused("eps", omni.omni_rotary, q, None, None, q_weight=torch.ones(64), eps=value)
        if value != float("inf"):
            refused("factor", omni.omni_rotary, q, None, omni.OmniRotary(torch.ones(4, dtype=torch.float64), factor=value))


# ---------------------------------------------------------------------------------------------------------------------
# the C entry points
# ---------------------------------------------------------------------------------------------------------------------
class Heads(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("sb", ctypes.c_longlong), ("sh", ctypes.c_longlong), ("sn", ctypes.c_longlong), ("heads", ctypes.c_int)]


class Rotary(ctypes.Structure):
    _fields_ = [("inv_freq", ctypes.c_void_p), ("rotary_dim", ctypes.c_int), ("half", ctypes.c_int), ("factor", ctypes.c_float),
                ("positions", ctypes.c_void_p), ("pos64", ctypes.c_int), ("psb", ctypes.c_longlong), ("psn", ctypes.c_longlong),
                ("qw", ctypes.c_void_p), ("kw", ctypes.c_void_p), ("wf32", ctypes.c_int), ("wph", ctypes.c_int), ("eps", ctypes.c_float)]


class Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("table", ctypes.c_void_p), ("stride", ctypes.c_longlong),
                ("lengths", ctypes.c_void_p), ("num_pages", ctypes.c_int), ("max_pages", ctypes.c_int), ("page", ctypes.c_int), ("heads", ctypes.c_int)]


def codes():
    import re
    from test_abi import HEADER
    return {m.group(1): int(m.group(2)) for m in re.finditer(r"#define\s+(OMNI_\w+)\s+\(?(-?\d+)\)?", open(HEADER).read())}


def test_c_entries_return_codes():
    E, lib = codes(), ops.load_library()
    A = 0x10000   # stands for an aligned address: nothing is read
    ref = lambda x: None if x is None else ctypes.byref(x)
    P, L, F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_float

    def heads(data=A, heads=2, s=64):
        return Heads(data, s, s, s, heads)

    def rotary(q=heads(), k=heads(), qo=A, ko=A, rot=Rotary(A, 64, 0, 1.0), B=1, N=1, D=64, dtype=0, inverse=0):
        return lib.omni_attn_rotary_sm100(ref(q), ref(k), P(qo), P(ko), ref(rot), B, N, D, dtype, inverse, None)
    assert rotary(q=None, k=None) == rotary(qo=None) == rotary(rot=None) == rotary(k=heads(None)) == E["OMNI_ERR_NULL_POINTER"]
    assert rotary(dtype=3) == rotary(dtype=-1) == E["OMNI_ERR_DTYPE"]
    assert rotary(D=96) == E["OMNI_ERR_HEAD_DIM"]
    assert rotary(B=0) == rotary(N=-1) == rotary(B=2 ** 20, N=2 ** 20) == rotary(q=heads(heads=0)) == rotary(k=heads(heads=70000)) == E["OMNI_ERR_SHAPE"]
    assert rotary(rot=Rotary(A, 63)) == rotary(rot=Rotary(A, 66)) == rotary(rot=Rotary(A, -2)) == rotary(rot=Rotary(None, 2)) == E["OMNI_ERR_ROTARY"]
    assert rotary(rot=Rotary(A, 64, qw=A), inverse=1) == E["OMNI_ERR_ROTARY"]

    need = lib.omni_attn_rotary_bwd_workspace_bytes
    need.restype = L
    assert need(2, 2, 1, 1, 64, 0) > 0 and need(0, 0, 1, 1, 64, 0) == need(2, 2, 0, 1, 64, 0) == need(2, 2, 1, 1, 65, 0) == 0

    def bwd(q=heads(), g=heads(), dq=A, dw=A, rot=Rotary(A, 64, qw=A), ws=A, size=1 << 30, D=64, dtype=1):
        return lib.omni_attn_rotary_bwd_sm100(ref(q), None, ref(g), None, P(dq), None, P(dw), None, ref(rot), 1, 1, D, dtype, P(ws), L(size), None)
    assert bwd(q=None) == bwd(g=None) == bwd(dq=None) == bwd(dw=None) == bwd(rot=Rotary(A, 64)) == bwd(ws=None) == E["OMNI_ERR_NULL_POINTER"]
    assert bwd(size=16) == E["OMNI_ERR_WORKSPACE"]
    assert bwd(ws=A + 4) == E["OMNI_ERR_ALIGNMENT"]
    assert bwd(g=heads(heads=3)) == E["OMNI_ERR_SHAPE"]
    assert bwd(dtype=4) == E["OMNI_ERR_DTYPE"]

    full = dict(k=A, v=A, table=A, stride=4, lengths=A, num_pages=4, max_pages=4, page=16, heads=2)

    def append(k=heads(), v=heads(), q=None, qo=None, rot=None, D=64, dtype=0, B=1, **c):
        return lib.omni_attn_cache_append_sm100(ref(q), ref(k), ref(v), P(qo), ref(Cache(**{**full, **c})), None, ref(rot), B, 1, D, dtype, None, None)

    def attend(q=heads(heads=4), out=A, ws=A, size=1 << 30, D=64, dtype=0, softcap=0.0, prefix=0, T=1, B=1, **c):
        return lib.omni_attn_cache_attention_sm100(ref(q), P(out), None, ref(Cache(**{**full, **c})), None, None, 1, B, T, D, dtype, F(0), F(softcap),
                                                   prefix, P(ws), L(size), None, None)
    for fn in (append, attend):
        for name in ("k", "v", "table", "lengths"):
            if fn is attend or name in ("table", "lengths"):
                assert fn(**{name: None}) == E["OMNI_ERR_NULL_POINTER"], name
        for bad in (dict(page=8), dict(page=24), dict(page=2048), dict(num_pages=0), dict(max_pages=0)):
            assert fn(**bad) == E["OMNI_ERR_CACHE"], bad
        assert fn(max_pages=2 ** 31 - 1) == E["OMNI_ERR_TOO_LONG"]
        assert fn(dtype=2) == E["OMNI_ERR_DTYPE"] and fn(D=256) == E["OMNI_ERR_HEAD_DIM"] and fn(B=0) == E["OMNI_ERR_SHAPE"]
    assert append(k=None) == append(v=None) == append(q=heads()) == E["OMNI_ERR_NULL_POINTER"]
    assert append(heads=3) == E["OMNI_ERR_CACHE"]
    assert append(rot=Rotary(A, 65)) == E["OMNI_ERR_ROTARY"]
    assert attend(q=None) == attend(out=None) == attend(ws=None, size=0, max_pages=100) == attend(ws=None, prefix=16) == E["OMNI_ERR_NULL_POINTER"]
    assert attend(heads=3) == attend(heads=0) == E["OMNI_ERR_CACHE"]
    assert attend(q=heads(A + 2, 4)) == attend(q=heads(A, 4, 65)) == attend(out=A + 8) == attend(k=A + 2) == E["OMNI_ERR_ALIGNMENT"]
    assert attend(softcap=-1.0) == attend(softcap=float("nan")) == attend(softcap=float("inf")) == E["OMNI_ERR_SOFTCAP"]
    assert attend(prefix=-1) == attend(prefix=80) == E["OMNI_ERR_SEQLEN"]
    assert attend(size=100, max_pages=100) == E["OMNI_ERR_WORKSPACE"]
    size = lib.omni_attn_cache_attention_workspace_bytes
    size.restype = L
    assert size(1, 4, 2, 1, 64, 0, L(64)) == 0 and size(1, 4, 2, 1, 64, 0, L(1600)) > 0 and size(1, 4, 2, 1, 64, 16, L(64)) > 0
    assert size(1, 3, 2, 1, 64, 0, L(1600)) == size(0, 2, 2, 1, 64, 0, L(1600)) == 0
    assert attend(T=2 ** 30) == E["OMNI_ERR_SHAPE"]
    for name in ("OMNI_ERR_ROTARY", "OMNI_ERR_CACHE"):
        lib.omni_attn_error_string.restype = ctypes.c_char_p
        assert lib.omni_attn_error_string(E[name]) != b"unknown error code"


def test_caps_out_of_range():
    """Caps whose quotients with the scale leave 32 bits: they came out as no cap, or as NaN and infinities."""
    q, c = t(2, 4, 1, 64), cache()
    for cap in (1e-300, 1e-50, 1e-40, 1e-8, 1.2e-7, 1e30, 2e37, 3e38):
        refused("softcap must be", omni.omni_cache_attention, q, c, softcap=cap)
    refused("softcap must be", omni.omni_cache_attention, q, c, softcap=50.0, scale=1e8)
    refused("softcap must be", omni.omni_cache_attention, q, c, softcap=50.0, scale=1e-29)
    for cap in (None, 0.0, -3.0, 1.5e-7, 50.0, 1e29):
        refused("CUDA", omni.omni_cache_attention, q, c, softcap=cap)
    E, lib, A, F, P = codes(), ops.load_library(), 0x10000, ctypes.c_float, ctypes.c_void_p   # nothing is read
    full = dict(k=A, v=A, table=A, stride=4, lengths=A, num_pages=4, max_pages=4, page=16, heads=2)
    for scale, cap in ((0.0, 1e-8), (0.0, 3e38), (1.0, 1e-7), (1e8, 50.0), (1e-30, 50.0), (1e30, 1e38)):
        assert lib.omni_attn_cache_attention_sm100(ctypes.byref(Heads(A, 64, 64, 64, 4)), P(A), None, ctypes.byref(Cache(**full)), None, None, 1, 1, 1, 64, 0,
                                                   F(scale), F(cap), 0, P(A), ctypes.c_longlong(1 << 30), None, None) == E["OMNI_ERR_SOFTCAP"]


def test_learned_frequencies():
    """Nothing here has a gradient of inv_freq: refused where one is asked for."""
    r = omni.OmniRotary(torch.ones(32, dtype=torch.float64).requires_grad_())
    refused("inv_freq", omni.omni_rotary, t(1, 1, 3, 64), None, r)
    refused("inv_freq", omni.omni_rotary, t(1, 1, 3, 64).requires_grad_(), None, r)
    refused("no backward", omni.omni_cache_append, cache(), t(2, 2, 3, 64), t(2, 2, 3, 64), rotary=r)
    with torch.no_grad():
        refused("CUDA", omni.omni_rotary, t(1, 1, 3, 64), None, r)


def test_pages_that_require_a_gradient():
    """Writing into them would cut their graph without a word, as an operation in place on such a leaf would: refused, but not
    under no_grad."""
    k = t(2, 2, 3, 64)
    for which in ("k_pages", "v_pages"):
        c = cache()
        getattr(c, which).requires_grad_()
        refused("no backward", omni.omni_cache_append, c, k, k)
        refused("no backward", omni.omni_cache_attention, k, c)
        with torch.no_grad():
            refused("CUDA", omni.omni_cache_append, c, k, k)


def test_forward_mode():
    """A tangent is refused, whether something requires a gradient or not: it would be dropped."""
    from torch.autograd import forward_ad as fw
    r = omni.OmniRotary.from_base(64)
    q, k, c = t(2, 4, 3, 64), t(2, 2, 3, 64), cache()
    with fw.dual_level():
        d = lambda x: fw.make_dual(x, torch.ones_like(x))
        for grad in (False, True):
            refused("forward-mode", omni.omni_rotary, d(q), k.clone().requires_grad_(grad), r)
        refused("forward-mode", omni.omni_rotary, q, d(k), r)
        refused("forward-mode", omni.omni_rotary, q, k, r, None, d(t(64)), t(64))
        refused("forward-mode", omni.omni_rotary, q, k, omni.OmniRotary(d(r.inv_freq)))
        for args in ((d(k), k, q), (k, d(k), q), (k, k, d(q))):
            refused("forward-mode", omni.omni_cache_append, c, *args)
        refused("forward-mode", omni.omni_cache_attention, d(q), c)
        c2 = omni.OmniPagedCache(c.k_pages, d(c.v_pages), c.page_table, c.lengths)
        refused("forward-mode", omni.omni_cache_attention, q, c2)
        refused("CUDA", omni.omni_rotary, q, k, r)
    refused("CUDA", omni.omni_cache_append, c, k, k, q)


def test_a_prompt_on_a_cache_that_is_not_empty():
    """The slot's own check, where it was asked for: before anything is computed."""
    from omni_attention_b200.transfusion import patch_attention, transfusion_block_mask, unpatch_attention
    from test_transfusion_gpu import AttentionLike
    mod = AttentionLike(32, 64, 2, learned_mix=False)
    mask = transfusion_block_mask(torch.tensor([[[1, 2, 3]], [[1, 0, 5]]], dtype=i32), 2, 128)
    c, x = cache(), torch.randn(2, 128, 32)
    c.lengths[1] = 3
    with torch.no_grad():
        assert patch_attention(mod, check_status=True) is mod
        refused("must be empty", mod, x, block_mask=mask, cache=c)
        patch_attention(mod)                        # not asked for any more: the next complaint is that there is no GPU
        refused("CUDA", mod, x, block_mask=mask, cache=c)
        patch_attention(mod, check_status=True)
        c.lengths.zero_()
        refused("CUDA|cuda", mod, x, block_mask=mask, cache=c, error=(OmniAttnError, RuntimeError))
    assert unpatch_attention(mod) is mod and not hasattr(mod, "_omni_check_status")
