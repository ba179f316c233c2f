"""omni_cache_append and omni_cache_attention against their definitions in 64 bits.

Tolerances of the attention. A result is rounded once (eps / 2 of its value). Before that: a score is a sum of D products of
16-bit values in 32 bits, off by at most 2^-20 of the sum of their absolute values (D / 16 steps of the tensor cores' sums);
with the scale that is SCORE = 2^-20 * scale * max sum |q k|; the exponential adds 2^-21 relative, P as the sum of two 16-bit
values 2^-16 (bf16: 8 + 8 bits and their signs; less in fp16). Each is a relative error e of a weight, and a mean of values
with weights off by e is off by at most 2 e max |v|.

With more than 16 query rows to a key/value head P is one 16-bit value, while the sum that divides has the unrounded ones: every
weight's value is off by half a step, so the mean by eps / 2 * sum(weight * |v|), which the oracle returns; where p is subnormal
in fp16 (below 2^-14, the largest of a row being at least 1/2) by 2^-25 each, 2^-24 * keys * max |v| over the sum."""
import math

import pytest
import torch

import omni_attention_b200 as omni
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


def make_cache(B, Hkv, D, page, lengths, T, dtype, seed=0, spare=2, shared=0, stale=math.nan):
    """Pages in random order. What lies behind a sequence's tokens (T new ones included) and in pages of nobody is `stale`."""
    g = torch.Generator().manual_seed(seed)
    per = max(1, -(-(max(lengths) + T) // page))
    sp = shared // page
    pages = sp + B * (per - sp) + spare
    order = torch.randperm(pages, generator=g).int()
    table = torch.empty(B, per, dtype=torch.int32)
    table[:, :sp] = order[:sp]
    table[:, sp:] = order[sp:sp + B * (per - sp)].view(B, per - sp)
    kp, vp = (torch.full((pages, Hkv, page, D), stale, dtype=dtype) for _ in range(2))
    for b in range(B):
        for i in range(lengths[b] + T):
            p = int(table[b, i // page])
            if b == 0 or i >= shared:
                kp[p, :, i % page] = torch.randn(Hkv, D, generator=g).to(dtype)
                vp[p, :, i % page] = torch.randn(Hkv, D, generator=g).to(dtype)
    return kp, vp, table, torch.tensor(lengths, dtype=torch.int32), g


def on_gpu(kp, vp, table, lengths):
    return omni.OmniPagedCache(kp.cuda(), vp.cuda(), table.cuda(), lengths.cuda())


def check(got, lse, want, want_lse, size, q, kp, vp, scale, what, wide=False):
    dtype = got.dtype
    finite = lambda t: torch.nan_to_num(t.double(), nan=0.0, posinf=0.0, neginf=0.0)
    vmax = float(finite(vp).abs().max())
    score = 2.0 ** -20 * scale * float((finite(q).abs().amax((0, 1, 2)) * finite(kp).abs().amax((0, 1, 2))).sum())
    e = score + 2.0 ** -21 + 2.0 ** -16
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2 * e * vmax + 2.0 ** -25
    if wide:
        tol = tol + torch.finfo(dtype).eps / 2 * size + (2.0 ** -24 * kp.shape[0] * kp.shape[2] * vmax if dtype == torch.float16 else 0)
    worst = float(((got - want).abs() / tol).max())
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"
    empty = torch.isinf(want_lse)
    assert not got[empty].any(), f"{what}: a row with no key is not zero"
    if lse is not None:
        lse = lse.double().cpu()
        assert torch.equal(torch.isinf(lse), empty), what
        err = (lse - want_lse)[~empty].abs()
        assert not len(err) or float(err.max()) <= score + 2.0 ** -20 + 2.0 ** -22 * float(want_lse[~empty].abs().max()), what


def run(q, kp, vp, table, lengths, what="", **kw):
    cache = on_gpu(kp, vp, table, lengths)
    gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    got, lse = omni.omni_cache_attention(q.cuda(), cache, return_lse=True, **gpu)
    ref = {k: v for k, v in kw.items() if k not in ("shared_prefix", "check_status")}
    if ref.get("softcap") is None:
        ref.pop("softcap", None)
    B, H, T, D = q.shape
    wide = H // kp.shape[1] * T * (B if kw.get("shared_prefix") else 1) > 16
    check(got, lse, *orc.attention(q, kp, vp, table, lengths, **ref), q, kp, vp, kw.get("scale") or D ** -0.5, what, wide)
    plain = omni.omni_cache_attention(q.cuda(), cache, **gpu)
    assert torch.equal(plain, got), "with and without lse, and again: the same bits"
    return got


ATTEND = [  # B, H, Hkv, T, D, page, lengths, dtype, causal, softcap
    (1, 1, 1, 1, 64, 16, [0], torch.float16, True, None),
    (1, 2, 2, 1, 64, 16, [1], torch.bfloat16, True, None),
    (1, 16, 16, 1, 64, 16, [511], torch.float16, True, 50.0),
    (3, 8, 2, 1, 128, 64, [5, 0, 700], torch.bfloat16, True, None),
    (2, 4, 1, 1, 32, 32, [63, 64], torch.float16, True, 5.0),
    (2, 32, 2, 1, 64, 16, [129, 15], torch.bfloat16, True, None),      # 16 heads to one
    (1, 24, 1, 1, 128, 128, [257], torch.float16, True, None),         # 24 heads to one: two row tiles
    (2, 4, 2, 5, 128, 16, [40, 3], torch.bfloat16, True, None),
    (2, 2, 1, 33, 64, 64, [0, 90], torch.float16, True, None),
    (1, 4, 4, 70, 32, 16, [100], torch.bfloat16, False, 30.0),
    (2, 2, 2, 130, 128, 32, [17, 300], torch.bfloat16, False, None),
    (1, 4, 2, 129, 64, 1024, [31], torch.float16, True, None),
    (5, 2, 1, 2, 128, 256, [1, 2, 255, 256, 257], torch.bfloat16, True, 1.0),
    (1, 2, 1, 1, 128, 64, [6000], torch.bfloat16, True, None),
    (2, 8, 2, 40, 64, 64, [900, 1500], torch.bfloat16, True, None),    # 160 rows: two tiles, many tiles of keys
    (1, 2, 1, 257, 128, 512, [1, ], torch.bfloat16, False, 3.0),
    (3, 4, 1, 9, 32, 128, [300, 128, 127], torch.float16, True, None),
    (70, 1, 1, 1, 32, 16, [(7 * i) % 40 for i in range(70)], torch.float16, True, None),
]


@pytest.mark.parametrize("B,H,Hkv,T,D,page,lengths,dtype,causal,softcap", ATTEND)
def test_attention(cuda_device, B, H, Hkv, T, D, page, lengths, dtype, causal, softcap):
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, lengths, T, dtype)
    q = torch.randn(B, H, T, D, generator=g).to(dtype)
    run(q, kp, vp, table, lens, "attention", causal=causal, softcap=softcap)


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_scores_of_every_size(cuda_device, D, dtype):
    """Scores from flat to one that takes everything, and a maximum that grows along the keys."""
    for gain in (0.0, 1.0, 8.0):
        kp, vp, table, lens, g = make_cache(2, 2, D, 16, [200, 333], 1, dtype, seed=3)
        q = (gain * torch.randn(2, 48, 1, D, generator=g)).to(dtype)
        run(q[:, :4], kp, vp, table, lens, f"gain {gain}")
        run(q, kp, vp, table, lens, f"gain {gain}, many rows")
    kp, vp, table, lens, g = make_cache(1, 1, D, 16, [400], 1, dtype, seed=4)
    for i in range(401):
        kp[int(table[0, i // 16]), 0, i % 16] = 0.02 * i
    for heads in (2, 20):
        run(torch.ones(1, heads, 1, D, dtype=dtype), kp, vp, table, lens, "growing")
        run(-torch.ones(1, heads, 1, D, dtype=dtype), kp, vp, table, lens, "falling")
        run(torch.ones(1, heads, 1, D, dtype=dtype), kp, vp, table, lens, "scale", scale=0.003)


@pytest.mark.parametrize("H", [4, 16])      # 12 and 48 rows to a key/value head
def test_limits_counts_and_empty_rows(cuda_device, H):
    B, Hkv, T, D, page = 4, 2, 6, 64, 16
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, [0, 30, 47, 160], T, torch.bfloat16)
    q = torch.randn(B, H, T, D, generator=g).bfloat16()
    limits = torch.tensor([[0, 1, 2, -5, 6, 1000], [36, 35, 1, 0, 16, 17], [0] * 6, [-2 ** 31, 2 ** 31 - 1, 5, 150, 166, 16]], dtype=torch.int32)
    run(q, kp, vp, table, lens, "limits", limits=limits)
    counts = torch.tensor([6, 0, 3, -1], dtype=torch.int32)
    q2 = q.clone()
    q2[1] = math.nan                 # padding may hold anything
    q2[2, :, 3:] = math.inf
    q2[3] = math.nan
    # behind a sequence's count nothing has been written: stale again
    for b, c in enumerate(counts.clamp(min=0).tolist()):
        for i in range(int(lens[b]) + c, int(lens[b]) + T):
            kp[int(table[b, i // page]), :, i % page] = math.nan
            vp[int(table[b, i // page]), :, i % page] = math.nan
    for causal in (True, False):
        got = run(q2, kp, vp, table, lens, f"counts causal={causal}", counts=counts, causal=causal)
        assert not got[1].any() and not got[3].any() and not got[2, :, 3:].any()


def test_lengths_at_the_ends(cuda_device):
    """Negative lengths count as none, lengths beyond the table as all it holds."""
    kp, vp, table, lens, g = make_cache(3, 1, 64, 16, [60, 60, 60], 4, torch.float16)
    q = torch.randn(3, 2, 1, 64, generator=g).half()
    lens = torch.tensor([-7, 64, 2 ** 31 - 1], dtype=torch.int32)
    run(q, kp, vp, table, lens, "ends")
    run(q, kp, vp, table, lens, "ends", causal=False)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("H,T,lengths", [(4, 6, [40, 300]), (2, 4, [0, 17]), (8, 30, [100, 2100]), (4, 130, [0, 500])])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(cuda_device, value, H, T, lengths):
    """Keys and values of new tokens that are infinite or NaN: rows before them are as if they were not there."""
    B, Hkv, D, page = 2, 2, 64, 16
    for dtype in (torch.float16, torch.bfloat16):
        kp, vp, table, lens, g = make_cache(B, Hkv, D, page, lengths, T, dtype, seed=5)
        q = torch.randn(B, H, T, D, generator=g).to(dtype)
        at = T // 2
        kp2, vp2 = kp.clone(), vp.clone()
        for b in range(B):
            for t in (at, T - 1):
                i = lengths[b] + t
                p, row = int(table[b, i // page]), i % page
                vp2[p, :, row, 5] = value
                if t == T - 1:
                    kp2[p, :, row] = math.nan
                    vp2[p, :, row] = value
        clean = omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens))
        got = omni.omni_cache_attention(q.cuda(), on_gpu(kp2, vp2, table, lens))
        assert torch.equal(got[:, :, :at], clean[:, :, :at]), "rows that do not see it"
        seen = got[:, :, at:T - 1].double().cpu()
        rest = [c for c in range(D) if c != 5]
        assert not torch.isfinite(seen[..., 5]).any(), "rows that see it, its column"
        want, _, size = orc.attention(q, kp, vp, table, lens)
        # the other columns are the product's and one more addition, rounded once more
        tol = torch.finfo(dtype).eps * (size[:, :, at:T - 1] + want[:, :, at:T - 1].abs()) + 1e-3
        assert ((seen - want[:, :, at:T - 1]).abs() <= tol)[..., rest].all()
        assert not torch.isfinite(got[:, :, T - 1]).any()


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (32, torch.bfloat16)])
def test_append_without_rotation_stores_what_it_is_given(cuda_device, D, dtype):
    g = torch.Generator().manual_seed(6)
    k, v, q = (torch.randn(2, 3, 20, D, generator=g).to(dtype) for _ in range(3))
    for t in (k, v, q):
        where = torch.rand(t.shape, generator=g) < 0.2
        t[where] = torch.tensor([math.inf, -math.inf, math.nan], dtype=dtype)[torch.arange(int(where.sum())) % 3]
    cache = omni.OmniPagedCache.allocate(4, 3, 16, D, 2, 2, dtype)
    cache.page_table.copy_(torch.arange(4).view(2, 2))
    back = omni.omni_cache_append(cache, k.cuda(), v.cuda(), q=q.cuda())
    stored = lambda pages: pages.view(2, 2, 3, 16, D).transpose(1, 2).reshape(2, 3, 32, D)[:, :, :20].cpu()
    for got, given in ((stored(cache.k_pages), k), (stored(cache.v_pages), v), (back.cpu(), q)):
        assert torch.equal(got.isnan(), given.isnan())
        assert torch.equal(got.nan_to_num(nan=7.0), given.nan_to_num(nan=7.0))


@pytest.mark.parametrize("softcap", [50.0, None])
@pytest.mark.parametrize("H,T,causal", [(2, 1, True), (4, 3, True), (16, 1, True), (24, 2, True), (4, 30, False), (3, 40, True)])
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (32, torch.float16)])
def test_what_nobody_sees_changes_no_bit(cuda_device, D, dtype, H, T, causal, softcap):
    """Pages behind the tokens, queries of padding, and what ran before: zeros, large numbers, infinities or NaN there, the same bits."""
    B, page, lengths, counts = 3, 16, [37, 5, 300], torch.tensor([T, (T + 1) // 2, T], dtype=torch.int32)
    results = []
    big = make_cache(2, 1, D, page, [900, 700], T, dtype, seed=8, stale=0.0)
    for stale in (0.0, 300.0, -1e4, math.nan, math.inf):
        kp, vp, table, lens, g = make_cache(B, 1, D, page, lengths, T, dtype, seed=7, stale=stale)
        q = torch.randn(B, H, T, D, generator=g).to(dtype)
        for b, c in enumerate(counts.tolist()):
            q[b, :, c:] = stale
            for i in range(lengths[b] + c, lengths[b] + T):
                kp[int(table[b, i // page]), :, i % page] = stale
                vp[int(table[b, i // page]), :, i % page] = stale
        if stale != 0.0:    # what shared memory holds
            omni.omni_cache_attention(torch.full((2, H, T, D), 100.0, dtype=dtype, device="cuda"), on_gpu(big[0] * 100, big[1] * 100, *big[2:4]))
        results.append(omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens), counts=counts.cuda(), causal=causal, softcap=softcap, return_lse=True))
    for out, lse in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(lse, results[0][1])


@pytest.mark.parametrize("H", [4, 40])
@pytest.mark.parametrize("cap", [1.5e-7, 1e-3, 1e5, 1e29])
def test_caps_near_the_ends_of_their_range(cuda_device, cap, H):
    """From a cap that leaves nothing of the scores to one that changes nothing, zero scores among them."""
    kp, vp, table, lens, g = make_cache(2, 2, 64, 16, [300, 20], 2, torch.float16, seed=13)
    q = torch.randn(2, H, 2, 64, generator=g).half()
    q[0, 1] = 0
    run(q, kp, vp, table, lens, f"cap {cap}", softcap=cap)


def same_kinds(got, want, tol, what):
    """Infinite with the sign, NaN and finite where the definition says so; the finite ones within tol."""
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN"
    for sign in (math.inf, -math.inf):
        assert torch.equal(got == sign, want == sign), f"{what}: {sign}"
    fin = want.isfinite()
    worst = float(((got - want).abs() / tol)[fin].max())
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"


def infinite_values(B, H, Hkv, T, D, page, lengths, dtype, seed, gain=1.0, **kw):
    """A call on keys whose values are infinite or NaN here and there: (out, 64-bit out, mean of |v|, vmax, scores' bound)."""
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, lengths, T, dtype, seed=seed, shared=kw.get("shared_prefix", 0))
    q = (gain * torch.randn(B, H, T, D, generator=g)).to(dtype)
    plain = vp.clone()
    for b in range(B):
        n = lengths[b] + T
        # column 0: +inf everywhere; 1: -inf; 2: both; 3: NaN; 4..: +inf at one key of every sixteenth place
        for i in torch.randint(0, n, (6,), generator=g).tolist():
            p, row = int(table[b, i // page]), i % page
            vp[p, :, row, 0], vp[p, :, row, 1], vp[p, :, row, 3] = math.inf, -math.inf, math.nan
            vp[p, :, row, 2] = math.inf if i % 2 else -math.inf
        for i in range(0, n, max(1, n // (D // 3))):
            vp[int(table[b, i // page]), :, i % page, 4 + i % (D - 4)] = math.inf if i % 3 else -math.inf
    gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    got = omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens), **gpu)
    ref = {k: v for k, v in kw.items() if k != "shared_prefix"}
    want = orc.attention(q, kp, vp, table, lens, **ref)[0]
    fin = lambda t: torch.nan_to_num(t.double(), nan=0.0, posinf=0.0, neginf=0.0)
    score = 2.0 ** -20 * D ** -0.5 * float((fin(q).abs().amax((0, 1, 2)) * fin(kp).abs().amax((0, 1, 2))).sum())
    size = orc.attention(q, kp, plain, table, lens, **ref)[2]
    return got, want, size, float(fin(plain).abs().max()), score


# B, H, Hkv, T, D, page, lengths, dtype, more: up to 16 rows to a key/value head
INFINITE_FEW = [
    (1, 2, 2, 1, 64, 16, [40], torch.float16, {}),
    (2, 8, 2, 1, 128, 64, [300, 17], torch.bfloat16, {}),
    (2, 4, 1, 1, 32, 32, [63, 129], torch.float16, dict(softcap=20.0)),
    (1, 16, 1, 1, 128, 16, [2000], torch.bfloat16, {}),                        # 16 rows, cut among CTAs
    (3, 2, 1, 4, 64, 128, [5, 0, 700], torch.bfloat16, {}),                    # 8 rows that see different numbers of keys
    (2, 3, 1, 5, 128, 16, [100, 40], torch.float16, dict(causal=False)),
    (1, 1, 1, 1, 32, 16, [6000], torch.bfloat16, {}),
    (4, 2, 2, 1, 64, 16, [100, 80, 90, 300], torch.float16, dict(shared_prefix=64)),
]


@pytest.mark.parametrize("B,H,Hkv,T,D,page,lengths,dtype,more", INFINITE_FEW)
def test_infinite_values_with_few_rows(cuda_device, B, H, Hkv, T, D, page, lengths, dtype, more):
    for seed in range(3):
        got, want, size, vmax, score = infinite_values(B, H, Hkv, T, D, page, lengths, dtype, seed, **more)
        assert want.isinf().any() and want.isnan().any() and want.isfinite().any()
        # as in check(): the result's rounding, the weights' errors
        tol = torch.finfo(dtype).eps / 2 * want.abs() + 2 * (score + 2.0 ** -21 + 2.0 ** -16) * vmax + 2.0 ** -25
        same_kinds(got, want, tol, f"seed {seed}")


# more than 16 rows to a key/value head
INFINITE_MANY = [
    (1, 24, 1, 1, 128, 128, [257], torch.float16, {}),
    (2, 2, 1, 33, 64, 64, [0, 90], torch.float16, {}),
    (1, 4, 4, 70, 32, 16, [100], torch.bfloat16, dict(causal=False, softcap=30.0)),
    (2, 2, 2, 130, 128, 32, [17, 300], torch.bfloat16, dict(causal=False)),
    (1, 2, 1, 20, 64, 16, [3000], torch.bfloat16, {}),                         # cut among CTAs
    (1, 2, 1, 20, 128, 64, [300], torch.float16, dict(causal=False, gain=8.0)),  # weights below fp16's smallest
    (1, 20, 1, 1, 64, 64, [300], torch.float16, dict(gain=8.0)),
    (12, 2, 1, 1, 64, 16, [100 + i for i in range(12)], torch.float16, dict(shared_prefix=64)),
]


@pytest.mark.parametrize("B,H,Hkv,T,D,page,lengths,dtype,more", INFINITE_MANY)
def test_infinite_values_with_many_rows(cuda_device, B, H, Hkv, T, D, page, lengths, dtype, more):
    for seed in range(2):
        got, want, size, vmax, score = infinite_values(B, H, Hkv, T, D, page, lengths, dtype, seed, **more)
        assert want.isinf().any() and want.isnan().any() and want.isfinite().any()
        # as in check(), P rounded to 16 bits; the shared prefix of two rows a sequence has 24 rows
        tol = torch.finfo(dtype).eps / 2 * (want.abs() + size) + 2 * (score + 2.0 ** -21 + 2.0 ** -16) * vmax + 2.0 ** -25
        if dtype == torch.float16:
            tol = tol + 2.0 ** -24 * (max(lengths) + T) * vmax
        same_kinds(got, want, tol, f"seed {seed}")


@pytest.mark.parametrize("H", [1, 12, 40])
@pytest.mark.parametrize("length", [60, 700, 5000])
@pytest.mark.parametrize("late", [True, False])
def test_an_infinite_value_of_a_key_that_weighs_next_to_nothing(cuda_device, H, length, late):
    """Its weight is exp(-110) of the largest, nothing in 32 bits: by the definition the result is infinite all the same, wherever
    the keys are cut."""
    D, page = 64, 16
    kp, vp, table, lens, g = make_cache(1, 1, D, page, [length], 1, torch.bfloat16, seed=16)
    n = length + 1
    heavy = range(n // 2, n) if late else range(0, n // 2)
    for i in range(n):
        p, row = int(table[0, i // page]), i % page
        kp[p, 0, row] = 0.0
        kp[p, 0, row, 0] = 110.0 if i in heavy else 0.0      # the scores: 110 and 0
    light = 0 if late else n - 1
    vp[int(table[0, light // page]), 0, light % page, 3] = math.inf
    q = torch.zeros(1, H, 1, D, dtype=torch.bfloat16)
    q[..., 0] = 8.0
    got = omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens)).cpu()
    want = orc.attention(q, kp, vp, table, lens)[0]
    assert (want[..., 3] == math.inf).all() and (got[..., 3] == math.inf).all()
    rest = [c for c in range(D) if c != 3]
    assert torch.isfinite(got[..., rest]).all() and float((got.double() - want)[..., rest].abs().max()) <= 2.0 ** -8 * 5


@pytest.mark.parametrize("B,T,most,dtype", [(100, 3, 200, torch.bfloat16), (44, 1, 1500, torch.float16), (60, 12, 150, torch.float16), (44, 10, 900, torch.bfloat16)])
def test_infinite_values_of_some_sequences(cuda_device, B, T, most, dtype):
    """More (sequence, head) pairs than CTAs: what one piece of a CTA's work finds stays out of its next ones."""
    H, Hkv, D, page = 8, 4, 64, 16
    g = torch.Generator().manual_seed(14)
    lengths = torch.randint(0, most, (B,), generator=g).tolist()
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, lengths, T, dtype, seed=15)
    q = torch.randn(B, H, T, D, generator=g).to(dtype)
    clean = omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens)).cpu()
    for b in range(0, B, 3):
        n = lengths[b] + T
        for i, col, sign in ((n - 1, 3, 1), (0, 9, -1), (n // 2, 20, 1)):
            vp[int(table[b, i // page]), b % Hkv, i % page, col] = sign * math.inf
    got = omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens)).cpu()
    want = clean.clone()
    for b in range(0, B, 3):
        heads = slice(2 * (b % Hkv), 2 * (b % Hkv) + 2)
        n = lengths[b] + T
        for i, col, sign in ((n - 1, 3, 1), (0, 9, -1), (n // 2, 20, 1)):
            for t in range(T):
                if i <= lengths[b] + t:
                    want[b, heads, t, col] = sign * math.inf
    assert torch.equal(got, want)


@pytest.mark.parametrize("B,H,Hkv,T,D,page,lengths,dtype,more", [
    (1, 2, 1, 20, 128, 64, [300], torch.float16, {}),
    (2, 4, 2, 30, 64, 16, [100, 40], torch.bfloat16, {}),
])
def test_finite_columns_beside_infinite_ones(cuda_device, B, H, Hkv, T, D, page, lengths, dtype, more):
    """The columns of a key that are finite go through the product like any other's, although rows of the tile see different
    numbers of keys: the same bits as without the infinite ones."""
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, lengths, T, dtype, seed=9)
    q = torch.randn(B, H, T, D, generator=g).to(dtype)
    clean = omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens))
    for b in range(B):
        for t in range(T):
            i = lengths[b] + t
            vp[int(table[b, i // page]), :, i % page, t % 3] = math.inf
    got = omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens))
    assert torch.equal(got[..., 3:], clean[..., 3:])
    assert (got[:, :, 3:, :3] == math.inf).all() and (got[:, :, 0, 0] == math.inf).all()


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("heads", [4, 48])
def test_pages_that_are_not_there(cuda_device, bad, heads):
    kp, vp, table, lens, g = make_cache(3, 2, 64, 16, [100, 40, 10], 1, torch.float16)
    q = torch.randn(3, heads, 1, 64, generator=g).half()
    table[0, 2] = bad
    table[0, 6] = bad
    table[2, 0] = bad        # all of the sequence's tokens
    run(q, kp, vp, table, lens, "bad pages")
    with pytest.raises(omni.OmniAttnError, match="page_table"):
        omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens), check_status=True)
    table[0, 2], table[0, 6], table[2, 0] = 0, 1, 2
    omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens), check_status=True)
    table[1, 6] = bad        # beyond the sequence's tokens: never looked at
    omni.omni_cache_attention(q.cuda(), on_gpu(kp, vp, table, lens), check_status=True)


PREFIX = [  # B, H, Hkv, T, D, page, prefix, lengths, dtype
    (3, 4, 2, 1, 64, 16, 32, [32, 40, 100], torch.float16),
    (20, 8, 2, 1, 128, 16, 160, [160 + 3 * i for i in range(20)], torch.bfloat16),
    (2, 2, 1, 5, 32, 64, 128, [200, 128], torch.bfloat16),
    (40, 4, 4, 1, 64, 32, 320, [320 + i for i in range(40)], torch.float16),
    (1, 2, 2, 1, 128, 16, 64, [90], torch.bfloat16),
    (9, 32, 2, 2, 128, 128, 256, [256 + 60 * i for i in range(9)], torch.bfloat16),
]


@pytest.mark.parametrize("B,H,Hkv,T,D,page,prefix,lengths,dtype", PREFIX)
def test_shared_prefix(cuda_device, B, H, Hkv, T, D, page, prefix, lengths, dtype):
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, lengths, T, dtype, shared=prefix)
    q = torch.randn(B, H, T, D, generator=g).to(dtype)
    run(q, kp, vp, table, lens, "prefix", shared_prefix=prefix, check_status=True)
    run(q, kp, vp, table, lens, "half a page more", shared_prefix=prefix + page // 2)
    run(q, kp, vp, table, lens, "softcap", shared_prefix=prefix, softcap=20.0, causal=False)
    # rows that end inside the prefix, sequences shorter than it (one a padding entry without pages), the first among them
    lens2, table2 = lens.clone(), table.clone()
    if B > 2:
        lens2[0], table2[0] = 0, -1
        table2[0, 0] = table2[1, 0]
        lens2[2] = prefix // 2
    limits = torch.full((B, T), 10 ** 6, dtype=torch.int32)
    limits[-1, 0] = prefix // 2 + 3
    run(q, kp, vp, table2, lens2, "short sequences", shared_prefix=prefix, limits=limits)


def test_a_prefix_that_is_not_shared_is_reported(cuda_device):
    kp, vp, table, lens, g = make_cache(4, 1, 64, 16, [50] * 4, 1, torch.float16)
    q = torch.randn(4, 2, 1, 64, generator=g).half().cuda()
    cache = on_gpu(kp, vp, table, lens)
    omni.omni_cache_attention(q, cache, check_status=True)
    with pytest.raises(omni.OmniAttnError, match="page_table"):
        omni.omni_cache_attention(q, cache, shared_prefix=32, check_status=True)


APPEND = [  # B, H, Hkv, T, D, page, lengths, counts, rd, layout, norm, dtype
    (1, 1, 1, 1, 64, 16, [0], None, 64, "interleaved", None, torch.float16),
    (3, 4, 2, 1, 128, 16, [15, 16, 17], None, 128, "half", "shared", torch.bfloat16),
    (2, 4, 2, 50, 64, 32, [10, 0], [50, 7], 32, "interleaved", "head", torch.float16),
    (2, 2, 1, 40, 32, 16, [31, 3], [0, 40], 8, "half", None, torch.bfloat16),
    (1, 8, 8, 300, 128, 64, [100], None, 64, "half", "shared", torch.bfloat16),
    (4, 2, 2, 9, 64, 1024, [0, 1020, 5, 1], [9, 9, -3, 100], 0, "interleaved", None, torch.float16),
]


@pytest.mark.parametrize("B,H,Hkv,T,D,page,lengths,counts,rd,layout,norm,dtype", APPEND)
def test_append(cuda_device, B, H, Hkv, T, D, page, lengths, counts, rd, layout, norm, dtype):
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, lengths, T, dtype)
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(dtype).transpose(1, 2) for h in (H, Hkv, Hkv))
    shape = lambda h: (D,) if norm == "shared" else (h, D)
    wq, wk = (None, None) if norm is None else ((1 + 0.3 * torch.randn(shape(h), generator=g)) for h in (H, Hkv))
    rot = omni.OmniRotary.from_base(rd, layout=layout) if rd else None
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    for positions in (None, torch.randint(0, 99999, (B, T), generator=g)):
        cache = on_gpu(kp, vp, table, lens)
        opt = lambda t: None if t is None else t.cuda()
        got = omni.omni_cache_append(cache, k.cuda(), v.cuda(), q.cuda(), None if rot is None else rot.to("cuda"), opt(positions), opt(cnt),
                                     opt(wq), opt(wk))
        pos = positions if positions is not None else lens[:, None].clamp(min=0) + torch.arange(T)
        inv = None if rot is None else rot.inv_freq
        want_q, want_k = (orc.rotate(x, pos, inv, layout, 1.0, w) for x, w in ((q, wq), (k, wk)))
        terms = lambda y: torch.finfo(dtype).eps / 2 * y.abs() + 2.0 ** -20 * 2 * y.abs().amax(-1, keepdim=True) + 2.0 ** -25
        kp2, vp2 = kp.clone(), vp.clone()
        written = torch.zeros(kp.shape[0], page, dtype=torch.bool)
        gk, gv = cache.k_pages.cpu(), cache.v_pages.cpu()
        for b, t, p, row in orc.slots(table, lens, cnt, T, page, kp.shape[0]):
            assert ((gk[p, :, row].double() - want_k[b, :, t]).abs() <= terms(want_k[b, :, t])).all()
            assert torch.equal(gv[p, :, row], v[b, :, t])
            written[p, row] = True
        for now, old in ((gk, kp2), (gv, vp2)):   # everything else is as it was, bit for bit
            rest = ~written[:, None, :, None].expand_as(old)
            assert torch.equal(now.view(torch.int16)[rest], old.view(torch.int16)[rest])
        live = torch.arange(T) < (torch.tensor([T] * B) if cnt is None else cnt)[:, None]
        want_q = torch.where(live[:, None, :, None], want_q, torch.zeros(()).double())
        assert ((got.cpu().double() - want_q).abs() <= terms(want_q)).all()
        assert torch.equal(cache.lengths.cpu(), lens)
        # without q: the same pages
        again = on_gpu(kp, vp, table, lens)
        assert omni.omni_cache_append(again, k.cuda(), v.cuda(), None, None if rot is None else rot.to("cuda"), opt(positions), opt(cnt), None,
                                      opt(wk)) is None
        assert torch.equal(again.k_pages.view(torch.int16), cache.k_pages.view(torch.int16))
        assert torch.equal(again.v_pages.view(torch.int16), cache.v_pages.view(torch.int16))


def test_append_where_there_is_no_page(cuda_device):
    kp, vp, table, lens, g = make_cache(3, 2, 64, 16, [14, 14, 14], 6, torch.float16)
    k, v = (torch.randn(3, 2, 6, 64, generator=g).half() for _ in range(2))
    table[0, 1] = -1
    table[1, 1] = kp.shape[0]
    lens[2] = 30           # two slots left in the table
    cache = on_gpu(kp, vp, table, lens)
    omni.omni_cache_append(cache, k.cuda(), v.cuda())
    gk = cache.k_pages.cpu()
    want = kp.clone()
    for b, t, p, row in orc.slots(table, lens, None, 6, 16, kp.shape[0]):
        want[p, :, row] = k[b, :, t]
    assert torch.equal(gk.view(torch.int16), want.view(torch.int16))
    with pytest.raises(omni.OmniAttnError, match="page_table"):
        omni.omni_cache_append(cache, k.cuda(), v.cuda(), check_status=True)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_strides_and_alignment(cuda_device, layout):
    kp, vp, table, lens, g = make_cache(2, 2, 64, 16, [20, 33], 3, torch.bfloat16)
    base = torch.randn(2, 3, 8, 64, generator=g).bfloat16().cuda()      # fused projection: 4 query, 2 key, 2 value heads
    q, k, v = base.transpose(1, 2).split([4, 2, 2], 1)
    rot = omni.OmniRotary.from_base(64, layout=layout, device="cuda")
    first = on_gpu(kp, vp, table, lens)
    q1 = omni.omni_cache_append(first, k.contiguous(), v.contiguous(), q.contiguous(), rot)
    out1 = omni.omni_cache_attention(q1, first)
    shifted = torch.zeros(2, 3, 8, 65, dtype=torch.bfloat16, device="cuda")
    shifted[..., 1:] = base
    for src in (base, shifted[..., 1:], base.transpose(2, 3).contiguous().transpose(2, 3)):
        a, b, c = src.transpose(1, 2).split([4, 2, 2], 1)
        cache = on_gpu(kp, vp, table, lens)
        wide = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
        wide[:, 2:2 + table.shape[1]] = cache.page_table
        cache.page_table = wide[:, 2:2 + table.shape[1]]
        q2 = omni.omni_cache_append(cache, b, c, a, rot)
        assert torch.equal(q2, q1) and torch.equal(cache.k_pages.view(torch.int16), first.k_pages.view(torch.int16))
        room = torch.zeros(2, 3, 4, 65, dtype=torch.bfloat16, device="cuda")
        room[..., 1:] = q2.transpose(1, 2)
        for x in (q2, q2.transpose(1, 2).contiguous().transpose(1, 2), room[..., 1:].transpose(1, 2), q2.transpose(2, 3).contiguous().transpose(2, 3)):
            assert torch.equal(omni.omni_cache_attention(x, cache), out1)


def test_offsets_beyond_32_bits(cuda_device):
    """A cache of more than 2^31 elements (and 2^32 bytes): pages at its far end."""
    page, D, Hkv = 1024, 128, 8
    pages = (2 ** 31 + 2 ** 28) // (page * D * Hkv)
    kp, vp = (torch.zeros(pages, Hkv, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 0], [pages - 2, 1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([1020, 3], dtype=torch.int32, device="cuda")
    cache = omni.OmniPagedCache(kp, vp, table, lengths)
    g = torch.Generator(device="cuda").manual_seed(5)
    for p in (0, 1, pages - 1, pages - 2):
        kp[p].normal_(generator=g)
        vp[p].normal_(generator=g)
    k, v = (torch.randn(2, Hkv, 8, D, generator=g, device="cuda").half() for _ in range(2))
    omni.omni_cache_append(cache, k, v)
    assert torch.equal(kp[pages - 1, :, 1020:], k[0, :, :4]) and torch.equal(vp[0, :, :4], v[0, :, 4:])
    assert torch.equal(kp[pages - 2, :, 3:11], k[1])
    q = torch.randn(2, Hkv, 8, D, generator=g, device="cuda").half()
    got, lse = omni.omni_cache_attention(q, cache, return_lse=True)
    small = [torch.stack((t[pages - 1], t[0], t[pages - 2], t[1])).cpu() for t in (kp, vp)]
    st = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    check(got, lse, *orc.attention(q.cpu(), *small, st, lengths.cpu()), q.cpu(), *small, D ** -0.5, "far pages")


def test_a_captured_step_is_replayed_as_the_cache_grows(cuda_device):
    """Two sequences generate 40 tokens: append, attention and the step of the lengths in one graph, replayed; the same
    steps one call at a time, and the whole result against 64 bits."""
    B, H, Hkv, D, page = 2, 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    xs = [[torch.randn(B, h, 1, D, generator=g, device="cuda").half() for h in (H, Hkv, Hkv)] for _ in range(40)]
    rot = omni.OmniRotary.from_base(D, device="cuda")

    def fresh():
        c = omni.OmniPagedCache.allocate(8, Hkv, page, D, B, 4, torch.float16)
        c.k_pages.fill_(math.nan)
        c.v_pages.fill_(math.nan)
        c.page_table.copy_(torch.tensor([[3, 1, 6, 0], [2, 7, 5, 4]]))
        c.lengths.copy_(torch.tensor([0, 11]))
        c.k_pages[2, :, :11].zero_()
        c.v_pages[2, :, :11].zero_()
        return c

    eager = fresh()
    outs = []
    for q, k, v in xs:
        outs.append(omni.omni_cache_attention(omni.omni_cache_append(eager, k, v, q, rot), eager, softcap=50.0))
        eager.lengths.add_(1)
    cache = fresh()
    inp = [t.clone() for t in xs[0]]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):   # two captured steps, replayed in turn and side by side with eager calls on another cache
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = omni.omni_cache_attention(omni.omni_cache_append(cache, inp[1], inp[2], inp[0], rot), cache, softcap=50.0)
            cache.lengths.add_(1)
        graphs.append((graph, out))
    other = fresh()
    for i, x in enumerate(xs):
        for dst, src in zip(inp, x):
            dst.copy_(src)
        graph, out = graphs[i % 2]
        graph.replay()
        omni.omni_cache_attention(x[0], other)
        assert torch.equal(out, outs[i]), f"step {i}"
    assert torch.equal(cache.lengths, eager.lengths)
    want = orc.attention(omni.omni_rotary(xs[-1][0], None, rot, (eager.lengths - 1)[:, None].contiguous())[0].cpu(), eager.k_pages.cpu(),
                         eager.v_pages.cpu(), eager.page_table.cpu(), eager.lengths.cpu() - 1, softcap=50.0)
    check(outs[-1], None, *want, xs[-1][0].cpu(), eager.k_pages.cpu(), eager.v_pages.cpu(), D ** -0.5, "last step")


@pytest.mark.parametrize("H", [8, 64])
def test_two_streams_at_once(cuda_device, H):
    kp, vp, table, lens, g = make_cache(4, 2, 128, 64, [3000, 100, 2000, 7], 1, torch.bfloat16)
    cache = on_gpu(kp, vp, table, lens)
    qs = [torch.randn(4, H, 1, 128, generator=g).bfloat16().cuda() for _ in range(2)]
    want = [omni.omni_cache_attention(q, cache) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(omni.omni_cache_attention(qs[i], cache))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_a_denoised_block_is_written_again(cuda_device):
    """An image's tokens appended twice at the same lengths: the second pass replaces the first."""
    kp, vp, table, lens, g = make_cache(2, 2, 64, 16, [37, 5], 40, torch.float16)
    cache = on_gpu(kp, vp, table, lens)
    for _ in range(2):
        q, k, v = (torch.randn(2, h, 40, 64, generator=g).half().cuda() for h in (4, 2, 2))
        omni.omni_cache_append(cache, k, v)
        got, lse = omni.omni_cache_attention(q, cache, causal=False, return_lse=True)
    want = orc.attention(q.cpu(), cache.k_pages.cpu(), cache.v_pages.cpu(), table, lens, causal=False)
    check(got, lse, *want, q.cpu(), cache.k_pages.cpu(), cache.v_pages.cpu(), 64 ** -0.5, "second pass", True)


@pytest.mark.parametrize("H", [4, 48])      # 16-row and 128-row tiles
@pytest.mark.parametrize("lengths", [[300, 20], [9000, 5000]])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(cuda_device, H, lengths):
    """With a budget of one cycle every hand-over that is not there yet counts as run out: the CTAs give up, what they have
    in flight is waited for, the status says so, and the next call is right."""
    from omni_attention_b200 import ops

    kp, vp, table, lens, g = make_cache(2, 2, 64, 64, lengths, 1, torch.float16)
    q = torch.randn(2, H, 1, 64, generator=g).half().cuda()
    cache = on_gpu(kp, vp, table, lens)
    want = omni.omni_cache_attention(q, cache, check_status=True)
    lib = ops.load_library()
    lib.omni_attn_set_wait_cycles(1)
    try:
        with pytest.raises(omni.OmniAttnError, match="gave up waiting"):
            omni.omni_cache_attention(q, cache, check_status=True)
    finally:
        lib.omni_attn_set_wait_cycles(0)       # back to the default budget
    assert torch.equal(omni.omni_cache_attention(q, cache, check_status=True), want)


@pytest.mark.parametrize("H,prefix", [(8, 0), (64, 0), (8, 1024)])
def test_graphs_side_by_side(cuda_device, H, prefix):
    """Two captured calls replayed at once on two streams: each has a workspace of its own."""
    kp, vp, table, lens, g = make_cache(4, 2, 128, 64, [6000, 1100, 3000, 1024], 1, torch.bfloat16, shared=prefix)
    cache = on_gpu(kp, vp, table, lens)
    qs = [torch.randn(4, H, 1, 128, generator=g).bfloat16().cuda() for _ in range(2)]
    want = [omni.omni_cache_attention(q, cache, shared_prefix=prefix) for q in qs]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(omni.omni_cache_attention(q, cache, shared_prefix=prefix))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_a_captured_step_among_copies_and_other_streams(cuda_device):
    """A captured step whose kernels stand behind copies, another stream's work and each other, as launches that may begin
    before their predecessor ends do: the values are those of the same calls with a wait after each."""
    B, H, Hkv, D, page, T = 3, 4, 2, 64, 16, 2
    kp, vp, table, lens, g = make_cache(B, Hkv, D, page, [1500, 40, 700], T, torch.float16)
    rot = omni.OmniRotary.from_base(D, device="cuda")
    src = [torch.randn(B, h, T, D, generator=g).half().cuda() for h in (H, Hkv, Hkv)]
    weight = (1 + 0.1 * torch.randn(D, generator=g)).cuda()

    def step(cache, x, wait=lambda: None, side=None):
        q, k, v = (t.clone() for t in x)                       # copies
        wait()
        if side is not None:                                   # keys from another stream
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                k = k * 2
            torch.cuda.current_stream().wait_stream(side)
        else:
            k = k * 2
        wait()
        q, _ = omni.omni_rotary(q, None, None, None, weight)
        wait()
        q = omni.omni_cache_append(cache, k, v, q, rot)
        wait()
        out, lse = omni.omni_cache_attention(q, cache, return_lse=True)
        wait()
        again = omni.omni_cache_attention(q, cache, shared_prefix=0, causal=False)
        wait()
        q2, _ = omni.omni_rotary(out, None, rot)
        wait()
        return out, lse, again, q2

    plain = on_gpu(kp, vp, table, lens)
    want = step(plain, src, torch.cuda.synchronize)
    cache, side = on_gpu(kp, vp, table, lens), torch.cuda.Stream()
    inp = [torch.zeros_like(t) for t in src]
    step(cache, inp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, inp, side=side)
    for dst, x in zip(inp, src):
        dst.copy_(x)
    for _ in range(10):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(cache.k_pages.view(torch.int16), plain.k_pages.view(torch.int16))
    for a, b in zip(step(cache, src), want):                   # and without a graph
        assert torch.equal(a, b)


def test_host_threads_on_one_stream(cuda_device):
    """Calls that threads enqueue onto one stream, in whatever order their launches interleave."""
    import threading

    kp, vp, table, lens, g = make_cache(4, 2, 128, 64, [3000, 100, 2100, 1024], 1, torch.bfloat16, shared=64)
    cache = on_gpu(kp, vp, table, lens)
    calls = []
    for H, prefix in ((8, 0), (64, 0), (8, 64), (32, 64)):
        q = torch.randn(4, H, 1, 128, generator=g).bfloat16().cuda()
        calls.append((q, prefix, omni.omni_cache_attention(q, cache, shared_prefix=prefix)))
    torch.cuda.synchronize()
    wrong = []

    def work(q, prefix, want):
        outs = [omni.omni_cache_attention(q, cache, shared_prefix=prefix) for _ in range(40)]
        torch.cuda.current_stream().synchronize()
        wrong.extend(1 for o in outs if not torch.equal(o, want))

    threads = [threading.Thread(target=work, args=c) for c in calls]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_a_backward_does_not_use_pages_written_since(cuda_device):
    """Pages that an autograd graph saved and that are appended to before its backward: an error, as behind k_pages.add_(...)."""
    c = omni.OmniPagedCache.allocate(4, 1, 16, 32, 1, 4, torch.float16, cuda_device)
    c.page_table.copy_(torch.arange(4, dtype=torch.int32)[None])
    new = torch.ones(1, 1, 3, 32, dtype=torch.float16, device=cuda_device)
    for pages in (c.k_pages, c.v_pages):
        x = torch.ones(32, dtype=torch.float16, device=cuda_device, requires_grad=True)
        y = (pages * x).sum()
        with torch.no_grad():
            omni.omni_cache_append(c, new, new)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        c = omni.OmniPagedCache.allocate(4, 1, 16, 32, 1, 4, torch.float16, cuda_device)
        c.page_table.copy_(torch.arange(4, dtype=torch.int32)[None])
        omni.omni_cache_append(c, new, new)
        assert torch.equal(c.k_pages[0, 0, :3], new[0, 0])
