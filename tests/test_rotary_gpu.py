"""omni_rotary against its definition in 64 bits: both layouts, part of the head, every dtype, norms, strides, far positions,
gradients.

Tolerances. A result is rounded once: at most half a step, eps / 2 of its value. Before that, in 32 bits: a cosine or sine
is off by less than 2^-22 (its argument, a fraction of half a turn, has 24 bits; sincospif adds an ulp), the norm's factor by
4 * 2^-24 of itself (D terms added up by up to 16 threads in pairs: 7 roundings, halved by the root; rsqrtf 2 ulp), two
products and a sum add 3 * 2^-24 of their terms: together less than 2^-20 of |u| + |v|, the largest element a row holds after its norm
twice. ROUND(...) counts that, and 2^-25 where an fp16 result is subnormal."""
import math

import pytest
import torch

import omni_attention_b200 as omni
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu


def bound(y, dtype, terms, ulps=1.0):
    return torch.finfo(dtype).eps / 2 * y.abs() + ulps * 2.0 ** -20 * terms + (2.0 ** -25 if dtype == torch.float16 else 0)


def check(got, want, dtype, terms, what, ulps=1.0):
    err = (got.detach().double().cpu() - want).abs()
    tol = bound(want, dtype, terms, ulps)
    assert got.shape == want.shape and not torch.isnan(got).any(), what
    worst = float((err / tol).max())
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance, max err {float(err.max()):.3g}"


def make(B, H, Hkv, N, D, dtype, norm=None, wdtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(B, h, N, D, generator=g).to(dtype) for h in (H, Hkv))
    if norm is None:
        return q, k, None, None
    shape = lambda h: (D,) if norm == "shared" else (h, D)
    return q, k, *((1 + 0.3 * torch.randn(shape(h), generator=g)).to(wdtype) for h in (H, Hkv))


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


CASES = [  # B, H, Hkv, N, D, rotary_dim, layout, norm, dtype
    (1, 1, 1, 1, 64, 64, "interleaved", None, torch.bfloat16),
    (2, 4, 2, 7, 128, 128, "interleaved", "shared", torch.bfloat16),
    (2, 3, 1, 33, 128, 128, "half", "head", torch.float16),
    (1, 5, 5, 65, 64, 64, "half", None, torch.float16),
    (3, 2, 2, 129, 32, 32, "interleaved", "head", torch.float32),
    (1, 8, 4, 70, 32, 8, "half", "shared", torch.bfloat16),      # rotary_dim / 2 = 4: elements one by one
    (1, 2, 1, 40, 64, 20, "half", None, torch.float32),
    (2, 2, 1, 31, 64, 6, "interleaved", "shared", torch.float16),
    (1, 4, 4, 50, 128, 32, "half", "shared", torch.float32),
    (1, 2, 2, 17, 128, 2, "half", None, torch.bfloat16),
    (1, 40, 8, 300, 128, 64, "interleaved", None, torch.bfloat16),
    (1, 2, 2, 1000, 64, 64, "interleaved", "shared", torch.bfloat16),
]


@pytest.mark.parametrize("B,H,Hkv,N,D,rd,layout,norm,dtype", CASES)
def test_forward_and_backward(cuda_device, B, H, Hkv, N, D, rd, layout, norm, dtype):
    q, k, wq, wk = make(B, H, Hkv, N, D, dtype, norm, torch.float32 if norm == "shared" else dtype)
    rot = omni.OmniRotary.from_base(rd, layout=layout, device="cuda")
    pos = torch.randint(0, 200000, (B, N), generator=torch.Generator().manual_seed(1))
    leaves = [t.requires_grad_() for t in cuda(q, k, wq, wk) if t is not None]
    out = omni.omni_rotary(leaves[0], leaves[1], rot, pos.cuda(), *leaves[2:])
    gq, gk = make(B, H, Hkv, N, D, dtype, seed=2)[:2]
    grads = torch.autograd.grad(out, leaves, cuda(gq, gk))
    for i, (x, w, g, name) in enumerate(((q, wq, gq, "q"), (k, wk, gk, "k"))):
        ref = x.double().requires_grad_()
        rw = None if w is None else w.double().requires_grad_()
        y = orc.rotate(ref, pos, rot.inv_freq.cpu(), layout, 1.0, rw)
        terms = 2 * y.detach().abs().amax(-1, keepdim=True)
        check(out[i], y.detach(), dtype, terms, name)
        y.backward(g.double())
        gmax = 2 * g.double().abs().amax(-1, keepdim=True)
        if w is None:
            check(grads[i], ref.grad, dtype, gmax, f"d{name}")
            continue
        # dx = r (gw - x_hat mean(gw x_hat)): terms up to r |g| |w| (1 + |x_hat| max|x_hat|), each a few roundings
        r = 1 / (x.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        xh = (x.double() * r).abs().amax(-1, keepdim=True)
        check(grads[i], ref.grad, dtype, r * gmax * w.double().abs().max() * (1 + xh * xh), f"d{name}", ulps=2)
        # dw: a sum of M products in 32 bits, in blocks: rounding grows like the square root of a block's length at most, a
        # fifth of 2^-20 per term is far above it
        full = (orc.rotate(g, pos, rot.inv_freq.cpu(), layout, 1.0).abs().amax() * xh.max()) * x.shape[0] * x.shape[2] * (
            x.shape[1] if w.dim() == 1 else 1)
        check(grads[2 + i], rw.grad, w.dtype, 0.2 * full, f"d{name}_weight")


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_gradients_of_fp32_weights_have_exact_angles(cuda_device, dtype, layout):
    """A row of ones without eps has the norm 1, and the gradient (1, 0) of each pair makes the weight's gradient the pair's cosine
    and minus its sine, with no rounding beside theirs: in 32 bits, whatever the data's dtype. A cosine or sine is off by less
    than 2^-22 (see above)."""
    D, calls = 128, 200
    rot = omni.OmniRotary.from_base(D, layout=layout, device="cuda")
    first = (slice(0, D, 2), slice(1, D, 2)) if layout == "interleaved" else (slice(0, D // 2), slice(D // 2, D))
    x = torch.ones(1, 1, 1, D, dtype=dtype, device="cuda")
    g = torch.zeros_like(x)
    g[..., first[0]] = 1
    positions = torch.randint(0, 100000, (calls, 1), generator=torch.Generator().manual_seed(2))
    worst = 0.0
    for pos in positions:
        w = torch.ones(D, device="cuda", requires_grad=True)
        dw, = torch.autograd.grad(omni.omni_rotary(x, None, rot, pos.cuda(), w, eps=0.0)[0], w, g)
        a = pos.double() * rot.inv_freq.cpu()
        dw = dw.double().cpu()
        worst = max(worst, float((dw[first[0]] - a.cos()).abs().max()), float((dw[first[1]] + a.sin()).abs().max()))
    assert worst <= 2.0 ** -22, f"2^{math.log2(worst):.2f}"


@pytest.mark.parametrize("norm", [None, "shared", "head"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sixteen_bit_results(cuda_device, dtype, layout, norm):
    """fp16 and bf16 results use the special function unit: a cosine or sine is off by 2^-21.2 (the unit's own error within half a
    turn), 2^-23.4 (the turns in 32 bits), 2^-23 (their product with 2 pi) and 2^-23.4 (2 pi itself), less than 2^-20.4 together. The
    norm's factor adds 2^-22, two products and a sum 3 * 2^-24: less than 2^-19.7 of |u| + |v| for the pair (u, v), then the rounding."""
    D = 128
    q, _, w, _ = make(2, 3, 1, 300, D, dtype, norm, torch.float32, seed=11)
    pos = torch.randint(0, 200000, (2, 300), generator=torch.Generator().manual_seed(12))
    rot = omni.OmniRotary.from_base(D, layout=layout, device="cuda")
    got, _ = omni.omni_rotary(q.cuda(), None, rot, pos.cuda(), None if w is None else w.cuda())
    want = orc.rotate(q, pos, rot.inv_freq.cpu(), layout, 1.0, w)
    before = orc.rotate(q, pos, None, weight=w).abs()
    if layout == "interleaved":
        terms = (before[..., 0::2] + before[..., 1::2]).repeat_interleave(2, -1)
    else:
        terms = (before[..., :D // 2] + before[..., D // 2:]).repeat(1, 1, 1, 2)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -19.7 * terms + (2.0 ** -25 if dtype == torch.float16 else 0)
    worst = float(((got.double().cpu() - want).abs() / tol).max())
    assert worst <= 1.0, f"{worst:.3g} times the tolerance"


@pytest.mark.parametrize("where", [0, 1 << 20, 3_000_000_000])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_far_positions_are_as_exact_as_near_ones(cuda_device, where, layout):
    q, k, _, _ = make(1, 2, 1, 64, 128, torch.float32)
    pos = torch.arange(64)[None] + where
    rot = omni.OmniRotary.from_base(128, layout=layout, device="cuda")
    got, _ = omni.omni_rotary(q.cuda(), None, rot, pos.cuda())
    want = orc.rotate(q, pos, rot.inv_freq.cpu(), layout)
    # the angle in 64 bits: off by 2^-52 of itself
    check(got, want, torch.float32, 2 * want.abs().amax(-1, keepdim=True) * (1 + where * 2.0 ** -32), f"position {where}")


def test_positions_forms_and_scaling(cuda_device):
    q, k, _, _ = make(2, 2, 2, 9, 64, torch.float32)
    q, k = cuda(q, k)
    for scaling in (None, {"type": "linear", "factor": 4}, {"type": "ntk", "factor": 8},
                    {"type": "yarn", "factor": 8, "original_length": 512}):
        rot = omni.OmniRotary.from_base(64, scaling=scaling, device="cuda")
        pos = torch.arange(9).expand(2, 9)
        want = orc.rotate(q.cpu(), pos, rot.inv_freq.cpu(), "interleaved", rot.factor)
        for p in (None, pos[0].cuda(), pos[:1].int().cuda(), pos.cuda(), pos.contiguous().int().cuda(),
                  torch.arange(18).cuda()[::2] // 2, torch.arange(9).cuda()[:, None].expand(9, 2).t()):
            got, _ = omni.omni_rotary(q, None, rot, p)
            check(got, want, torch.float32, 2 * want.abs().amax(-1, keepdim=True), f"{scaling} {None if p is None else p.shape}")
        _, got = omni.omni_rotary(None, q, rot)     # as keys
        check(got, want, torch.float32, 2 * want.abs().amax(-1, keepdim=True), "keys alone")


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_strided_and_unaligned_inputs_give_the_same_bits(cuda_device, layout):
    q, k, wq, wk = cuda(*make(2, 4, 2, 21, 64, torch.bfloat16, "shared"))
    rot = omni.OmniRotary.from_base(32, layout=layout, device="cuda")
    want = omni.omni_rotary(q, k, rot, None, wq, wk)
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def views(t):
        yield t.transpose(1, 2).contiguous().transpose(1, 2)                     # the projections' layout
        wide = torch.empty(*t.shape[:3], 80, dtype=t.dtype, device="cuda")
        wide[..., 3:67] = t
        yield wide[..., 3:67]                                                    # rows off their 16-byte boundaries
        yield t.transpose(2, 3).contiguous().transpose(2, 3)                     # strided along D
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        yield flat[1:].view(t.shape)
    first = None
    for a, b in zip(views(q), views(k)):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        got = omni.omni_rotary(a, b, rot, None, wq, wk)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for u, v in zip(views(gq), views(gk)):
            grads = torch.autograd.grad(got, (a, b), (u, v), retain_graph=True)
            first = grads if first is None else first
            assert torch.equal(grads[0], first[0]) and torch.equal(grads[1], first[1])
    # expanded along the batch: read as it is; its gradient is summed by autograd
    one = q[:1].detach().requires_grad_()
    out, _ = omni.omni_rotary(one.expand(2, 4, 21, 64), None, rot, None, wq)
    g, = torch.autograd.grad(out, one, gq)
    parts = [torch.autograd.grad(omni.omni_rotary(one, None, rot, None, wq)[0], one, gq[i:i + 1])[0].double() for i in (0, 1)]
    assert float((g.double() - parts[0] - parts[1]).abs().max()) <= 3 * 2.0 ** -8 * float(parts[0].abs().max() + parts[1].abs().max())


def test_gradients_of_what_is_asked_for(cuda_device):
    q, k, wq, wk = cuda(*make(1, 2, 2, 12, 64, torch.float32, "head"))
    rot = omni.OmniRotary.from_base(64, device="cuda")
    everything = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    full = torch.autograd.grad([o.square().sum() for o in omni.omni_rotary(everything[0], everything[1], rot, None, *everything[2:])], everything)
    for i in range(4):   # one leaf at a time
        ts = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, wq, wk))]
        a, b = omni.omni_rotary(ts[0], ts[1], rot, None, ts[2], ts[3])
        (a.square().sum() + b.square().sum()).backward()
        assert torch.equal(ts[i].grad, full[i]) and all(t.grad is None for j, t in enumerate(ts) if j != i)
    a, _ = omni.omni_rotary(*everything[:2], rot, None, *everything[2:])     # k's result is not used
    gs = torch.autograd.grad(a.square().sum(), everything, allow_unused=True)
    assert torch.equal(gs[0], full[0]) and torch.equal(gs[2], full[2])
    assert all(g is None or not g.any() for g in (gs[1], gs[3]))
    # a norm on one of the two only
    a, b = omni.omni_rotary(*everything[:2], rot, None, everything[2])
    gs = torch.autograd.grad((a.square().sum() + b.square().sum()), everything[:3])
    assert torch.equal(gs[0], full[0]) and torch.equal(gs[2], full[2])
    want = torch.autograd.grad(omni.omni_rotary(None, everything[1], rot)[1].square().sum(), everything[1])[0]
    assert torch.equal(gs[1], want)


def test_gradients_against_differences(cuda_device):
    """fp32, central differences of a smooth function of both results at step 1e-2 in 64-bit sums: the truncation is
    h^2 / 6 of a third derivative of order one, the 32-bit outputs' rounding 2^-24 * 100 / h."""
    q, k, wq, wk = cuda(*make(1, 2, 1, 3, 32, torch.float32, "shared"))
    rot = omni.OmniRotary.from_base(16, layout="half", device="cuda")
    f = lambda ts: sum(torch.sin(o.double()).sum() for o in omni.omni_rotary(ts[0], ts[1], rot, None, ts[2], ts[3]))
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(f(leaves), leaves)
    g = torch.Generator().manual_seed(3)
    for i in range(4):
        d = torch.randn(leaves[i].shape, generator=g).cuda()
        d /= d.norm()
        h = 1e-2
        with torch.no_grad():
            at = lambda s: f([t + (s * h * d if j == i else 0) for j, t in enumerate(leaves)])
            num = float((at(1) - at(-1)) / (2 * h))
        assert abs(num - float((grads[i] * d).sum())) <= 2e-3 * max(1.0, abs(num))


def test_captured_replayed_and_on_another_stream(cuda_device):
    q, k, wq, wk = cuda(*make(2, 4, 2, 100, 64, torch.bfloat16, "shared"))
    rot = omni.OmniRotary.from_base(64, device="cuda")
    pos = torch.arange(100, device="cuda").expand(2, 100).contiguous()
    run = lambda: omni.omni_rotary(q, k, rot, pos, wq, wk)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    q.normal_()
    pos.add_(77)
    graph.replay()
    want = run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    side.synchronize()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_infinite_and_zero_rows_stay_where_they_are(cuda_device):
    q, k, wq, _ = make(1, 2, 2, 8, 64, torch.bfloat16, "shared")
    q[0, 0, 3] = math.nan
    q[0, 1, 5, 7] = math.inf
    q[0, 1, 6] = 0
    rot = omni.OmniRotary.from_base(64, device="cuda")
    out, _ = omni.omni_rotary(q.cuda(), None, rot, None, wq.cuda())
    clean = torch.ones(2, 8, dtype=torch.bool)
    clean[0, 3] = clean[1, 5] = False
    assert torch.isfinite(out[0].cpu()[clean]).all() and not torch.isfinite(out[0, 0, 3]).any()
    assert not out[0, 1, 6].any()


@pytest.mark.parametrize("D,rd", [(64, 32), (64, 20), (64, 6), (128, 64), (128, 2), (32, 8), (32, 16)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_not_rotated_passes_through(cuda_device, D, rd, layout, dtype):
    """Every element behind rotary_dim comes out bit for bit, an infinite or NaN neighbour or not; the same in the gradients."""
    q, g, _, _ = make(2, 3, 3, 19, D, dtype)
    marks = torch.tensor([math.inf, -math.inf, math.nan], dtype=dtype)
    at = torch.rand(q.shape, generator=torch.Generator().manual_seed(4))
    at[..., :rd] = 1.0
    for t in (q, g):
        where = at < 0.3
        t[where] = marks[torch.arange(int(where.sum())) % 3]
    rot = omni.OmniRotary.from_base(rd, layout=layout, device="cuda")
    x = q.cuda().requires_grad_()
    y, _ = omni.omni_rotary(x, None, rot)
    dx, = torch.autograd.grad(y, x, g.cuda())
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(nan=7.0), b.nan_to_num(nan=7.0)) and torch.equal(a.cpu().isnan(), b.isnan())
    for got, given in ((y.detach(), q), (dx, g)):
        assert torch.isfinite(got[..., :rd]).all() and same(got[..., rd:], given[..., rd:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_normed_rows_with_an_infinite_element(cuda_device, dtype):
    """By the definition: the row's factor is 0, its finite elements come out 0 and the infinite one NaN; rotation mixes it with
    the other member of its pair, and with nothing that is not rotated."""
    q, _, w, _ = make(1, 2, 1, 4, 64, dtype, "shared")
    q[0, 0, 1, 40], q[0, 1, 2, 4] = math.inf, -math.inf
    rot = omni.OmniRotary.from_base(32, device="cuda")
    got = omni.omni_rotary(q.cuda(), None, rot, None, w.cuda())[0].cpu()
    want = orc.rotate(q, torch.arange(4)[None], rot.inv_freq.cpu(), weight=w)
    assert torch.equal(got.isnan(), want.isnan()) and int(want.isnan().sum()) == 3
    assert not got[0, 0, 1, :40].any() and not got[0, 0, 1, 41:].any()


def test_no_second_derivative(cuda_device):
    q = torch.randn(1, 1, 4, 32, device="cuda", requires_grad=True)
    out, _ = omni.omni_rotary(q, None, omni.OmniRotary.from_base(32, device="cuda"))
    with pytest.raises(omni.OmniAttnError, match="second derivative"):
        torch.autograd.grad(out.square().sum(), q, create_graph=True)


@pytest.mark.parametrize("alive", ["nothing", "default", "side"])
def test_a_captured_backward_and_graphs_of_the_same_leaves(cuda_device, alive):
    """An eager graph of the leaves that lives on the default stream would end the capture inside autograd: refused before that."""
    q, k, wq, wk = cuda(*make(1, 2, 1, 40, 64, torch.bfloat16, "shared"))
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    rot = omni.OmniRotary.from_base(64, device="cuda")
    go = [torch.randn_like(x) for x in (q, k)]
    run = lambda: omni.omni_rotary(q, k, rot, None, wq, wk)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = torch.autograd.grad(run(), leaves, go)
        kept = run() if alive == "side" else None
    torch.cuda.current_stream().wait_stream(side)
    if alive == "default":
        kept = run()
    graph, got = torch.cuda.CUDAGraph(), None
    try:
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(run(), leaves, go)
    except omni.OmniAttnError as e:
        assert alive == "default" and "captured" in str(e)
    assert (got is None) == (alive == "default")
    if got is not None:
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del kept
    again = torch.autograd.grad(run(), leaves, go)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
