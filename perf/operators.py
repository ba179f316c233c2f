"""The operators next to the block-mask attention, as measurable cases: rotary positions with the norms of queries and
keys (training and prefill), and the paged key/value cache of generation (append, attention, shared prefix).

A case is one pass of a user's program:

  op = "rotary"  omni_rotary(q, k, rotary, positions, q_weight, k_weight); with train also the gradients of all of these
       "append"  omni_cache_append(cache, k, v, q, ...): the new tokens' keys (normed, rotated) and values into the
                 pages, their queries rotated in the same call
       "attend"  omni_cache_attention(q, cache, ...): the new tokens' attention over cache and themselves; with
                 shared > 0 the sequences have their first `shared` tokens in the same pages

q, k and v are what a projection leaves: views [B, H, N, D] of [B, N, H, D] memory. `context` is the longest sequence's
number of cached tokens, T the number of new ones; the sequences' lengths, the order of the pages and the data come from
the seed.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def _rotary(name, B, H, Hkv, N, D, rd, layout, norm, dtype, train, scaling="none", far=0):
    c = dict(op="rotary", B=B, H=H, Hkv=Hkv, N=N, D=D, rd=rd, layout=layout, norm=norm, dtype=dtype, train=train,
             scaling=scaling, far=far)
    return dict(c, name=name) if name else c


def _append(name, B, H, Hkv, T, D, rd, layout, norm, dtype, page, context, ragged):
    c = dict(op="append", B=B, H=H, Hkv=Hkv, T=T, D=D, rd=rd, layout=layout, norm=norm, dtype=dtype, page=page,
             context=context, ragged=ragged)
    return dict(c, name=name) if name else c


def _attend(name, B, H, Hkv, T, D, dtype, page, context, causal=True, softcap=0.0, lse=False, ragged=True, shared=0):
    c = dict(op="attend", B=B, H=H, Hkv=Hkv, T=T, D=D, dtype=dtype, page=page, context=context, causal=causal,
             softcap=softcap, lse=lse, ragged=ragged, shared=shared)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a short training step of a small Transfusion-style model: launches count
        _rotary("rotary train 512", 1, 8, 8, 512, 64, 64, "interleaved", "none", "bf16", True),
        # one layer of the 8K training workload with normed queries and keys
        _rotary("norm rotary train 8192", 1, 32, 32, 8192, 128, 128, "interleaved", "shared", "bf16", True),
        # prefill of a ragged length at far positions, grouped heads, half of the head rotated, scaled frequencies
        _rotary("norm rotary prefill 1999", 2, 32, 8, 1999, 128, 64, "half", "head", "fp16", False, "yarn", 120000),
        # one token of one sequence
        _append("append 1 token", 1, 16, 16, 1, 64, 64, "interleaved", "none", "fp16", 16, 500, False),
        # a serving batch's step
        _append("append batch 64", 64, 32, 8, 1, 128, 128, "half", "shared", "bf16", 64, 4096, True),
        # prompts of different lengths go into the cache
        _append("append prompt 4096", 4, 32, 8, 4096, 128, 128, "interleaved", "none", "bf16", 64, 300, True),
        # one token of one short sequence, the Transfusion slot's soft-cap: latency counts
        _attend("decode 512 softcap", 1, 16, 16, 1, 64, "fp16", 16, 512, softcap=50.0, ragged=False),
        # a serving batch of different lengths
        _attend("decode ragged 8192", 16, 32, 8, 1, 128, "bf16", 64, 8192, lse=True),
        # two very long sequences: work split over the keys
        _attend("decode long 131072", 2, 32, 8, 1, 128, "bf16", 128, 131071, ragged=False),
        # an image being denoised: its tokens attend to the context and to each other
        _attend("image block 256", 2, 32, 32, 256, 128, "bf16", 64, 4096, causal=False, ragged=False),
        # a few continuations of one prompt
        _attend("prefix 2048 x 16", 16, 16, 16, 1, 64, "fp16", 64, 2300, shared=2048),
        # many continuations of one long prompt
        _attend("prefix 16384 x 64", 64, 32, 8, 1, 128, "bf16", 64, 17000, shared=16384),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    D, dtype = rng.choice([32, 64, 64, 128, 128, 128]), rng.choice(["fp16", "bf16", "bf16"])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    H = Hkv * rng.choice([1, 1, 2, 4, 8])
    op = rng.choice(["rotary", "append", "attend", "attend", "prefix"])
    rd = rng.choice([D, D, D // 2, D // 4])
    layout, norm = rng.choice(["interleaved", "half"]), rng.choice(["none", "shared", "head"])
    if op == "rotary":
        B, N = _log(rng, 1, 8), _log(rng, 1, 8192)
        while B * N * (H + Hkv) * D > 8192 * 64 * 128:
            N = max(1, N // 2)
        return _rotary(None, B, H, Hkv, N, D, rd, layout, norm, rng.choice([dtype, dtype, "fp32"]), rng.random() < 0.6,
                       rng.choice(["none", "linear", "yarn"]), rng.choice([0, 5000, 400000]))
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        B, T = _log(rng, 1, 64), _log(rng, 1, 4096)
        while B * T * (H + 2 * Hkv) * D > 4 * 4096 * 48 * 128:
            T = max(1, T // 2)
        return _append(None, B, H, Hkv, T, D, rd, layout, norm, dtype, page, _log(rng, 1, 4096), rng.random() < 0.7)
    B, T, context = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, _log(rng, 6, 300)]), _log(rng, 1, 131072)
    while B * context * Hkv * D > 32 * 8192 * 8 * 128 or B * H * T * (context + T) * D > 2 * 32 * 256 * 4096 * 128:
        context, T = max(1, context // 2), max(1, T * 2 // 3)
    shared = context * rng.randint(1, 9) // 10 // page * page if op == "prefix" else 0
    return _attend(None, B, H, Hkv, T, D, dtype, page, context, rng.random() < 0.6, rng.choice([0.0, 0.0, 30.0, 50.0]),
                   rng.random() < 0.4, rng.random() < 0.7, shared)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _frequencies(rd, scaling):
    """(inv_freq float64 [rd / 2] on the host, factor on cos and sin), base 10000."""
    i = torch.arange(0, rd, 2, dtype=torch.float64)
    inv = 10000.0 ** (-i / rd)
    if scaling == "linear":
        return inv / 4.0, 1.0
    if scaling == "yarn":   # by parts: fast pairs as they are, slow ones stretched 8 times, from 4096 trained positions
        at = lambda turns: rd * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rd // 2 - 1)
        keep = 1.0 - ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv / 8.0 * (1 - keep) + inv * keep, 0.1 * math.log(8.0) + 1.0
    return inv, 1.0


def _views(g, dtype, *shapes):
    """[B, H, N, D] views of [B, N, H, D] memory."""
    return [torch.randn(B, N, H, D, generator=g, device="cuda").to(dtype).transpose(1, 2) for B, H, N, D in shapes]


def _weights(c, g, dtype):
    if c["norm"] == "none":
        return None, None
    shape = lambda h: (c["D"],) if c["norm"] == "shared" else (h, c["D"])
    wdtype = torch.float32 if c["norm"] == "shared" else dtype
    return tuple((1 + 0.3 * torch.randn(shape(h), generator=g, device="cuda")).to(wdtype) for h in (c["H"], c["Hkv"]))


def _cache(c, g, dtype, new):
    """Pages in random order, some of them nobody's; lengths of the sequences before the new tokens."""
    B, page = c["B"], c["page"]
    shared = c.get("shared", 0)
    per = -(-(c["context"] + new) // page)
    spages = shared // page
    pages = spages + B * (per - spages) + 3
    kp, vp = (torch.randn(pages, c["Hkv"], page, c["D"], generator=g, device="cuda").to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.empty(B, per, dtype=torch.int32, device="cuda")
    table[:, :spages] = order[:spages]
    table[:, spages:] = order[spages:spages + B * (per - spages)].view(B, per - spages)
    lengths = torch.full((B,), c["context"], dtype=torch.int32, device="cuda")
    if c["ragged"] and B > 1:
        lengths[1:] = torch.randint(max(shared, c["context"] // 3), c["context"] + 1, (B - 1,), generator=g, device="cuda")
    return kp, vp, table, lengths


def prepare(case, seed):
    c, dtype = case, DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": c}
    if c["op"] == "attend":
        s["q"], = _views(g, dtype, (c["B"], c["H"], c["T"], c["D"]))
        s["kp"], s["vp"], s["table"], s["lengths"] = _cache(c, g, dtype, c["T"])
    else:
        n = c["N"] if c["op"] == "rotary" else c["T"]
        s["q"], s["k"], s["v"] = _views(g, dtype, *[(c["B"], h, n, c["D"]) for h in (c["H"], c["Hkv"], c["Hkv"])])
        s["wq"], s["wk"] = _weights(c, g, dtype)
        inv, s["factor"] = _frequencies(c["rd"], c.get("scaling", "none"))
        s["inv_freq"] = inv.cuda()
        if c["op"] == "rotary":
            # an image's tokens share one position, as in the interleaved model: positions stand still now and then
            move = (torch.rand(c["B"], n, generator=g, device="cuda") < 0.8).long()
            s["positions"] = move.cumsum(1) + c["far"]
            if c["train"]:
                s["gq"], s["gk"] = _views(g, dtype, (c["B"], c["H"], n, c["D"]), (c["B"], c["Hkv"], n, c["D"]))
        else:
            s["kp"], s["vp"], s["table"], s["lengths"] = _cache(c, g, dtype, n)
            s["counts"] = None
            if c["ragged"] and n > 1:
                s["counts"] = torch.randint(max(1, n // 3), n + 1, (c["B"],), generator=g, device="cuda").to(torch.int32)
    if own:   # the handles a program keeps
        import omni_attention_b200 as omni
        if "inv_freq" in s:
            s["rotary"] = omni.OmniRotary(s["inv_freq"], c["layout"], s["factor"])
        if "kp" in s:
            s["cache"] = omni.OmniPagedCache(s["kp"], s["vp"], s["table"], s["lengths"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[s["case"]["op"]](s)


def _run_own(s):
    import omni_attention_b200 as omni
    c = s["case"]
    if c["op"] == "rotary":
        if not c["train"]:
            return omni.omni_rotary(s["q"], s["k"], s["rotary"], s["positions"], s["wq"], s["wk"], eps=EPS)
        leaves = [t.detach().requires_grad_() for t in (s["q"], s["k"], s["wq"], s["wk"]) if t is not None]
        q, k = omni.omni_rotary(leaves[0], leaves[1], s["rotary"], s["positions"], *leaves[2:], eps=EPS)
        return q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (s["gq"], s["gk"]))
    if c["op"] == "append":
        q = omni.omni_cache_append(s["cache"], s["k"], s["v"], q=s["q"], rotary=s["rotary"], counts=s["counts"],
                                   q_weight=s["wq"], k_weight=s["wk"], eps=EPS)
        return q, s["kp"], s["vp"]
    return omni.omni_cache_attention(s["q"], s["cache"], causal=c["causal"], softcap=c["softcap"], return_lse=c["lse"],
                                     shared_prefix=c["shared"])


def _angles(positions, inv_freq, factor):
    """cos and sin [B, 1, N, rd / 2]: the angle in 64 bits (far positions), the rest in 32."""
    t = positions[:, None, :, None].double() * inv_freq
    return (t.cos() * factor).float(), (t.sin() * factor).float()


def _halves(x, rd, layout):
    """The two members of each pair, and what is not rotated."""
    if layout == "interleaved":
        return x[..., 0:rd:2], x[..., 1:rd:2], x[..., rd:]
    return x[..., :rd // 2], x[..., rd // 2:rd], x[..., rd:]


def _joined(a, b, rest, layout):
    pairs = torch.stack((a, b), -1).flatten(-2) if layout == "interleaved" else torch.cat((a, b), -1)
    return torch.cat((pairs, rest), -1)


def _per_head(w):
    """A weight as [.., 1, D] next to [B, H, N, D]."""
    return w.float() if w.dim() == 1 else w.float()[:, None, :]


def _plain_turn(x, w, cos, sin, rd, layout):
    """32 bits in and out."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * _per_head(w)
    a, b, rest = _halves(x, rd, layout)
    return _joined(a * cos - b * sin, a * sin + b * cos, rest, layout)


def _plain_turn_back(x, w, g, cos, sin, rd, layout):
    """Gradients of x and w for the gradient g of the result."""
    a, b, rest = _halves(g, rd, layout)
    g = _joined(a * cos + b * sin, b * cos - a * sin, rest, layout)
    if w is None:
        return g, None
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    x_hat = x * r
    dw = (g * x_hat).sum((0, 2))
    gw = g * _per_head(w)
    return r * (gw - x_hat * (gw * x_hat).mean(-1, keepdim=True)), dw.sum(0) if w.dim() == 1 else dw


def _plain_rotary(s):
    c, dtype = s["case"], s["q"].dtype
    cos, sin = _angles(s["positions"], s["inv_freq"], s["factor"])
    q, k = s["q"].float(), s["k"].float()
    out = [_plain_turn(x, w, cos, sin, c["rd"], c["layout"]).to(dtype) for x, w in ((q, s["wq"]), (k, s["wk"]))]
    if c["train"]:
        back = [_plain_turn_back(x, w, g.float(), cos, sin, c["rd"], c["layout"])
                for x, w, g in ((q, s["wq"], s["gq"]), (k, s["wk"], s["gk"]))]
        out += [dx.to(dtype) for dx, _ in back]
        out += [dw.to(w.dtype) for (_, dw), w in zip(back, (s["wq"], s["wk"])) if w is not None]
    return tuple(out)


def _plain_append(s):
    c, dtype = s["case"], s["q"].dtype
    t = torch.arange(c["T"], device="cuda")
    slots = s["lengths"].long()[:, None] + t                                        # [B, T]
    cos, sin = _angles(slots, s["inv_freq"], s["factor"])
    q, k = (_plain_turn(s[n].float(), s["w" + n], cos, sin, c["rd"], c["layout"]).to(dtype) for n in ("q", "k"))
    live = torch.ones_like(slots, dtype=torch.bool) if s["counts"] is None else t < s["counts"][:, None]
    page = s["table"].long().gather(1, (slots // c["page"]).clamp(max=s["table"].shape[1] - 1))
    page, row = page[live], (slots % c["page"])[live]
    s["kp"][page, :, row] = k.transpose(1, 2)[live]
    s["vp"][page, :, row] = s["v"].transpose(1, 2)[live]
    return torch.where(live[:, None, :, None], q, torch.zeros_like(q)), s["kp"], s["vp"]


def _plain_attend(s):
    c, B, T, D = s["case"], s["case"]["B"], s["case"]["T"], s["case"]["D"]
    G, L = c["H"] // c["Hkv"], c["context"] + T
    k, v = (p[s["table"].long()].transpose(1, 2).reshape(B, c["Hkv"], -1, D)[:, :, :L].float() for p in (s["kp"], s["vp"]))
    q = s["q"].float().reshape(B, c["Hkv"], G * T, D)
    scores = (q @ k.transpose(2, 3)) * D ** -0.5
    if c["softcap"] > 0:
        scores = torch.tanh(scores / c["softcap"]) * c["softcap"]
    t = torch.arange(T, device="cuda")
    limit = s["lengths"].long()[:, None] + (t + 1 if c["causal"] else T)            # [B, T or 1]
    seen = torch.arange(L, device="cuda") < limit.expand(B, T)[:, None, None, :, None]
    seen = seen.expand(B, 1, G, T, L).reshape(B, 1, G * T, L)
    scores = scores.masked_fill(~seen, -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - m)
    l = p.sum(-1, keepdim=True)
    out = ((p @ v) / l).reshape(B, c["H"], T, D).to(s["q"].dtype)
    return (out, (m + torch.log(l)).reshape(B, c["H"], T)) if c["lse"] else out


# ---------------------------------------------------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    c, size = case, 4 if case["dtype"] == "fp32" else 2
    if c["op"] == "rotary":
        n = c["B"] * c["N"] * (c["H"] + c["Hkv"]) * c["D"]
        passes = 2 if not c["train"] else 4 if c["norm"] == "none" else 4   # x, y, and in training also dy, dx
        return {"bytes": n * size * passes + c["B"] * c["N"] * 8, "flops": n * (4 if c["norm"] == "none" else 8) * passes / 2}
    if c["op"] == "append":
        n = c["B"] * c["T"] * c["D"] * (0.7 if c["ragged"] and c["T"] > 1 else 1.0)
        return {"bytes": 2 * size * n * (c["H"] + 2 * c["Hkv"]), "flops": 4 * n * (c["H"] + c["Hkv"])}
    B, T = c["B"], c["T"]
    mean = c["context"] if not c["ragged"] or B == 1 else (c["context"] + max(c["shared"], c["context"] // 3)) / 2
    rows = B * c["H"] * T
    keys = c["shared"] + B * (mean + T - c["shared"])
    return {"bytes": 2 * size * c["Hkv"] * c["D"] * keys + 2 * size * rows * c["D"], "flops": 4 * rows * (mean + T) * c["D"]}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _turned(x, angle, factor, layout):
    """Each pair of x as a complex number, times factor * e^(i angle); angle [B, N, rd / 2]."""
    rd = 2 * angle.shape[-1]
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]
    y = x.clone()
    first, second = (slice(0, rd, 2), slice(1, rd, 2)) if layout == "interleaved" else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _normed(x, w):
    """(x / rms(x) * w, 1 / rms(x))"""
    if w is None:
        return x, None
    rms = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    w = w.double()
    return x / rms * (w if w.dim() == 1 else w.unsqueeze(1)), 1 / rms


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "attend":
        return _exact_attend(c, s)
    if c["op"] == "append":
        pos = (s["lengths"].double()[:, None] + torch.arange(c["T"], device="cuda", dtype=torch.float64))
    else:
        pos = s["positions"].double()
    angle = pos[:, :, None] * s["inv_freq"]
    q, k = (_turned(_normed(s[n].double(), s["w" + n])[0], angle, s["factor"], c["layout"]) for n in ("q", "k"))
    if c["op"] == "append":
        kp, vp = s["kp"].double(), s["vp"].double()
        lengths, counts = s["lengths"].tolist(), [c["T"]] * c["B"] if s["counts"] is None else s["counts"].tolist()
        for b in range(c["B"]):
            at = lengths[b] + torch.arange(counts[b], device="cuda")
            page, row = s["table"][b].long()[at // c["page"]], at % c["page"]
            kp[page, :, row] = k[b, :, :counts[b]].transpose(0, 1)
            vp[page, :, row] = s["v"][b, :, :counts[b]].transpose(0, 1).double()
            q[b, :, counts[b]:] = 0
        return q, kp, vp
    if not c["train"]:
        return q, k
    dx, dw = [], []
    for n in ("q", "k"):
        x, w = s[n].double(), s["w" + n]
        g = _turned(s["g" + n].double(), -angle, s["factor"], c["layout"])
        if w is None:
            dx.append(g)
            continue
        inv = _normed(x, w)[1]
        full = (g * x * inv).sum(2).sum(0)
        dw.append(full.sum(0) if w.dim() == 1 else full)
        g = g * (w.double() if w.dim() == 1 else w.double().unsqueeze(1))
        dx.append(g * inv - x * inv ** 3 * ((g * x).sum(-1, keepdim=True) / x.shape[-1]))
    return q, k, *dx, *dw


def _exact_attend(c, s):
    outs, lses = [], []
    G = c["H"] // c["Hkv"]
    for b, n in enumerate(s["lengths"].tolist()):
        total = n + c["T"]
        pages = s["table"][b, :-(-total // c["page"])].long()
        k, v = (p[pages].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :total].repeat_interleave(G, 0) for p in (s["kp"], s["vp"]))
        x = torch.einsum("htd,hnd->htn", s["q"][b].double(), k) / math.sqrt(c["D"])
        if c["softcap"] > 0:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        if c["causal"]:
            x = x + torch.full((c["T"], total), -math.inf, dtype=torch.float64, device="cuda").triu(n + 1)
        lses.append(torch.logsumexp(x, -1))
        outs.append(torch.einsum("htn,hnd->htd", torch.softmax(x, -1), v))
    out, lse = torch.stack(outs), torch.stack(lses)
    return (out, lse) if c["lse"] else out
