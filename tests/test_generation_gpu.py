"""Rotary, cache append and cache attention together, as the Transfusion attention slot runs them: a prompt with an image
through the block mask into the cache, text tokens one at a time, an image denoised in place; and a training step through
norms and rotation. Against plain 64-bit arithmetic on the module's own 16-bit q, k and v; the tolerance is the parity
contract of the other operators (conftest.assert_parity)."""
import pytest
import torch

import omni_attention_b200 as omni
from conftest import assert_parity
from omni_attention_b200.transfusion import patch_attention, transfusion_block_mask, unpatch_attention
from oracle import cache_oracle as orc
from oracle.omni_oracle import naive_attn_mask
from test_transfusion_gpu import AttentionLike

pytestmark = pytest.mark.gpu


def reference(mod, x, allowed, positions, rot, w=None):
    """The patched module on the whole sequence: x [b, n, dim] fp16, allowed [b, n, n] bool."""
    q, k = mod.to_qk(x)
    v = mod.to_v(x).double().cpu()
    q, k = (orc.rotate(t.cpu(), positions, rot.inv_freq.cpu(), rot.layout, rot.factor, None if w is None else w.cpu()) for t in (q, k))
    s = q @ k.transpose(2, 3) * mod.scale
    s = torch.tanh(s / mod.softcap_value) * mod.softcap_value
    o = (s.masked_fill(~allowed[:, None], -torch.inf).softmax(-1) @ v).to(x)
    if mod.to_gates is not None:
        o = o * mod.to_gates(x).sigmoid()
    return mod.to_out(o)


@pytest.mark.parametrize("dim_head,layout,page", [(64, "interleaved", 16), (128, "half", 64)])
def test_prompt_text_and_image(cuda_device, dim_head, layout, page):
    torch.manual_seed(1)
    b, heads, dim, prompt, image = 2, 4, 128, 150, 40
    mod = patch_attention(AttentionLike(dim, dim_head, heads, learned_mix=False)).to("cuda").half()
    rot = omni.OmniRotary.from_base(dim_head, layout=layout, device="cuda")
    total = prompt + 5 + image
    x = torch.randn(b, total, dim, device="cuda").half()
    spans = torch.tensor([[[1, 20, 64]], [[1, 3, 100]]], dtype=torch.int32)
    # an image's tokens share a position
    positions = torch.arange(total).repeat(b, 1)
    for i, (_, at, n) in enumerate(spans[:, 0].tolist()):
        positions[i, at:at + n] = at
        positions[i, at + n:] -= n - 1
    positions[:, -image:] = positions[:, -image:-image + 1]
    allowed = torch.ones(total, total, dtype=torch.bool).tril().repeat(b, 1, 1)
    allowed[:, :prompt, :prompt] = naive_attn_mask(prompt, spans)
    allowed[:, -image:, -image:] = True
    with torch.no_grad():
        want = reference(mod, x, allowed, positions, rot)
        pages = -(-total // page)
        cache = omni.OmniPagedCache.allocate(b * pages + 1, heads, page, dim_head, b, pages, torch.float16)
        cache.page_table.copy_(torch.randperm(b * pages, device="cuda").view(b, pages))
        at = lambda lo, hi: rot.at(positions[:, lo:hi].cuda())
        mask = transfusion_block_mask(spans.cuda(), heads, prompt)
        got, kept = mod(x[:, :prompt], block_mask=mask, rotary_emb=at(0, prompt), cache=cache, return_kv_cache=True)
        assert kept is cache
        assert_parity(got, None, want[:, :prompt], None, "prompt")
        cache.lengths += prompt
        for i in range(prompt, prompt + 5):
            got = mod(x[:, i:i + 1], rotary_emb=at(i, i + 1), cache=cache, causal=True)
            assert_parity(got, None, want[:, i:i + 1], None, f"token {i}")
            cache.lengths += 1
        for noise in (1.0, 0.0):     # the last pass counts
            y = x[:, -image:] + noise * torch.randn_like(x[:, -image:])
            got = mod(y, rotary_emb=at(total - image, total), cache=cache)
        assert_parity(got, None, want[:, -image:], None, "image")
        # the same through the model's own rotary function
        mod.apply_rotary = lambda emb, t: omni.omni_rotary(t, None, rot, emb)[0]
        again = mod(x[:, -image:], rotary_emb=positions[:, -image:].cuda(), cache=cache)
        assert torch.equal(again, got)
        for bad in (dict(attn_mask=torch.ones(1, 1)), dict(block_mask=mask, causal=True), dict(block_mask="flex")):
            with pytest.raises(ValueError, match="OmniPagedCache"):
                mod(x[:, -image:], cache=cache, **bad)
    with pytest.raises(omni.OmniAttnError, match="no backward"):
        mod(x[:, -image:], cache=cache)
    unpatch_attention(mod)


def prompt_and_cache(module_dtype, cache_dtype, rot, weight=None, n=50, heads=2, dim_head=64):
    """(module, x, mask, empty cache, the prompt's stored keys and values as [b, h, n, d])"""
    torch.manual_seed(4)
    mod = patch_attention(AttentionLike(96, dim_head, heads, learned_mix=False)).to("cuda").to(module_dtype)
    x = torch.randn(2, n, 96, device="cuda").to(module_dtype)
    mask = transfusion_block_mask(torch.tensor([[[1, 10, 20]], [[1, 0, 7]]], dtype=torch.int32).cuda(), heads, n)
    cache = omni.OmniPagedCache.allocate(8, heads, 16, dim_head, 2, 4, cache_dtype)
    cache.page_table.copy_(torch.arange(8, device="cuda").view(2, 4))
    stored = lambda pages: pages.view(2, 4, heads, 16, dim_head).transpose(1, 2).reshape(2, heads, 64, dim_head)[:, :, :n]
    return mod, x, mask, cache, stored


DTYPES = [(m, c) for m in (torch.float16, torch.bfloat16, torch.float32) for c in (torch.float16, torch.bfloat16)]


@pytest.mark.parametrize("module_dtype,cache_dtype", DTYPES)
def test_prompt_and_text_with_a_module_and_a_cache_of_any_dtype(cuda_device, module_dtype, cache_dtype):
    rot = omni.OmniRotary.from_base(64, device="cuda")
    mod, x, mask, cache, stored = prompt_and_cache(module_dtype, cache_dtype, rot)
    with torch.no_grad():
        want = mod(x, block_mask=mask, rotary_emb=rot.at())      # the same without a cache
        got = mod(x, block_mask=mask, rotary_emb=rot.at(), cache=cache)
        assert got.dtype == module_dtype
        if module_dtype != torch.float32:     # (an fp32 module's core is computed in the cache's dtype)
            assert torch.equal(got, want)
        k = omni.omni_rotary(None, mod.to_qk(x)[1], rot)[1]
        assert torch.equal(stored(cache.k_pages), k.to(cache_dtype)) and torch.equal(stored(cache.v_pages), mod.to_v(x).to(cache_dtype))
        cache.lengths += 50
        one = mod(x[:, :1], rotary_emb=rot.at(torch.full((2, 1), 50, device="cuda")), cache=cache, causal=True)
        assert one.dtype == module_dtype and torch.isfinite(one).all()


@pytest.mark.parametrize("module_dtype,cache_dtype", DTYPES)
@pytest.mark.parametrize("given", [True, False])
def test_keys_are_the_same_from_a_prompt_and_from_tokens(cuda_device, module_dtype, cache_dtype, given):
    """The same tokens through the block mask and through generation leave the same bits in the cache (norm, rotation, one
    rounding to the cache's dtype), whether their positions are given or follow from the cache's lengths."""
    rot = omni.OmniRotary.from_base(64, device="cuda")
    w = 1 + 0.2 * torch.randn(64, device="cuda")
    mod, x, mask, cache, stored = prompt_and_cache(module_dtype, cache_dtype, rot)
    positions = torch.arange(50, device="cuda").expand(2, 50).contiguous()
    at = lambda lo, hi: rot.at(positions[:, lo:hi] if given else None, w, w)
    with torch.no_grad():
        mod(x, block_mask=mask, rotary_emb=rot.at(positions, w, w), cache=cache)
        k, v = stored(cache.k_pages).clone(), stored(cache.v_pages).clone()
        cache.k_pages.zero_(), cache.v_pages.zero_()
        for lo, hi in ((0, 20), (20, 50)):
            mod(x[:, lo:hi], rotary_emb=at(lo, hi), cache=cache, causal=True)
            cache.lengths += hi - lo
        # the projections of 20 and 30 tokens may differ from those of 50 in their last bits: compared on the module's own k
        own = torch.cat([mod.to_qk(x[:, lo:hi])[1] for lo, hi in ((0, 20), (20, 50))], 2)
        own_v = torch.cat([mod.to_v(x[:, lo:hi]) for lo, hi in ((0, 20), (20, 50))], 2)
        want = omni.omni_rotary(None, own, rot, positions, None, w)[1].to(cache_dtype)
        assert torch.equal(stored(cache.k_pages), want) and torch.equal(stored(cache.v_pages), own_v.to(cache_dtype))
        if torch.equal(own, mod.to_qk(x)[1]):
            assert torch.equal(k, want)


def test_a_checked_slot(cuda_device):
    """check_status: the same results, and an error for a prompt on a cache that is not empty or a page that is not there."""
    rot = omni.OmniRotary.from_base(64, device="cuda")
    mod, x, mask, cache, stored = prompt_and_cache(torch.float16, torch.float16, rot)
    with torch.no_grad():
        want = mod(x, block_mask=mask, rotary_emb=rot.at(), cache=cache)
        patch_attention(mod, check_status=True)
        assert torch.equal(mod(x, block_mask=mask, rotary_emb=rot.at(), cache=cache), want)
        cache.lengths += 50
        mod(x[:, :1], rotary_emb=rot.at(), cache=cache, causal=True)
        with pytest.raises(omni.OmniAttnError, match="must be empty"):
            mod(x, block_mask=mask, rotary_emb=rot.at(), cache=cache)
        cache.page_table[1, 3] = -1
        with pytest.raises(omni.OmniAttnError, match="page_table"):
            mod(x[:, :1], rotary_emb=rot.at(), cache=cache, causal=True)
        patch_attention(mod)
        mod(x[:, :1], rotary_emb=rot.at(), cache=cache, causal=True)


def test_training_through_norms_and_rotation(cuda_device):
    torch.manual_seed(2)
    b, n, dim, heads, dh = 1, 200, 64, 2, 64
    mod = AttentionLike(dim, dh, heads, gate_values=False, learned_mix=False)
    rot = omni.OmniRotary.from_base(dh)
    w = (1 + 0.2 * torch.randn(dh)).requires_grad_()
    x = torch.randn(b, n, dim)
    spans = torch.tensor([[[1, 50, 60]]], dtype=torch.int32)
    pos = torch.arange(n)[None]
    q, k = mod.to_qk(x)
    inv = rot.inv_freq
    q, k = (orc.rotate(t, pos, inv, weight=w).float() for t in (q, k))
    s = torch.tanh(q @ k.transpose(2, 3) * mod.scale / mod.softcap_value) * mod.softcap_value
    o = s.masked_fill(~naive_attn_mask(n, spans)[:, None].expand_as(s), -torch.inf).softmax(-1) @ mod.to_v(x)
    mod.to_out(o).square().sum().backward()
    want_w, want_qk = w.grad.clone(), mod.qk.weight.grad.clone()

    gpu = AttentionLike(dim, dh, heads, gate_values=False, learned_mix=False)
    gpu.load_state_dict(mod.state_dict())
    gpu = patch_attention(gpu).to("cuda")
    wg = w.detach().cuda().requires_grad_()
    out = gpu(x.cuda(), block_mask=transfusion_block_mask(spans.cuda(), heads, n), rotary_emb=rot.to("cuda").at(pos.cuda(), wg, wg))
    out.square().sum().backward()
    for got, want in ((wg.grad, want_w), (gpu.qk.weight.grad, want_qk)):
        assert float((got.cpu() - want).abs().max()) <= 3e-2 * float(want.abs().max())
