"""64-bit CPU restatement of the rotary, cache-append and cache-attention operators (test infrastructure only), one row
at a time where that keeps it plain."""
import math

import torch


def rotate(x, positions, inv_freq, layout="interleaved", factor=1.0, weight=None, eps=1e-6):
    """x [B, H, N, D] any dtype -> float64: norm (with a weight [D] or [H, D]) and rotation. positions [B, N]."""
    x = x.double()
    if weight is not None:
        w = weight.double()
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (w if w.dim() == 1 else w[None, :, None, :])
    if inv_freq is None:
        return x
    rd2 = inv_freq.shape[0]
    a = positions.double()[:, None, :, None] * inv_freq.double()
    c, s = a.cos() * factor, a.sin() * factor
    y = x.clone()
    for p in range(rd2):
        i, j = (2 * p, 2 * p + 1) if layout == "interleaved" else (p, p + rd2)
        u, v = x[..., i], x[..., j]
        y[..., i], y[..., j] = u * c[..., p] - v * s[..., p], u * s[..., p] + v * c[..., p]
    return y


def slots(page_table, lengths, counts, T, page_size, num_pages):
    """[(b, t, page, row)] of the new tokens that have a slot."""
    out = []
    for b in range(page_table.shape[0]):
        n = max(int(lengths[b]), 0)
        for t in range(T if counts is None else max(0, min(int(counts[b]), T))):
            e = (n + t) // page_size
            page = int(page_table[b, e]) if e < page_table.shape[1] else -1
            if 0 <= page < num_pages:
                out.append((b, t, page, (n + t) % page_size))
    return out


def attention(q, k_pages, v_pages, page_table, lengths, counts=None, causal=True, limits=None, scale=None, softcap=0.0):
    """(out [B, H, T, D], lse [B, H, T], the same mean of |v| as out is of v) in float64."""
    B, H, T, D = q.shape
    P, Hkv, page, _ = k_pages.shape
    G, cap = H // Hkv, page_table.shape[1] * page
    out = torch.zeros(B, H, T, D, dtype=torch.float64)
    size = torch.zeros(B, H, T, D, dtype=torch.float64)
    lse = torch.full((B, H, T), -math.inf, dtype=torch.float64)
    scale = D ** -0.5 if scale is None else scale
    for b in range(B):
        n = max(int(lengths[b]), 0)
        c = T if counts is None else max(0, min(int(counts[b]), T))
        total = min(n + c, cap)
        ids = [int(page_table[b, i // page]) * page + i % page if 0 <= int(page_table[b, i // page]) < P else -1 for i in range(total)]
        ids = torch.tensor(ids, dtype=torch.long)
        for t in range(c):
            lim = total if not causal else min(n + t + 1, total)
            if limits is not None:
                lim = min(int(limits[b, t]), total)
            if lim <= 0:
                continue
            seen = ids[:lim]
            seen = seen[seen >= 0]
            if len(seen) == 0:
                continue
            for h in range(H):
                k = k_pages[:, h // G].reshape(-1, D)[seen].double()
                v = v_pages[:, h // G].reshape(-1, D)[seen].double()
                x = k @ q[b, h, t].double() * scale
                if softcap > 0:
                    x = softcap * torch.tanh(x / softcap)
                lse[b, h, t] = torch.logsumexp(x, 0)
                w = torch.softmax(x, 0)
                out[b, h, t], size[b, h, t] = w @ v, w @ v.abs()
    return out, lse, size
