"""The paged key/value cache of generation: ``OmniPagedCache``, ``omni_cache_append`` and ``omni_cache_attention``.

The reference model decodes with a dense cache that it concatenates to at every step (transfusion_pytorch/
transfusion.py:933-939) and attends to it with a dense score matrix (:963-983). Here keys and values live in pages, the
new tokens' keys and values are written to their slots (normed and turned by their positions on the way), and the
attention reads the pages where they lie.

One step of generation, layer by layer:

    q = omni_cache_append(cache[layer], k, v, q=q, rotary=rotary, positions=positions)
    out = omni_cache_attention(q, cache[layer])
    ...
    lengths += T          # once, after the last layer; all layers share page_table and lengths

Both calls read ``lengths`` (the tokens that were there before the step) on the device and wait for nothing, so a step can
be captured into a CUDA graph and replayed as the cache grows. A step may be repeated before the lengths move on (an image
that is denoised): the same slots are written again.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from .ops import STATUS_BAD_INDEX, STATUS_WAIT_TIMEOUT, OmniAttnError, load_extension
from .rotary import OmniRotary, rotary_fields


class OmniPagedCache:
    """Keys and values of B sequences for one layer.

    k_pages, v_pages [num_pages, Hkv, page_size, D] fp16 or bf16, contiguous; page_size a power of two from 16 to 1024.
    page_table int32 [B, max_pages]: token i of sequence b is row i % page_size of page page_table[b, i // page_size]; an
    id outside [0, num_pages) is a page that is not there. lengths int32 [B]: tokens in the cache before the current step.
    The tensors are the caller's and may be shared between layers (page_table, lengths) and sequences (pages of a common
    prefix, which must not be appended to)."""

    __slots__ = ("k_pages", "v_pages", "page_table", "lengths")

    def __init__(self, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor):
        if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
            raise OmniAttnError("k_pages and v_pages must be [num_pages, heads, page_size, D] of one shape and dtype")
        if k_pages.dtype not in (torch.float16, torch.bfloat16):
            raise OmniAttnError(f"unsupported cache dtype {k_pages.dtype}: fp16 or bf16")
        if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
            raise OmniAttnError("k_pages and v_pages must be contiguous")
        size = k_pages.shape[2]
        if size < 16 or size > 1024 or size & (size - 1):
            raise OmniAttnError(f"page_size must be a power of two from 16 to 1024, got {size}")
        if k_pages.shape[3] not in (32, 64, 128):
            raise ValueError(f"Unsupported head_dim={k_pages.shape[3]}. Supported: 32, 64, 128.")
        if page_table.dim() != 2 or page_table.dtype != torch.int32:
            raise OmniAttnError("page_table must be int32 [B, max_pages]")
        if lengths.dim() != 1 or lengths.dtype != torch.int32 or lengths.shape[0] != page_table.shape[0]:
            raise OmniAttnError("lengths must be int32 [B]")
        self.k_pages, self.v_pages, self.page_table, self.lengths = k_pages, v_pages, page_table, lengths

    @classmethod
    def allocate(cls, num_pages: int, heads: int, page_size: int, head_dim: int, batch: int, max_pages: int,
                 dtype=torch.bfloat16, device="cuda") -> "OmniPagedCache":
        """An empty cache: no page assigned (-1 everywhere in the table), no tokens."""
        pages = [torch.zeros(num_pages, heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2)]
        return cls(*pages, torch.full((batch, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(batch, dtype=torch.int32, device=device))

    @property
    def page_size(self) -> int:
        return self.k_pages.shape[2]

    def layer_like(self, k_pages: Tensor, v_pages: Tensor) -> "OmniPagedCache":
        """The cache of another layer of the same model: its own pages, this one's table and lengths."""
        return OmniPagedCache(k_pages, v_pages, self.page_table, self.lengths)


def _status(check: bool, device) -> Optional[Tensor]:
    return torch.zeros(1, dtype=torch.int32, device=device) if check else None


def _raise_for(status: Optional[Tensor]) -> None:
    code = 0 if status is None else int(status.item())
    if code & 0xFF == STATUS_WAIT_TIMEOUT:
        raise OmniAttnError(f"kernel gave up waiting (status {code:#x}); output is not valid")
    if code & 0xFF == STATUS_BAD_INDEX:
        raise OmniAttnError("page_table: a token's page is not there (id outside [0, num_pages), beyond the table's end, or "
                            "not the shared one); the token was left out")


def omni_cache_append(cache: OmniPagedCache, k: Tensor, v: Tensor, q: Optional[Tensor] = None,
                      rotary: Optional[OmniRotary] = None, positions: Optional[Tensor] = None,
                      counts: Optional[Tensor] = None, q_weight: Optional[Tensor] = None,
                      k_weight: Optional[Tensor] = None, eps: float = 1e-6, check_status: bool = False) -> Optional[Tensor]:
    """Stores T new tokens of each sequence behind its ``cache.lengths`` tokens, and returns their queries.

    k, v [B, Hkv, T, D], q [B, H, T, D] or None. k and q are normed (where a weight is given) and turned as in
    ``omni_rotary``; ``positions`` int32 / int64 [T], [1, T] or [B, T], None = the tokens' numbers in their sequences.
    ``counts`` int32 [B]: how many of the T tokens a sequence really has (None = all); those behind are not stored and
    their queries come back as zeros. Tokens whose page is not there, or that the page table has no room for, are not
    stored; ``check_status=True`` waits for the GPU and raises then. Returns q' [B, H, T, D], None without q. Reads
    ``cache.lengths`` and leaves it as it is. No gradients: call it under ``torch.no_grad()``."""
    inv_freq, half, factor = rotary_fields(rotary)
    status = _status(check_status, k.device)
    out = load_extension().cache_append(cache.k_pages, cache.v_pages, cache.page_table, cache.lengths, k, v, q, inv_freq, half,
                                        factor, positions, counts, q_weight, k_weight, eps, status)
    _raise_for(status)
    return out


def omni_cache_attention(q: Tensor, cache: OmniPagedCache, counts: Optional[Tensor] = None, causal: bool = True,
                         limits: Optional[Tensor] = None, scale: Optional[float] = None, softcap: Optional[float] = None,
                         return_lse: bool = False, shared_prefix: int = 0,
                         check_status: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Attention of the T new tokens of each sequence, which are in the cache already, over the cache.

    q [B, H, T, D]; H a multiple of the cache's heads (query head h reads key/value head h // (H / Hkv)). Row t of sequence
    b attends its first ``cache.lengths[b] + t + 1`` tokens, with ``causal=False`` all ``cache.lengths[b] + counts[b]`` of
    them, with ``limits`` (int32 [B, T]) its first ``limits[b, t]``. Rows behind a sequence's count (``counts`` int32 [B],
    None = T) and rows with no key are zero (LSE -inf). ``scale`` (positive) defaults to D ** -0.5, ``softcap`` > 0 caps the scaled
    scores with tanh (from 1e-6 to 1e30 times the scale; None, 0 or less: no cap). ``shared_prefix``: that many first tokens of all sequences are in the same pages (a prompt with
    several continuations): they are read once for the whole batch. Keys in pages that are not there are left out;
    ``check_status=True`` waits for the GPU and raises then, also when ``shared_prefix`` tokens are not in the same pages.
    Up to 16 query rows to a key/value head (H / Hkv * T, with ``shared_prefix`` times B) the result is off by its own rounding only,
    with more the weights are rounded to 16 bits, as in ``omni_attention``.
    Returns out [B, H, T, D] (and lse [B, H, T], natural log, with ``return_lse``). No gradients."""
    if scale is not None and not scale >= torch.finfo(torch.float32).tiny:
        raise OmniAttnError(f"scale must be finite and positive (not zero, negative or NaN), got {scale}")
    status = _status(check_status, q.device)
    res = load_extension().cache_attention(q, cache.k_pages, cache.v_pages, cache.page_table, cache.lengths, counts, causal,
                                           limits, scale or 0.0, softcap or 0.0, return_lse, shared_prefix, status)
    _raise_for(status)
    return res
