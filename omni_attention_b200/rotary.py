"""Rotary positions and norms of the heads: ``omni_rotary(q, k, rotary, positions, q_weight, k_weight)``.

The reference's model turns queries and keys with an imported rotary embedding between its projections and the attention
core (transfusion_pytorch/transfusion.py:941-942: interleaved pairs, positions that stand still inside an image); models
with normed heads take the RMS norm of every head row first. Here both are one pass over q and k on the GPU, with its
backward, in fp16, bf16 or fp32.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from .ops import OmniAttnError, load_extension

LAYOUTS = ("interleaved", "half")


class OmniRotary:
    """The rotation a model uses: frequencies, which elements form a pair, a factor.

    ``inv_freq`` float64 [rotary_dim / 2]: radians per position (64 bits, because the angle of a far position is a large
    number of which only the rest of the last turn counts). ``layout``: the members of pair p are the elements 2p and
    2p + 1 ("interleaved") or p and p + rotary_dim / 2 ("half"); elements from rotary_dim on pass through. ``factor``
    multiplies cosine and sine. Build it once and keep it; ``from_base`` computes the frequencies."""

    __slots__ = ("inv_freq", "layout", "factor")

    def __init__(self, inv_freq: Tensor, layout: str = "interleaved", factor: float = 1.0):
        if layout not in LAYOUTS:
            raise OmniAttnError(f"rotary layout must be one of {LAYOUTS}, got {layout!r}")
        if inv_freq.dim() != 1 or inv_freq.dtype != torch.float64:
            raise OmniAttnError(f"inv_freq must be float64 [rotary_dim / 2], got {inv_freq.dtype} {tuple(inv_freq.shape)}")
        if not math.isfinite(factor):
            raise OmniAttnError("the rotary factor must be finite")
        self.inv_freq, self.layout, self.factor = inv_freq.contiguous(), layout, float(factor)

    @property
    def rotary_dim(self) -> int:
        return 2 * self.inv_freq.shape[0]

    @classmethod
    def from_base(cls, rotary_dim: int, base: float = 10000.0, layout: str = "interleaved", scaling: Optional[dict] = None,
                  device=None) -> "OmniRotary":
        """inv_freq[p] = base ** (-2 p / rotary_dim), scaled for contexts longer than the trained ones by ``scaling``:

        {"type": "linear", "factor": s}                    positions divided by s
        {"type": "ntk", "factor": s}                       base * s ** (rotary_dim / (rotary_dim - 2))
        {"type": "yarn", "factor": s, "original_length": n, "beta_fast": 32, "beta_slow": 1}
            pairs that turn more than beta_fast times in n positions stay, those below beta_slow are divided by s, those
            between are mixed linearly in the pair number (from the last whole number that is still "more" to the first that is
            "below", which may lie behind the last pair, at most at rotary_dim - 1); cosine and sine are multiplied by
            0.1 ln(s) + 1 (or by "attention_factor")."""
        if rotary_dim < 2 or rotary_dim % 2:
            raise OmniAttnError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
        if not (math.isfinite(base) and base > 1.0):
            raise OmniAttnError(f"the rotary base must be finite and above 1, got {base}")
        pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
        inv = base ** (-2.0 * pair / rotary_dim)
        factor = 1.0
        if scaling is not None:
            known = {"linear": {"factor"}, "ntk": {"factor"},
                     "yarn": {"factor", "original_length", "beta_fast", "beta_slow", "attention_factor"}}
            kind = scaling.get("type")
            if kind not in known:
                raise OmniAttnError(f"rotary scaling type must be one of {sorted(known)}, got {kind!r}")
            odd = set(scaling) - known[kind] - {"type"}
            if odd:
                raise OmniAttnError(f"rotary scaling {kind!r} does not know {sorted(odd)}")
            s = float(scaling.get("factor", 0.0))
            if not (math.isfinite(s) and s >= 1.0):
                raise OmniAttnError(f"rotary scaling factor must be finite and at least 1, got {scaling.get('factor')}")
            if kind == "linear":
                inv = inv / s
            elif kind == "ntk":
                if rotary_dim == 2:
                    raise OmniAttnError("rotary scaling 'ntk' needs a rotary_dim above 2")
                inv = (base * s ** (rotary_dim / (rotary_dim - 2))) ** (-2.0 * pair / rotary_dim)
            else:
                n = float(scaling.get("original_length", 0))
                fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
                if not (n > 0 and fast > slow > 0):
                    raise OmniAttnError("rotary scaling 'yarn' needs original_length > 0 and beta_fast > beta_slow > 0")
                at = lambda turns: rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))
                lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
                keep = 1.0 - ((pair - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
                inv = inv / s * (1 - keep) + inv * keep
                factor = float(scaling.get("attention_factor", 0.1 * math.log(s) + 1.0))
        return cls(inv.to(device), layout, factor)

    def to(self, device) -> "OmniRotary":
        return OmniRotary(self.inv_freq.to(device), self.layout, self.factor)

    def at(self, positions: Optional[Tensor] = None, q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None,
           eps: float = 1e-6) -> "RotaryAt":
        """This rotation at the positions of a batch, with the norms before it if there are any: what a patched attention
        module takes as ``rotary_emb`` (``transfusion.patch_attention``)."""
        return RotaryAt(self, positions, q_weight, k_weight, eps)


class RotaryAt(NamedTuple):
    rotary: OmniRotary
    positions: Optional[Tensor] = None
    q_weight: Optional[Tensor] = None
    k_weight: Optional[Tensor] = None
    eps: float = 1e-6


def rotary_fields(rotary: Optional[OmniRotary]):
    """(inv_freq, half layout, factor) for the extension module."""
    if rotary is None:
        return None, False, 1.0
    if not isinstance(rotary, OmniRotary):
        raise OmniAttnError(f"rotary must be an OmniRotary, got {type(rotary).__name__}")
    return rotary.inv_freq, rotary.layout == "half", rotary.factor


def omni_rotary(q: Optional[Tensor], k: Optional[Tensor], rotary: Optional[OmniRotary] = None,
                positions: Optional[Tensor] = None, q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None,
                eps: float = 1e-6) -> Tuple[Optional[Tensor], Optional[Tensor]]:
    """Queries and keys, normed per head (where a weight is given) and turned by their positions; differentiable with
    respect to q, k and the weights (not to ``inv_freq``, not twice, not in forward mode: refused).

    q [B, H, N, D], k [B, Hkv, N, D]: CUDA tensors of one dtype (fp16, bf16, fp32), D 32, 64 or 128, any strides (rows that
    are contiguous along D and start on 16-byte boundaries are read where they lie; others are read element by element,
    or copied when D itself is strided). Either may be None. ``positions`` int32 or int64 [N], [1, N] or [B, N], None =
    0..N-1. ``q_weight``, ``k_weight``: [D] or [heads, D], fp32 or the data's dtype, both of one form;
    y = x / sqrt(mean(x ** 2) + eps) * weight. ``rotary`` None: norm only. Returns contiguous (q', k')."""
    inv_freq, half, factor = rotary_fields(rotary)
    if rotary is None and q_weight is None and k_weight is None:
        raise OmniAttnError("omni_rotary: neither a rotation nor a norm weight given")
    return load_extension().rotary(q, k, inv_freq, half, factor, positions, q_weight, k_weight, eps)
