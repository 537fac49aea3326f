"""Fused rotary embedding wrappers (CDNA4 kernels; backward = rotation by −θ)."""

import math
from typing import Optional

import torch

from . import _load_extension


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin):
        ext = _load_extension(required=True)
        ctx.save_for_backward(cos, sin)
        return ext.rope_bf16(x.contiguous(), cos, sin, False)

    @staticmethod
    def backward(ctx, dy):
        ext = _load_extension(required=True)
        cos, sin = ctx.saved_tensors
        return ext.rope_bf16(dy.contiguous(), cos, sin, True), None, None


def fused_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x: [B, H, S, D] bf16; cos/sin: [>=S, D/2] fp32 (position-offset applied
    by the caller via slicing)."""
    return _RopeFn.apply(x, cos.contiguous(), sin.contiguous())


def rope_is_fusable(x, cos) -> bool:
    return (
        x.is_cuda
        and x.dtype == torch.bfloat16
        and x.shape[-1] % 16 == 0
        and cos.dtype == torch.float32
        and cos.is_cuda
    )


# ---------------------------------------------------------------------------
# Rotary positions of q and k together: positions per token, part of the head,
# half or interleaved pairs, tables scaled for long contexts.
# ---------------------------------------------------------------------------

_SCALING_KEYS = {
    "rope_type", "type", "factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor",
    "beta_fast", "beta_slow", "attention_factor",
}


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None):
    """(angle per position of each pair [rotary_dim / 2], factor of cos and sin), in 64 bits.

    ``scaling`` stretches a trained length to a longer one:

    - ``{"rope_type": "linear", "factor"}``: all positions are divided by the factor.
    - ``{"rope_type": "llama3", "factor", "low_freq_factor", "high_freq_factor",
      "original_max_position_embeddings"}``: pairs that turn less than ``low_freq_factor`` times over the
      original length are slowed by the factor, those that turn more than ``high_freq_factor`` times are kept,
      the ones between are mixed.
    - ``{"rope_type": "yarn", "factor", "original_max_position_embeddings"}``, with ``beta_fast`` (32) and
      ``beta_slow`` (1) turns as the ends of a ramp over the pairs, and ``attention_factor``
      (0.1 ln(factor) + 1) on cos and sin.

    Other keys are refused: they would change the tables.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not theta > 1:
        raise ValueError(f"theta must be above 1, got {theta}")
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = float(theta) ** (-2.0 * pair / rotary_dim)
    if scaling is None:
        return freq, 1.0
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind in (None, "default"):
        return freq, 1.0
    if kind not in ("linear", "llama3", "yarn"):
        raise ValueError(f"unknown rope_type {kind!r}: linear, llama3 or yarn")
    unknown = set(scaling) - _SCALING_KEYS
    if unknown:
        raise ValueError(f"unknown keys of the rotary scaling: {sorted(unknown)}")
    factor = float(scaling["factor"])
    if factor < 1:
        raise ValueError(f"the scaling factor must be at least 1, got {factor}")
    if kind == "linear":
        return freq / factor, 1.0
    trained = float(scaling["original_max_position_embeddings"])
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        turns = trained * freq / (2 * math.pi)
        kept = ((turns - low) / (high - low)).clamp(0, 1)
        return freq * (kept + (1 - kept) / factor), 1.0

    def pair_of(turns):  # the pair, as a real number, that turns so often over the trained length
        return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))

    first = max(math.floor(pair_of(float(scaling.get("beta_fast", 32)))), 0)
    last = min(math.ceil(pair_of(float(scaling.get("beta_slow", 1)))), rotary_dim - 1)
    slowed = ((pair - first) / max(last - first, 0.001)).clamp(0, 1)
    attention_factor = scaling.get("attention_factor")
    if attention_factor is None:
        attention_factor = 0.1 * math.log(factor) + 1.0
    return freq * (1 - slowed) + freq / factor * slowed, float(attention_factor)


def rope_tables(max_len: int, rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None, device=None):
    """cos and sin [max_len, rotary_dim / 2] in fp32. The angles are products in 64 bits: in 32, position
    131071 would be off by a hundredth of a radian."""
    freq, factor = rope_frequencies(rotary_dim, theta, scaling)
    angle = torch.arange(max_len, dtype=torch.float64, device=device)[:, None] * freq.to(device)[None]
    return (angle.cos() * factor).float(), (angle.sin() * factor).float()


def _rotary_reference(q, k, cos, sin, positions, interleaved):
    def need(ok, message):
        if not ok:
            raise RuntimeError(f"rotary_embedding: {message}")

    need(q.dim() == 4 and q.is_floating_point(), "q must be a [B, H, S, D] tensor of floats")
    B, _, S, D = q.shape
    need(
        k is None or (k.dim() == 4 and k.dtype == q.dtype and (k.shape[0], *k.shape[2:]) == (B, S, D)),
        "k must be [B, Hk, S, D] of q's type",
    )
    need(
        cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32,
        "cos and sin must be float32 tables [positions, rotary_dim / 2]",
    )
    half = cos.shape[1]
    need(2 * half <= D, f"the tables rotate {2 * half} elements, head_dim is {D}")
    if positions is None:
        need(S <= cos.shape[0], f"{S} positions, the tables have {cos.shape[0]}")
        c, s = cos[None, None, :S], sin[None, None, :S]
    else:
        need(positions.dtype in (torch.int64, torch.int32), "positions must be int64 or int32")
        need(
            1 <= positions.dim() <= 2
            and positions.shape[-1] == S
            and (positions.dim() == 1 or positions.shape[0] in (1, B)),
            "positions must be [S] or [B, S]",
        )
        at = positions.long().expand(B, S)
        known = ((at >= 0) & (at < cos.shape[0]))[:, None, :, None]
        if cos.shape[0] == 0:  # no position is known
            cos = sin = cos.new_zeros(1, half)
        at = at.clamp(0, cos.shape[0] - 1)
        c = torch.where(known, cos[at][:, None], float("nan"))
        s = torch.where(known, sin[at][:, None], float("nan"))

    def rotate(x):
        wide = x.to(torch.promote_types(x.dtype, torch.float32))
        a, b = wide[..., : 2 * half].unflatten(-1, (half, 2) if interleaved else (2, half)).unbind(-1 if interleaved else -2)
        y = torch.stack((a * c - b * s, b * c + a * s), -1 if interleaved else -2).flatten(-2)
        return torch.cat((y, wide[..., 2 * half :]), -1).to(x.dtype)

    return rotate(q), None if k is None else rotate(k)


def rotary_embedding(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
):
    """Rotate q [B, Hq, S, D] and k [B, Hk, S, D] (or None) by their positions, in one launch; returns both
    (q alone where k is None).

    ``cos`` and ``sin`` are fp32 tables [P, R / 2] (``rope_tables``). The first R <= D elements of a head are
    rotated, the rest is copied; pair i is the elements (i, i + R / 2), or (2 i, 2 i + 1) where ``interleaved``.
    ``positions`` is int64 or int32, [S] or [B, S]; None means 0..S-1. A token whose position the tables do not
    have gets NaN in its rotated elements. bf16, fp16 and fp32, any strides (transposed views are read in
    place). The gradient of q and k is the rotation back; the tables have none. Forward-mode derivatives are refused
    on the GPU.
    """
    if q.is_cuda:
        out = _load_extension(required=True).rotary(q, k, cos, sin, positions, interleaved)
    else:
        out = _rotary_reference(q, k, cos, sin, positions, interleaved)
    return out[0] if k is None else out
