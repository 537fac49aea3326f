"""A cache of keys and values for decoding, in 16 or 8 bits, and attention of a few tokens over it.

Formats of an 8-bit cache, for each row of head_dim values of one token and one head:

  int8: scale = amax / 127 (fp32), code = x / scale to the nearest integer, ties to even;
  fp8 (e4m3): scale = the least power of two with amax / scale <= 448, code = x / scale rounded to e4m3, ties to even.
  The scale is at most 2^119, where codes saturate: 2^120 times the code of 255 would be no fp32 number.

A row that holds an infinity or NaN reads back as NaN. A row of int8 whose scale would be subnormal reads as zeros.

``lengths[b]`` says how many tokens of sequence b stand. New tokens go into the slots behind them (``append``), attention
sees them there (``cache_attention``), and ``advance`` makes them stand. So drafted tokens can be tried and dropped: what
is not advanced over is written over. All of it works on device tensors without a synchronisation, so a decoding step can
be captured into a graph.

On a GPU the kernels are those of ``ops/csrc/kv_cache_kernels.hip`` and ``cache_attention_kernels.hip`` (bf16 or fp16,
head_dim 32, 64, 128 or 256); on a CPU plain torch operations serve unit tests, for any float type and head_dim.
"""

import math
from typing import Optional, Union

import torch

from . import _load_extension

_TILE = 32  # slots are allocated in multiples of the kernels' tile of keys
_KINDS = {None: None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
_HEAD_DIMS = (32, 64, 128, 256)


def _need(ok, message):
    if not ok:
        raise RuntimeError(message)


def _no_grad(who, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{who} has no backward pass: call it under torch.no_grad()")


def _no_tangent(who, *tensors):  # the bindings check this where the kernels run
    _need(
        all(torch.autograd.forward_ad.unpack_dual(t).tangent is None for t in tensors), f"{who} has no forward-mode derivative"
    )


class KVCache:
    """Keys and values of one layer: ``batch_size`` sequences, ``num_kv_heads`` heads, up to ``max_len`` tokens.

    ``quant`` is None (held in ``dtype``), "int8" or "fp8". ``lengths`` is an int32 tensor [B] that the layers of a
    model share; by default the cache makes its own, of zeros. ``k`` and ``v`` are views of what is held
    ([B, H, max_len, D]), ``k_scale`` and ``v_scale`` ([B, H, max_len]) of the scales of an 8-bit cache (of "fp8" powers
    of two: attention goes by their exponents).
    """

    def __init__(
        self,
        batch_size: int,
        num_kv_heads: int,
        max_len: int,
        head_dim: int,
        dtype: torch.dtype = torch.bfloat16,
        quant: Optional[str] = None,
        device=None,
        lengths: Optional[torch.Tensor] = None,
    ):
        if quant not in _KINDS:
            raise ValueError(f"unknown quant {quant!r}: None, 'int8' or 'fp8'")
        if min(batch_size, num_kv_heads, max_len, head_dim) < 0:
            raise ValueError("sizes must not be negative")
        self.device = torch.device("cpu" if device is None else device)
        if self.device.type == "cuda":
            if dtype not in (torch.bfloat16, torch.float16):
                raise ValueError(f"a cache on the GPU is bfloat16 or float16, got {dtype}")
            if head_dim not in _HEAD_DIMS:
                raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
        self.max_len, self.dtype, self.quant = max_len, dtype, quant
        slots = -(-max_len // _TILE) * _TILE
        shape = (batch_size, num_kv_heads, slots)
        held = _KINDS[quant] or dtype
        self._k = torch.zeros(*shape, head_dim, dtype=held, device=self.device)
        self._v = torch.zeros_like(self._k)
        self.device = self._k.device
        self._k_scale = self._v_scale = None
        if quant is not None:
            self._k_scale = torch.zeros(shape, dtype=torch.float32, device=self.device)
            self._v_scale = torch.zeros_like(self._k_scale)
        if lengths is None:
            lengths = torch.zeros(batch_size, dtype=torch.int32, device=self.device)
        elif (
            lengths.dtype != torch.int32
            or lengths.shape != (batch_size,)
            or lengths.device != self.device
            or not lengths.is_contiguous()
        ):
            raise ValueError(f"lengths must be a contiguous int32 tensor [{batch_size}] on {self.device}")
        self.lengths = lengths

    @property
    def k(self):
        return self._k[:, :, : self.max_len]

    @property
    def v(self):
        return self._v[:, :, : self.max_len]

    @property
    def k_scale(self):
        return None if self._k_scale is None else self._k_scale[:, :, : self.max_len]

    @property
    def v_scale(self):
        return None if self._v_scale is None else self._v_scale[:, :, : self.max_len]

    def _held(self):
        return self._k, self._v, self._k_scale, self._v_scale, self.max_len

    def append(self, k: torch.Tensor, v: torch.Tensor, offset: int = 0, counts: Optional[torch.Tensor] = None):
        """Write k and v [B, H, T, D] into the slots lengths[b] + offset + t, quantised as the cache holds them.

        Of sequence b the first ``counts[b]`` tokens are written (int32 [B]; None: all T). A token whose slot the cache
        does not have is not written. Lengths stay as they are: see ``advance``.
        """
        _no_grad("KVCache.append", k, v)
        if self._k.is_cuda:
            _load_extension(required=True).kv_cache_append(*self._held(), k, v, self.lengths, offset, counts)
            return
        _no_tangent("KVCache.append", k, v)
        B, H, _, D = self._k.shape
        _need(
            k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and (k.shape[0], k.shape[1], k.shape[3]) == (B, H, D),
            f"KVCache.append: k and v must be [{B}, {H}, T, {D}] of one type",
        )
        _need(self.quant or k.dtype == self.dtype, f"KVCache.append: the cache holds {self.dtype}, got {k.dtype}")
        _need(offset >= 0, f"KVCache.append: bad offset {offset}")
        _need(
            counts is None or (counts.dtype == torch.int32 and counts.shape == (B,)),
            "KVCache.append: counts must be a contiguous int32 tensor [B]",
        )
        for b in range(B):
            n = k.shape[2] if counts is None else min(max(int(counts[b]), 0), k.shape[2])
            start = int(self.lengths[b]) + offset
            t0, t1 = max(0, -start), min(n, self.max_len - start)
            if t1 <= t0:
                continue
            for x, held, scales in ((k, self._k, self._k_scale), (v, self._v, self._v_scale)):
                code, scale = _quantise(x[b, :, t0:t1], self.quant)
                held[b, :, start + t0 : start + t1] = code
                if scales is not None:
                    scales[b, :, start + t0 : start + t1] = scale

    def read(self, start: Union[int, torch.Tensor] = 0, length: Optional[int] = None, dtype: Optional[torch.dtype] = None):
        """k and v [B, H, length, D] of the slots from ``start`` on (one int, or an int32 tensor [B]) as the values that
        they stand for, in ``dtype`` (bf16, fp16 or fp32; None: the cache's). Without a length, all up to max_len. Slots
        that the cache does not have read as zeros."""
        dtype = dtype or self.dtype
        each = start if isinstance(start, torch.Tensor) else None
        offset = 0 if each is not None else start
        if length is None:
            _need(each is None, "KVCache.read: starts that differ need a length")
            length = max(self.max_len - offset, 0)
        if self._k.is_cuda:
            return _load_extension(required=True).kv_cache_read(*self._held(), each, offset, length, dtype)
        _need(length >= 0 and offset >= 0, f"KVCache.read: bad length {length} or offset {offset}")
        B, H, _, D = self._k.shape
        _need(
            each is None or (each.dtype == torch.int32 and each.shape == (B,)),
            "KVCache.read: start must be a contiguous int32 tensor [B]",
        )
        first = torch.full((B,), offset) if each is None else each.long()
        at = first[:, None] + torch.arange(length)
        has = (at >= 0) & (at < self.max_len)
        at = at.clamp(0, max(self.max_len - 1, 0))
        rows = torch.arange(B)[:, None]
        out = []
        for held, scales in ((self._k, self._k_scale), (self._v, self._v_scale)):
            if self.max_len == 0:
                out.append(torch.zeros(B, H, length, D, dtype=dtype))
                continue
            x = held[rows, :, at].transpose(1, 2)  # [B, H, length, D]
            if scales is not None:
                x = x.float() * scales[rows, :, at].transpose(1, 2)[..., None]
            out.append(torch.where(has[:, None, :, None], x, torch.zeros((), dtype=x.dtype)).to(dtype).contiguous())
        return tuple(out)

    def keep(self, path: torch.Tensor):
        """Move the accepted nodes of a drafted tree together: the row of slot lengths[b] + path[b, i] to lengths[b] + i.

        ``path`` is int64 [B, T], ascending, and ends at the first -1 (``verify_draft``'s). Lengths stay as they are.
        """
        if self._k.is_cuda:
            _load_extension(required=True).kv_cache_keep(*self._held(), self.lengths, path)
            return
        _need(
            path.dtype == torch.int64 and path.dim() == 2 and path.shape[0] == self._k.shape[0],
            "KVCache.keep: path must be an int64 tensor [B, T]",
        )
        for b in range(path.shape[0]):
            start, last = int(self.lengths[b]), -1
            for i, node in enumerate(path[b].tolist()):
                if start < 0 or node <= last or node >= path.shape[1] or start + node >= self.max_len:
                    break
                last = node
                for t in (self._k, self._v, self._k_scale, self._v_scale):
                    if t is not None:
                        t[b, :, start + i] = t[b, :, start + node]

    def advance(self, n: Union[int, torch.Tensor]):
        """Let n more tokens stand (one int, or an integer tensor [B]), in place. Layers that share their lengths
        advance once."""
        self.lengths.add_(n)

    def reset(self):
        """Forget all tokens."""
        self.lengths.zero_()

    def attend(self, q: torch.Tensor, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None):
        """``cache_attention`` over this cache."""
        return cache_attention(q, self, mask=mask, scale=scale)


def _quantise(x, quant):
    if quant is None:
        return x.clone(), None  # the cache's own rows may overlap those that are written
    wide = x.float()
    amax = wide.abs().amax(-1) if x.shape[-1] else wide.new_zeros(wide.shape[:-1])
    bad = ~torch.isfinite(wide).all(-1)
    amax = torch.where(bad, 0.0, amax)
    if quant == "int8":
        scale = amax / 127.0
        scale = torch.where(scale < torch.finfo(torch.float32).tiny, 0.0, scale)
    else:
        mantissa, exponent = torch.frexp(amax / 448.0)
        exponent = (exponent - (mantissa == 0.5).int()).clamp(-126, 119)  # so that codes stand for finite values
        scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), exponent), 0.0)
    held = (~bad & (scale > 0))[..., None]
    quotient = torch.where(held, wide, 0.0).double() / torch.where(held[..., 0], scale, 1.0)[..., None].double()
    if quant == "int8":
        code = torch.round(quotient).to(torch.int8)
    else:
        code = quotient.float().clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return code, torch.where(bad, float("nan"), scale)


def cache_attention(
    q: torch.Tensor, cache: KVCache, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None
) -> torch.Tensor:
    """Attention of the new tokens q [B, Hq, T, D] over a cache of Hkv heads (Hkv divides Hq).

    Every query sees the lengths[b] tokens that stand and, of the slots behind them, slot lengths[b] + j where
    ``mask[..., i, j]`` is true: a bool mask [T, W] or [B, T, W] over the W first new slots (a tree of drafted tokens:
    ``draft_tree_mask``). Without a mask query i sees the new slots 0..i. A query that sees nothing gets zeros. The
    values of slots that a query does not see, NaN among them, do not reach it. ``scale`` defaults to 1 / sqrt(D).
    q is of the cache's type; an 8-bit cache takes bf16 and fp16. The result [B, Hq, T, D] is laid out [B, T, Hq, D] in
    memory. There is no backward pass and no forward-mode derivative.
    """
    _no_grad("cache_attention", q)
    if scale is None:
        scale = 1.0 / math.sqrt(max(q.shape[-1], 1))
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if cache._k.is_cuda:
        return _load_extension(required=True).kv_cache_attend(q, *cache._held(), cache.lengths, mask, scale)

    _no_tangent("cache_attention", q)
    B, H, _, D = cache._k.shape
    _need(q.dim() == 4 and q.shape[0] == B and q.shape[3] == D, f"cache_attention: q must be [{B}, Hq, T, {D}]")
    Hq, T = q.shape[1:3]
    _need(Hq % H == 0 if H else Hq == 0, f"cache_attention: {Hq} query heads are no multiple of the cache's {H}")
    _need(cache.quant or q.dtype == cache.dtype, f"cache_attention: the cache holds {cache.dtype}, q is {q.dtype}")
    if mask is None:
        _need(T <= cache.max_len, f"cache_attention: {T} new tokens, the cache has {cache.max_len} slots")
        mask = torch.ones(T, T, dtype=torch.bool).tril()
    _need(
        mask.dtype == torch.bool and mask.dim() in (2, 3) and mask.shape[-2] == T and (mask.dim() == 2 or mask.shape[0] in (1, B)),
        "cache_attention: mask must be a bool tensor [T, W] or [B, T, W]",
    )
    W = mask.shape[-1]
    _need(W <= cache.max_len, f"cache_attention: the mask covers {W} slots, the cache has {cache.max_len}")
    k, v = cache.read(dtype=torch.promote_types(q.dtype, torch.float32))
    at = torch.arange(cache.max_len) - cache.lengths.long().clamp(0, cache.max_len)[:, None]  # [B, L]
    inside = (at >= 0) & (at < W)
    new = torch.gather(mask.expand(B, T, W), 2, at.clamp(0, max(W - 1, 0))[:, None].expand(B, T, -1)) if W else inside[:, None]
    seen = ((at < 0)[:, None] | (inside[:, None] & new)).unsqueeze(1)  # [B, 1, T, L]
    rep = Hq // H if H else 1
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    scores = (q.to(k.dtype) @ k.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(scores, -1)
    p = torch.where(seen, p, 0.0)
    finite = torch.isfinite(v)
    out = p @ torch.where(finite, v, 0.0)
    if not finite.all():  # of the slots that a query sees, however little they weigh
        odd = torch.where(finite, 0.0, v)[:, :, None]
        out = out + torch.where(seen[..., None], odd, 0.0).sum(-2)
    return torch.where(seen.any(-1, keepdim=True), out, 0.0).to(q.dtype)


def draft_tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """The mask of a tree of drafted tokens: parents int64 [T] or [B, T], with -1 for a root (or an unused node) and
    otherwise a node before the own one, to bool [T, T] or [B, T, T]: whether node j is i or one that i follows."""
    T = parents.shape[-1]
    nodes = torch.arange(T, device=parents.device)
    reach = (parents[..., :, None] == nodes) | (nodes[:, None] == nodes)
    for _ in range(max(T - 1, 0).bit_length()):  # each squaring doubles how far it reaches
        reach = (reach.float() @ reach.float()) > 0
    return reach
