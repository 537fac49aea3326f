"""Rotary positions, the key/value cache, attention over it and draft verification, each against its formula in 64 bits.

Tolerances count roundings: half a step of a type is finfo.eps / 2 relative to the value.
"""

import itertools
import math

import pytest
import torch

from accelerate_amd.ops import KVCache, cache_attention, rope_tables, rotary_embedding, verify_draft
from accelerate_amd.ops.kv_cache import _quantise, draft_tree_mask
from accelerate_amd.ops.rope import rope_frequencies

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def randn(*shape, seed=0, dtype=FP32, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(device)


# ---- rotary positions -----------------------------------------------------------------------------------------------


def rotate64(x, cos, sin, positions, interleaved, inverse=False):
    """The formula, in 64 bits on the host: (result, sum of the products' sizes)."""
    x, cos, sin = x.detach().double().cpu(), cos.double().cpu(), sin.double().cpu()
    B, _, S, _ = x.shape
    half = cos.shape[1]
    positions = torch.arange(S).expand(B, S) if positions is None else positions.long().cpu().expand(B, S)
    known = (positions >= 0) & (positions < cos.shape[0])
    at = positions.clamp(0, cos.shape[0] - 1)
    c, s = cos[at][:, None], sin[at][:, None] * (-1 if inverse else 1)
    y, size = x.clone(), x.abs()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    y[..., : 2 * half][~known[:, None].expand(y.shape[:3])] = math.nan
    return y, size


def check_rotated(y, x, cos, sin, positions, interleaved, inverse=False):
    want, size = rotate64(x, cos, sin, positions, interleaved, inverse)
    y = y.detach().cpu()
    assert y.dtype == x.dtype and y.shape == x.shape
    # two products and a sum in 32 bits, then one rounding to the type
    tolerance = 3 * half_step(FP32) * size * 1.01 + half_step(y.dtype) * want.abs() * 1.01 + torch.finfo(y.dtype).tiny
    assert torch.equal(torch.isnan(want), torch.isnan(y))
    bad = (y.double() - want).abs() > tolerance
    assert not bad.any(), (y.double() - want).abs().max()


ROPE_SHAPES = [  # B, Hq, Hk, S, D, R
    (1, 32, 8, 1, 128, 128),
    (2, 4, 2, 37, 64, 64),
    (3, 2, 2, 5, 96, 48),
    (2, 3, 1, 130, 80, 40),
    (1, 5, 5, 9, 20, 6),
    (1, 1, 1, 3, 7, 4),
    (2, 2, 1, 4, 64, 0),
    (1, 40, 8, 700, 128, 64),
    (2, 8, 8, 33, 256, 256),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", ROPE_SHAPES)
def test_rotary_matches_formula(device, dtype, interleaved, shape):
    B, Hq, Hk, S, D, R = shape
    if R:
        cos, sin = rope_tables(1000, R, device=device)
    else:
        cos, sin = torch.empty(1000, 0, device=device), torch.empty(1000, 0, device=device)
    q = randn(B, S, Hq * D, seed=1, dtype=dtype, device=device).view(B, S, Hq, D).transpose(1, 2)
    k = randn(B, Hk, S, D, seed=2, dtype=dtype, device=device)
    yq, yk = rotary_embedding(q, k, cos, sin, interleaved=interleaved)
    check_rotated(yq, q, cos, sin, None, interleaved)
    check_rotated(yk, k, cos, sin, None, interleaved)
    positions = torch.randint(0, 1000, (B, S), generator=torch.Generator().manual_seed(3)).to(device)
    for p in (positions, positions.int(), positions[:1], positions[0], positions[:, :1].expand(B, S)):
        yq = rotary_embedding(q, None, cos, sin, positions=p, interleaved=interleaved)
        check_rotated(yq, q, cos, sin, p, interleaved)


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_positions_outside_the_tables_are_nan(device):
    cos, sin = rope_tables(16, 8, device=device)
    x = randn(1, 2, 4, 12, device=device)
    p = torch.tensor([0, -1, 16, 15], device=device)
    y = rotary_embedding(x, None, cos, sin, positions=p)
    check_rotated(y, x, cos, sin, p, False)
    assert torch.isnan(y[0, :, 1:3, :8]).all() and torch.isfinite(y[..., 8:]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_reads_odd_views(device, interleaved):
    """Slices of a fused projection, a shifted start, a step over tokens and over elements."""
    B, S, D = 2, 6, 32
    cos, sin = rope_tables(S, D, device=device)
    fused = randn(B, 2 * S, 6 * D + 3, seed=4, dtype=BF16, device=device)
    views = [
        fused[:, :S, 1 : 1 + 4 * D].unflatten(-1, (4, D)).transpose(1, 2),
        fused[:, ::2, : 4 * D].unflatten(-1, (4, D)).transpose(1, 2),
        fused[:, :S, : 4 * D].unflatten(-1, (2, 2 * D))[..., ::2].transpose(1, 2),
        fused[:, :S, :D][:, None].expand(B, 3, S, D),
    ]
    for x in views:
        yq, yk = rotary_embedding(x, views[0], cos, sin, interleaved=interleaved)
        check_rotated(yq, x, cos, sin, None, interleaved)
        check_rotated(yk, views[0], cos, sin, None, interleaved)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rotary_gradient_matches_formula(device, interleaved, dtype):
    B, Hq, Hk, S, D, R = 2, 4, 2, 9, 48, 32
    cos, sin = rope_tables(64, R, device=device)
    p = torch.randint(0, 64, (B, S), generator=torch.Generator().manual_seed(5)).to(device)
    q = randn(B, S, Hq, D, seed=6, dtype=dtype, device=device).transpose(1, 2).requires_grad_()
    k = randn(B, Hk, S, D, seed=7, dtype=dtype, device=device).requires_grad_()
    yq, yk = rotary_embedding(q, k, cos, sin, positions=p, interleaved=interleaved)
    dq, dk = randn(*q.shape, seed=8, dtype=dtype, device=device), randn(*k.shape, seed=9, dtype=dtype, device=device)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk), retain_graph=True)
    check_rotated(gq, dq, cos, sin, p, interleaved, inverse=True)
    check_rotated(gk, dk, cos, sin, p, interleaved, inverse=True)
    # one of the two alone, and a gradient without memory of its own
    (gk,) = torch.autograd.grad(yk, k, dk, retain_graph=True)
    check_rotated(gk, dk, cos, sin, p, interleaved, inverse=True)
    (gq,) = torch.autograd.grad(yq.sum(), q, retain_graph=True)
    check_rotated(gq, torch.ones_like(q), cos, sin, p, interleaved, inverse=True)


def test_rotary_gradient_matches_differences():
    cos, sin = rope_tables(8, 6)
    q, k = randn(1, 2, 4, 8).double().requires_grad_(), randn(1, 1, 4, 8, seed=1).double().requires_grad_()
    for interleaved in (False, True):
        f = lambda q, k: rotary_embedding(q, k, cos, sin, positions=torch.tensor([3, 0, 7, 7]), interleaved=interleaved)
        assert torch.autograd.gradcheck(f, (q, k))
        assert torch.autograd.gradgradcheck(f, (q, k))


@gpu
def test_rotary_gradient_matches_differences_on_gpu():
    """The rotation is linear: a central difference with a step of 1/2 has no error but its roundings."""
    cos, sin = rope_tables(8, 6, device="cuda")
    x = randn(1, 2, 4, 8, device="cuda").requires_grad_()
    weight = randn(1, 2, 4, 8, seed=1, device="cuda")
    (grad,) = torch.autograd.grad((rotary_embedding(x, None, cos, sin) * weight).sum(), x)
    for i in (0, 13, 40, 63):
        step = torch.zeros(64, device="cuda")
        step[i] = 0.5
        step = step.view_as(x)
        with torch.no_grad():
            up, down = ((rotary_embedding(x + s * step, None, cos, sin) * weight).double().sum() for s in (1, -1))
        # 64 products of sizes below 10, each with a few roundings of 2^-24
        assert abs((up - down).item() - grad.flatten()[i].item()) < 64 * 10 * 8 * 2**-24


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_refuses(device):
    cos, sin = rope_tables(8, 16, device=device)
    q, k = randn(2, 4, 6, 16, device=device), randn(2, 2, 6, 16, device=device)
    bad = [
        (q[0], None, cos, sin, {}),
        (q, k[:1], cos, sin, {}),
        (q, k[:, :, :5], cos, sin, {}),
        (q, k.to(BF16), cos, sin, {}),
        (q, k, cos, sin[:4], {}),
        (q, k, cos.to(BF16), sin.to(BF16), {}),
        (q[..., :8], None, cos, sin, {}),
        (randn(1, 1, 9, 16, device=device), None, cos, sin, {}),
        (q, k, cos, sin, {"positions": torch.zeros(2, 5, dtype=torch.long, device=device)}),
        (q, k, cos, sin, {"positions": torch.zeros(3, 6, dtype=torch.long, device=device)}),
        (q, k, cos, sin, {"positions": torch.zeros(2, 6, device=device)}),
    ]
    for q_, k_, c, s, kw in bad:
        with pytest.raises(RuntimeError):
            rotary_embedding(q_, k_, c, s, **kw)
    if device == "cuda":
        with pytest.raises(RuntimeError):
            rotary_embedding(q, k, cos.cpu(), sin.cpu())
        with pytest.raises(RuntimeError):
            rotary_embedding(q.double(), None, cos, sin)


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_empty(device):
    cos, sin = rope_tables(8, 16, device=device)
    for shape in ((0, 4, 6, 16), (2, 0, 6, 16), (2, 4, 0, 16)):
        assert rotary_embedding(torch.empty(shape, device=device), None, cos, sin).shape == shape


def test_rope_tables_scalings():
    theta, R, trained, s = 500000.0, 64, 8192, 8.0
    plain = [theta ** (-2 * i / R) for i in range(R // 2)]
    freq, factor = rope_frequencies(R, theta, {"rope_type": "linear", "factor": s})
    assert factor == 1 and all(math.isclose(f, p / s, rel_tol=1e-14) for f, p in zip(freq.tolist(), plain))

    scaling = {"rope_type": "llama3", "factor": s, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": trained}
    freq, factor = rope_frequencies(R, theta, scaling)
    for f, p in zip(freq.tolist(), plain):
        wave = 2 * math.pi / p
        if wave < trained / 4:
            want = p
        elif wave > trained:
            want = p / s
        else:
            smooth = (trained / wave - 1) / 3
            want = (1 - smooth) * p / s + smooth * p
        assert math.isclose(f, want, rel_tol=1e-12)

    freq, factor = rope_frequencies(R, theta, {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": trained})
    assert math.isclose(factor, 0.1 * math.log(s) + 1)
    turns = [trained * p / (2 * math.pi) for p in plain]
    assert all(math.isclose(f, p, rel_tol=1e-14) for f, p, t in zip(freq.tolist(), plain, turns) if t > 40)
    assert all(math.isclose(f, p / s, rel_tol=1e-14) for f, p, t in zip(freq.tolist(), plain, turns) if t < 0.6)
    assert all(p / s * 0.999 <= f <= p * 1.001 for f, p in zip(freq.tolist(), plain))

    cos, sin = rope_tables(131072, R, theta, scaling)
    assert cos.dtype == FP32 and cos.shape == (131072, R // 2)
    angle = 131071 * rope_frequencies(R, theta, scaling)[0]
    assert (cos[-1].double() - angle.cos()).abs().max() <= half_step(FP32)
    for bad in ({"rope_type": "other", "factor": 2.0}, {"rope_type": "linear", "factor": 0.5}):
        with pytest.raises(ValueError):
            rope_frequencies(R, theta, bad)
    with pytest.raises(ValueError):
        rope_frequencies(7)


# ---- the cache ------------------------------------------------------------------------------------------------------


def e4m3_values():
    """All finite values of e4m3, by the format's definition."""
    values = set()
    for sign, exponent, mantissa in itertools.product((1, -1), range(16), range(8)):
        if (exponent, mantissa) != (15, 7):
            values.add(sign * (mantissa / 8 * 2.0**-6 if exponent == 0 else (1 + mantissa / 8) * 2.0 ** (exponent - 7)))
    return sorted(values)


def quantised64(x, quant):
    """Values that the rows of x [..., D] are held as, and their scales, in 64 bits on the host."""
    x = x.double().cpu()
    amax = x.abs().amax(-1, keepdim=True)
    if quant == "int8":
        scale = (amax / 127).float().double()  # held in 32 bits
        return torch.where(scale > 0, torch.round(x / torch.where(scale > 0, scale, 1.0)) * scale, 0.0), scale[..., 0]
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448)))
    scale = torch.where(amax > 0, scale, 0.0)
    grid = torch.tensor(e4m3_values(), dtype=torch.float64)
    y = (x / torch.where(scale > 0, scale, 1.0)).contiguous()
    hi = torch.searchsorted(grid, y).clamp(1, len(grid) - 1)
    lo = hi - 1
    up, down = grid[hi] - y, y - grid[lo]
    # a tie goes to the even mantissa: every other value, counted from zero, which is in the middle
    even = (hi - (len(grid) - 1) // 2) % 2 == 0
    return torch.where((up < down) | ((up == down) & even), grid[hi], grid[lo]) * scale, scale[..., 0]


def tie_rows(D, dtype):
    """Rows whose quotients lie on and next to the borders between codes."""
    rows = []
    for top in (127.0, 448.0, 1.0, 3.0, 0.0117):
        x = torch.linspace(-1, 1, D).double() * top
        x[0] = top
        rows.append(x)
        x = ((torch.arange(D) % 253) - 126 + 0.5).double() * (top / 127)
        x[0] = top
        rows.append(x)
    rows.append(torch.zeros(D).double())
    rows.append(torch.linspace(-3, 3, D).double() * 2.0**-14)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("quant", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_quantise_reference_matches_definition(quant, dtype):
    for x in (tie_rows(128, dtype), randn(200, 64, dtype=dtype, seed=11) * 3):
        code, scale = _quantise(x, quant)
        want, want_scale = quantised64(x, quant)
        assert torch.equal(scale.double(), want_scale)
        assert torch.equal(code.double() * scale.double()[:, None], want)


@gpu
@pytest.mark.parametrize("quant", ["int8", "fp8", None])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_append_and_read_match_definition(quant, dtype, D):
    B, H, T, max_len = 3, 2, 41, 100
    x = randn(B, T, H, D, seed=12, dtype=dtype) * torch.exp(randn(B, T, H, 1, seed=13) * 3).to(dtype)
    rows = tie_rows(D, dtype)
    x[1, : len(rows), 0] = rows
    k, v = x.transpose(1, 2), randn(B, H, T, D, seed=14, dtype=dtype)
    cache = KVCache(B, H, max_len, D, dtype=dtype, quant=quant, device="cuda")
    cache.lengths.copy_(torch.tensor([0, 17, 80]))  # the last sequence runs out of slots
    cache.append(k.cuda().transpose(1, 2).contiguous().transpose(1, 2), v.cuda())
    for name, x in (("k", k), ("v", v)):
        held = getattr(cache, name).cpu()
        for b, n in enumerate(cache.lengths.tolist()):
            upto = min(T, max_len - n)
            code, scale = _quantise(x[b, :, :upto], quant)
            got = held[b, :, n : n + upto]
            assert torch.equal(got.float(), code.float())
            assert not held[b, :, :n].float().any() and not held[b, :, n + T :].float().any()
            if quant:
                got_scale = getattr(cache, name + "_scale").cpu()
                assert torch.equal(got_scale[b, :, n : n + upto], scale)
                want, _ = quantised64(x[b, :, :upto], quant)
                assert torch.equal(got.double() * got_scale[b, :, n : n + upto].double()[..., None], want)
    # read back: rounded once to 32 bits, then to the type
    reference = KVCache(B, H, max_len, D, dtype=dtype, quant=quant)
    for name in ("k", "v", "k_scale", "v_scale"):
        if getattr(reference, name) is not None:
            getattr(reference, name).copy_(getattr(cache, name).cpu())
    reference.lengths.copy_(cache.lengths.cpu())
    for kwargs in ({}, {"start": 3, "length": 60}, {"start": cache.lengths, "length": T}, {"dtype": FP32}, {"start": 99}, {"length": 0}):
        got = cache.read(**kwargs)
        host = {n: a.cpu() if isinstance(a, torch.Tensor) else a for n, a in kwargs.items()}
        for g, w in zip(got, reference.read(**host)):
            assert g.dtype == w.dtype and torch.equal(g.cpu(), w)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quant", ["int8", "fp8", None])
def test_append_counts_offset_and_bounds(device, quant):
    B, H, T, D, max_len = 4, 2, 5, 32, 40
    cache = KVCache(B, H, max_len, D, dtype=BF16, quant=quant, device=device)
    cache.lengths.copy_(torch.tensor([0, 10, 38, -3]))
    k = torch.ones(B, H, T, D, dtype=BF16, device=device)
    cache.append(k, -k, offset=1, counts=torch.tensor([5, 2, 5, 4], dtype=torch.int32, device=device))
    got = cache.read(dtype=FP32)[0].cpu()[:, :, :, 0]
    want = torch.zeros(B, H, max_len)
    want[0, :, 1:6] = 1
    want[1, :, 11:13] = 1
    want[2, :, 39:] = 1
    want[3, :, 0:2] = 1  # slots -2..1
    # int8: 127 times the scale of 1 / 127 in 32 bits, and a product
    assert (got - want).abs().max() <= 2 * half_step(FP32)
    assert torch.equal(cache.lengths.cpu(), torch.tensor([0, 10, 38, -3], dtype=torch.int32))
    cache.append(k[:, :, :0], k[:, :, :0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quant", ["int8", "fp8"])
def test_rows_without_codes(device, quant):
    """Infinities and NaN make their row NaN and no other; tiny and zero rows read as what they are held as."""
    cache = KVCache(1, 1, 8, 32, dtype=BF16, quant=quant, device=device)
    x = torch.ones(1, 1, 6, 32, dtype=BF16, device=device)
    x[0, 0, 1, 5] = math.inf
    x[0, 0, 2, 31] = math.nan
    x[0, 0, 3] = 0
    x[0, 0, 4] = 2.0**-126
    x[0, 0, 5, 0] = torch.finfo(BF16).max
    cache.append(x, x)
    y = cache.read(dtype=FP32)[0][0, 0].cpu()
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    assert torch.isfinite(y[[0, 3, 4, 5, 6, 7]]).all() and not y[3].any()
    # an int8 scale would be subnormal; e4m3 holds 2^-126 as 1 times the least scale
    assert torch.equal(y[4], torch.full((32,), 0.0 if quant == "int8" else 2.0**-126))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quant", ["int8", "fp8", None])
def test_keep_moves_the_path(device, quant):
    B, H, T, D = 3, 2, 6, 64
    cache = KVCache(B, H, 20, D, dtype=BF16, quant=quant, device=device)
    cache.lengths.copy_(torch.tensor([0, 4, 13]))
    cache.append(randn(B, H, T, D, seed=20, dtype=BF16, device=device), randn(B, H, T, D, seed=21, dtype=BF16, device=device))
    before = [x.clone() for x in cache.read(start=cache.lengths, length=T)]
    everything = [x.clone() for x in cache.read()]
    path = torch.tensor([[0, 2, 5, -1, -1, -1], [0, -1, -1, -1, -1, -1], [0, 1, 3, 4, 5, -1]], device=device)
    cache.keep(path)
    for now, was, all_was, all_now in zip(cache.read(start=cache.lengths, length=T), before, everything, cache.read()):
        for b, nodes in enumerate(path.tolist()):
            nodes = [n for n in nodes if n >= 0]
            assert torch.equal(now[b, :, : len(nodes)], was[b, :, nodes])
            n0 = int(cache.lengths[b])
            assert torch.equal(all_now[b, :, :n0], all_was[b, :, :n0])
            assert torch.equal(all_now[b, :, n0 + len(nodes) :], all_was[b, :, n0 + len(nodes) :])
    # what is no ascending path of the cache's slots ends it
    cache.keep(torch.tensor([[0, 9, 1, 1, 1, 1], [3, 2, -1, -1, -1, -1], [1, 1, 7, -1, -1, -1]], device=device))


@pytest.mark.parametrize("device", DEVICES)
def test_cache_refuses(device):
    with pytest.raises(ValueError):
        KVCache(1, 1, 8, 32, quant="int4", device=device)
    with pytest.raises(ValueError):
        KVCache(1, 1, -8, 32, device=device)
    with pytest.raises(ValueError):
        KVCache(2, 1, 8, 32, device=device, lengths=torch.zeros(3, dtype=torch.int32, device=device))
    if device == "cuda":
        for kwargs in ({"head_dim": 48}, {"dtype": FP32}):
            with pytest.raises(ValueError):
                KVCache(**{"batch_size": 1, "num_kv_heads": 1, "max_len": 8, "head_dim": 32, "device": device, **kwargs})
    cache = KVCache(2, 2, 8, 32, dtype=BF16, device=device)
    k = torch.zeros(2, 2, 3, 32, dtype=BF16, device=device)
    counts = torch.zeros(2, dtype=torch.int32, device=device)
    for args, kwargs in [
        ((k, k[:, :, :2]), {}),
        ((k[:1], k[:1]), {}),
        ((k[..., :16], k[..., :16]), {}),
        ((k.to(FP16), k.to(FP16)), {}),
        ((k, k), {"offset": -1}),
        ((k, k), {"counts": counts.long()}),
        ((k, k), {"counts": counts[:1]}),
        ((k.clone().requires_grad_(), k), {}),
    ]:
        with pytest.raises(RuntimeError):
            cache.append(*args, **kwargs)
    for kwargs in ({"length": -1}, {"start": -1, "length": 2}, {"start": counts}, {"start": counts.long(), "length": 2}):
        with pytest.raises(RuntimeError):
            cache.read(**kwargs)
    with pytest.raises(RuntimeError):
        cache.keep(torch.zeros(2, 3, dtype=torch.int32, device=device))
    q = torch.zeros(2, 4, 3, 32, dtype=BF16, device=device)
    mask = torch.ones(2, 3, 3, dtype=torch.bool, device=device)
    for q_, kwargs in [
        (q[:1], {}),
        (q[:, :3], {}),
        (q[..., :16], {}),
        (q.to(FP16), {}),
        (q.clone().requires_grad_(), {}),
        (q, {"mask": mask[:, :2]}),
        (q, {"mask": mask.float()}),
        (q, {"mask": torch.ones(3, 3, 3, dtype=torch.bool, device=device)}),
        (q, {"mask": torch.ones(3, 9, dtype=torch.bool, device=device)}),
        (torch.zeros(2, 4, 9, 32, dtype=BF16, device=device), {}),
    ]:
        with pytest.raises(RuntimeError):
            cache_attention(q_, cache, **kwargs)
    with pytest.raises(ValueError):
        cache_attention(q, cache, scale=math.inf)
    if device == "cuda":
        with pytest.raises(RuntimeError):
            cache_attention(q.cpu(), cache)
        with pytest.raises(RuntimeError):
            cache.append(k.cpu(), k.cpu())


# ---- attention over the cache ---------------------------------------------------------------------------------------


def attend64(q, cache, mask, scale):
    """(result, tolerance) by the definition in 64 bits on the host, sequence by sequence."""
    q = q.cpu()
    B, Hq, T, D = q.shape
    H = cache.k.shape[1]
    out, tol = torch.zeros(B, Hq, T, D, dtype=torch.float64), torch.zeros(B, Hq, T, D, dtype=torch.float64)
    step, step32 = half_step(q.dtype), half_step(FP32)
    for b, n in enumerate(cache.lengths.tolist()):
        n = min(max(n, 0), cache.max_len)
        W = T if mask is None else mask.shape[-1]
        end = min(n + W, cache.max_len)
        seen = torch.ones(T, end, dtype=torch.bool)
        new = torch.ones(T, T, dtype=torch.bool).tril() if mask is None else (mask if mask.dim() == 2 else mask.expand(B, T, W)[b]).cpu()
        seen[:, n:] = new[:, : end - n]
        k, v = cache.k[b, :, :end].cpu().double(), cache.v[b, :, :end].cpu().double()
        if cache.quant:
            k = k * cache.k_scale[b, :, :end].cpu().double()[..., None]
            v = v * cache.v_scale[b, :, :end].cpu().double()[..., None]
        k, v = k.repeat_interleave(Hq // H, 0), v.repeat_interleave(Hq // H, 0)
        x = q[b].double()
        s = torch.where(seen, x @ k.transpose(-1, -2) * scale, -math.inf)
        top = s.amax(-1, keepdim=True).clamp(min=-1e300) if end else s.new_zeros(Hq, T, 1)
        p = torch.where(seen, torch.exp(s - top), 0.0)
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        v0 = torch.nan_to_num(v, 0, 0, 0)
        o = p @ v0
        odd = ~torch.isfinite(v)
        if odd.any():
            o = o + torch.where(seen[None, :, :, None], torch.where(odd, v, 0.0)[:, None], 0.0).sum(-2)
        size = p @ v0.abs()
        # of a score in 32 bits: D products and sums, the scales, the shift; of its exponential a few more
        error = torch.where(seen, x.abs() @ torch.nan_to_num(k, 0, 0, 0).abs().transpose(-1, -2) * abs(scale), 0.0)
        ds = (D + 8) * step32 * 2 * (error.amax(-1, keepdim=True) if end else 0.0) + 16 * step32
        # each probability is given as two operands, the second of which is rounded (half a step of half a step), the
        # result is rounded once; sums of `end` terms are in 32 bits
        tol[b] = (step**2 * (1 + 2**-6) + 2 * ds + 2 * (end + 64) * step32) * size + step * 1.01 * torch.nan_to_num(o, 0, 0, 0).abs()
        # an exponential below 2^-126 of the largest, which is 1, may be lost in 32 bits: at most that times its value
        tol[b] += (end * 2.0**-126 * v0.abs().amax() if end else 0.0) * (total > 0)
        if q.dtype == FP16:  # probabilities below its normal range: half of its least step, relative to the largest scale
            unit = v0.abs().amax(-1).amax(-1)[:, None, None] if end else torch.zeros(Hq, 1, 1)
            tol[b] += (torch.where(total > 0, end * 2.0**-25 / total, 0.0) * unit * 2) + 2.0**-24
        out[b] = o
    return out, tol


def check_attention(out, q, cache, mask, scale=None):
    want, tol = attend64(q, cache, mask, q.shape[-1] ** -0.5 if scale is None else scale)
    assert out.shape == q.shape and out.dtype == q.dtype
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = (got == want) | torch.isnan(want)
    error = torch.where(same, 0.0, (got - want).abs())
    assert (error <= tol).all(), (error / tol.clamp(min=1e-30)).max()


def filled_cache(B, H, max_len, D, lengths, T, dtype, quant, device, seed=30):
    cache = KVCache(B, H, max_len, D, dtype=dtype, quant=quant, device=device)
    k, v = randn(B, H, max_len, D, seed=seed, dtype=dtype, device=device), randn(B, H, max_len, D, seed=seed + 1, dtype=dtype, device=device)
    v = v * torch.exp(randn(1, 1, max_len, 1, seed=seed + 2, device=device)).to(dtype)
    cache.append(k, v)  # every slot holds something
    cache.lengths.copy_(torch.tensor(lengths))
    return cache


CACHE_SHAPES = [  # B, H, rep, T, max_len, lengths
    (1, 1, 1, 1, 1, [0]),
    (2, 2, 4, 1, 300, [299, 0]),
    (3, 1, 8, 5, 700, [1, 31, 640]),
    (2, 4, 1, 17, 130, [32, 113]),
    (2, 2, 3, 9, 64, [60, 70]),  # the last sequences run out of slots
    (1, 1, 7, 16, 4096, [3333]),
    (2, 1, 16, 33, 200, [127, 128]),
]


@gpu
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", CACHE_SHAPES)
def test_cache_attention_matches_definition(quant, dtype, D, shape):
    B, H, rep, T, max_len, lengths = shape
    cache = filled_cache(B, H, max_len, D, lengths, T, dtype, quant, "cuda")
    q = randn(B, T, H * rep * D, seed=40, dtype=dtype, device="cuda").view(B, T, H * rep, D).transpose(1, 2)
    check_attention(cache_attention(q, cache), q, cache, None)
    g = torch.Generator().manual_seed(41)
    W = min(max_len, T + 3)
    mask = (torch.rand(B, T, W, generator=g) < 0.4).cuda()
    mask[0, 0] = False  # a row that sees nothing new, and nothing at all where its sequence is empty
    check_attention(cache_attention(q, cache, mask=mask, scale=0.3), q, cache, mask, 0.3)
    check_attention(cache.attend(q, mask=mask[0]), q, cache, mask[0])


@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
@pytest.mark.parametrize("shape", CACHE_SHAPES)
def test_cache_attention_on_the_host(quant, shape):
    B, H, rep, T, max_len, lengths = shape
    cache = filled_cache(B, H, max_len, 16, lengths, T, FP32, quant, "cpu")
    q = randn(B, H * rep, T, 16, seed=40)
    check_attention(cache_attention(q, cache), q, cache, None)
    mask = torch.rand(B, T, min(max_len, T + 3), generator=torch.Generator().manual_seed(41)) < 0.4
    mask[0, 0] = False
    check_attention(cache_attention(q, cache, mask=mask), q, cache, mask)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
def test_cache_attention_keeps_unseen_values_out(device, quant):
    """NaN and infinities behind the new tokens reach no query, those of new tokens the queries that see them."""
    B, H, T, D, max_len = 3, 1, 6, 64, 256
    dtype = BF16
    cache = filled_cache(B, H, max_len, D, [30, 0, 159], T, dtype, quant, device)
    parents = torch.tensor([-1, 0, 0, 1, 2, 2], device=device)
    mask = draft_tree_mask(parents)
    q = randn(B, 4, T, D, seed=42, dtype=dtype, device=device)
    k, v = randn(B, H, 20, D, seed=43, dtype=dtype, device=device), randn(B, H, 20, D, seed=44, dtype=dtype, device=device)
    k[:, :, T:], v[:, :, T:] = math.nan, math.inf
    cache.append(k, v)
    out = cache_attention(q, cache, mask=mask)
    check_attention(out, q, cache, mask)
    assert torch.isfinite(out).all()
    v[:, :, 3, 5] = math.nan
    v[:, :, 4, 7] = math.inf
    v[:, :, 5, 7] = -math.inf
    cache.append(k, v)
    out = cache_attention(q, cache, mask=mask)
    check_attention(out, q, cache, mask)
    assert torch.isfinite(out[:, :, [0, 1, 2]]).all()
    assert torch.isnan(out[:, :, 3, 5]).all()
    if quant is None:
        assert (out[:, :, 4, 7] == math.inf).all() and (out[:, :, 5, 7] == -math.inf).all()
    k[:, :, 1] = math.nan  # a key makes the scores of those that see it NaN
    cache.append(k, v)
    out = cache_attention(q, cache, mask=mask)
    assert torch.isnan(out[:, :, [1, 3]]).all() and torch.isfinite(out[:, :, [0, 2]]).all()
    if quant is None:  # in the tokens that stand, all see it
        cache.v[:, :, 29, 3] = math.inf
        cache.append(k[:, :, T:] * 0, v[:, :, T:] * 0)
        assert (cache_attention(q[:1, :, :1], _first(cache))[..., 3] == math.inf).all()


def _first(cache):
    """The first sequence of a cache, alone."""
    one = KVCache(1, cache.k.shape[1], cache.max_len, cache.k.shape[3], dtype=cache.dtype, quant=cache.quant, device=cache.device)
    one.k.copy_(cache.k[:1])
    one.v.copy_(cache.v[:1])
    one.lengths.copy_(cache.lengths[:1])
    one.append(torch.zeros_like(one.k[:, :, :1]), torch.zeros_like(one.k[:, :, :1]))
    return one


@gpu
@pytest.mark.parametrize("quant", [None, "int8"])
def test_cache_attention_large_scores(quant):
    """A large score late in the cache takes over from all before it; scores of 200 do not overflow."""
    D, n = 128, 2000
    cache = filled_cache(1, 1, 2100, D, [n], 1, BF16, quant, "cuda")
    q = randn(1, 4, 1, D, seed=50, dtype=BF16, device="cuda")
    k = cache.read()[0].clone()
    k[0, 0, 1777] = q[0, 0, 0] * 16
    k[0, 0, 40] = q[0, 1, 0] * 14
    v = cache.read()[1].clone()
    cache.lengths.zero_()
    cache.append(k, v)
    cache.lengths.fill_(n)
    check_attention(cache_attention(q, cache), q, cache, None)


@gpu
def test_cache_attention_small_value_scales_in_fp16():
    """Values of 10^-4 with int8 scales near 10^-6, below fp16's normal range."""
    cache = KVCache(1, 1, 500, 64, dtype=FP16, quant="int8", device="cuda")
    k, v = randn(1, 1, 450, 64, seed=51, dtype=FP16), randn(1, 1, 450, 64, seed=52, dtype=FP16) * 1e-4
    v[:, :, 200:] *= 30  # the unit grows along the way
    cache.append(k.cuda(), v.cuda())
    cache.lengths.fill_(449)
    q = randn(1, 2, 1, 64, seed=53, dtype=FP16, device="cuda")
    want, _ = attend64(q, cache, None, 64**-0.5)
    got = cache_attention(q, cache).cpu().double()
    # sums of 450 roundings of 2^-11 without a common sign, and the result's own at its subnormal step of 2^-24
    assert ((got - want).abs() <= 2 * half_step(FP16) * want.abs().amax() + 2.0**-25 * 1.01).all()


@gpu
@pytest.mark.parametrize("quant", ["int8", None])
def test_offsets_beyond_32_bits(quant):
    """A cache whose last head starts behind 2^31 elements, and whose sequence ends there."""
    B, H, D, max_len = 2, 2, 256, 2_900_000
    cache = KVCache(B, H, max_len, D, dtype=BF16, quant=quant, device="cuda")
    assert cache._k.stride(0) + cache._k.stride(1) > 2**31
    n = max_len - 40
    cache.lengths.copy_(torch.tensor([3, n]))
    k, v = randn(B, H, 8, D, seed=60, dtype=BF16, device="cuda"), randn(B, H, 8, D, seed=61, dtype=BF16, device="cuda")
    cache.append(k, v)
    small = KVCache(B, H, 8, D, dtype=BF16, quant=quant)
    small.append(k.cpu(), v.cpu())
    got, want = cache.read(start=cache.lengths, length=8), small.read()
    for g, w in zip(got, want):
        assert torch.equal(g.cpu(), w)
    cache.keep(torch.tensor([[0, 2, 3, -1], [0, 1, 3, -1]], device="cuda"))
    got = cache.read(start=cache.lengths, length=3)
    for g, w in zip(got, want):
        assert torch.equal(g[0].cpu(), w[0][:, [0, 2, 3]]) and torch.equal(g[1].cpu(), w[1][:, [0, 1, 3]])
    # the keys before are zeros: with scores near 256 * 30 / 16 the new ones have all the weight
    q = (k[:, :, :1] * 30).contiguous()
    out = cache_attention(q, cache)
    # |k|^2 is about 256 +- 5 * 23; all other scores lie below that of the query's own key by more than 100
    assert (out.cpu().double() - want[1][:, :, :1].double()).abs().max() <= 2 * half_step(BF16) * want[1].abs().max()


@gpu
def test_cache_attention_many_rows_and_splits():
    """Row blocks that share keys, and a cache that is split among many workgroups."""
    for B, H, rep, T, max_len, lengths in [(1, 1, 8, 100, 3000, [2500]), (1, 3, 4, 60, 900, [801]), (1, 1, 1, 1, 40000, [39000])]:
        cache = filled_cache(B, H, max_len, 128, lengths, T, BF16, "fp8", "cuda")
        q = randn(B, H * rep, T, 128, seed=70, dtype=BF16, device="cuda")
        check_attention(cache_attention(q, cache), q, cache, None)


@gpu
def test_cache_attention_odd_views():
    """Queries and masks whose strides and addresses do not suit wide loads."""
    cache = filled_cache(2, 2, 100, 64, [50, 20], 3, BF16, None, "cuda")
    wide = randn(2, 3, 4 * 64 + 5, seed=71, dtype=BF16, device="cuda")
    q = wide[:, :, 1:257].unflatten(-1, (4, 64)).transpose(1, 2)
    mask = (torch.rand(2, 3, 9, generator=torch.Generator().manual_seed(72)) < 0.6).cuda()
    check_attention(cache_attention(q, cache, mask=mask[..., 1:8]), q, cache, mask[..., 1:8])
    check_attention(cache_attention(q, cache, mask=mask[..., ::3]), q, cache, mask[..., ::3])
    check_attention(cache_attention(q, cache, mask=mask[:1, :, :5]), q, cache, mask[:1, :, :5])
    check_attention(cache_attention(q, cache, mask=mask[..., :0]), q, cache, mask[..., :0])


@pytest.mark.parametrize("device", DEVICES)
def test_cache_empty_sizes(device):
    for B, H, max_len in ((0, 2, 8), (2, 0, 8), (2, 2, 0)):
        cache = KVCache(B, H, max_len, 32, dtype=BF16, device=device)
        x = torch.zeros(B, H, 0, 32, dtype=BF16, device=device)
        cache.append(x, x)
        assert cache.read()[0].shape == (B, H, max_len, 32)
        assert cache_attention(torch.zeros(B, 2 * H, 0, 32, dtype=BF16, device=device), cache).shape == (B, 2 * H, 0, 32)
    cache = KVCache(2, 1, 8, 32, dtype=BF16, device=device)
    mask = torch.zeros(1, 0, dtype=torch.bool, device=device)
    assert not cache_attention(torch.ones(2, 3, 1, 32, dtype=BF16, device=device), cache, mask=mask).any()


def test_draft_tree_mask():
    parents = torch.tensor([[-1, 0, 0, 1, 3, 2], [-1, 0, 1, 2, 3, 4]])
    mask = draft_tree_mask(parents)
    assert mask[0].nonzero().tolist() == [
        [0, 0], [1, 0], [1, 1], [2, 0], [2, 2], [3, 0], [3, 1], [3, 3], [4, 0], [4, 1], [4, 3], [4, 4], [5, 0], [5, 2], [5, 5],
    ]
    assert torch.equal(mask[1], torch.ones(6, 6, dtype=torch.bool).tril())
    assert torch.equal(draft_tree_mask(parents[0]), mask[0])
    assert draft_tree_mask(parents[:, :1]).all()


# ---- verification ---------------------------------------------------------------------------------------------------


def verify64(target, tokens, u, draft, parents):
    """The walk in words: take children in order; where none is taken, draw from what is left."""
    B, T, V = target.shape
    target, u = target.double().cpu(), u.double().cpu()
    result = []
    for b in range(B):
        parent = list(range(-1, T - 1)) if parents is None else (parents if parents.dim() == 1 else parents[b]).tolist()
        at, said, path = 0, [], [0]
        while True:
            w = target[b, at].clone().nan_to_num(0).clamp(min=0)
            left, moved, gone = 1.0, False, set()
            for i in range(at + 1, T):
                x = int(tokens[b, i])
                if parent[i] != at:
                    continue
                if not 0 <= x < V:
                    if parents is None:
                        break
                    continue
                p = float(target[b, at, x])
                if draft is not None:
                    q = draft[b, i - 1].double().cpu()
                    if float(u[b, i]) * float(q[x]) < p:
                        moved = True
                    else:
                        w = (target[b, at] - q).nan_to_num(0).clamp(min=0)
                        break
                elif x in gone:
                    continue
                elif float(u[b, i]) * left < p:
                    moved = True
                if moved:
                    at = i
                    said.append(x)
                    path.append(i)
                    break
                left -= p
                gone.add(x)
            if moved:
                continue
            w[list(gone)] = 0
            break
        if not w.any():
            w = target[b, at].clone().nan_to_num(0).clamp(min=0)
        c = w.cumsum(0)
        hit = (c > float(u[b, 0]) * c[-1]).nonzero()
        said.append(int(hit[0]) if len(hit) else (int(w.nonzero()[-1]) if w.any() else 0))
        result.append((said, path))
    return result


def check_verdict(out, want):
    assert all(t.dtype == torch.int64 for t in out)
    for b, (said, path) in enumerate(want):
        assert int(out.counts[b]) == len(path) - 1
        assert out.path[b].tolist() == path + [-1] * (out.path.shape[1] - len(path))
        assert out.tokens[b].tolist() == said + [-1] * (out.tokens.shape[1] - len(said))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [1, 2, 7, 2048, 2049, 5000])
@pytest.mark.parametrize("T", [1, 2, 6, 33])
@pytest.mark.parametrize("mode", ["sampled", "chain", "tree", "shared"])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_verify_matches_walk(device, V, T, mode, dtype):
    B = 5
    g = torch.Generator().manual_seed(V * 100 + T)
    logits = torch.randn(B, T, V, generator=g) * 2
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :-1] + torch.randn(B, T - 1, V, generator=g), -1).to(dtype)
    tokens = torch.randint(0, V, (B, T), generator=g)
    if mode in ("sampled", "chain") and T > 1:
        tokens[:, 1:] = torch.multinomial(draft.float().reshape(-1, V), 1, generator=g).view(B, T - 1)
        tokens[0, T // 2] = -1  # a shorter draft
        tokens[1, 1] = V
    parents = None
    if mode in ("tree", "shared"):
        parents = torch.stack([torch.tensor([-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, T)]) for _ in range(B)])
        parents[2, T // 2 :] = -1
        best = target.float().topk(min(V, 4), -1).indices
        for b in range(B):
            for i in range(1, T):
                tokens[b, i] = best[b, max(int(parents[b, i]), 0), i % best.shape[-1]]  # the same token twice among them
        if mode == "shared":
            parents = parents[0]
    u = torch.rand(B, T, generator=g)
    u[3] = 0.0
    u[4, 0] = 1 - 2**-24
    args = [target, tokens, u, draft if mode == "sampled" else None, parents]
    out = verify_draft(*[a if a is None else a.to(device) for a in args])
    check_verdict(out, verify64(*args))


@pytest.mark.parametrize("device", DEVICES)
def test_verify_borders(device):
    """Comparisons at equality, residuals without weight, rows without weight, NaN."""
    V = 6
    rows = torch.tensor([
        [0.25, 0.25, 0.25, 0.25, 0.0, 0.0],
        [0.0, 0.0, 1.0, 0.0, 0.0, 0.0],
        [0.0, 0.0, 0.0, 0.0, 0.0, 0.0],
        [math.nan, 0.5, math.nan, 0.5, math.nan, math.nan],
    ])
    tokens = torch.tensor([[0, 1, 2]]).repeat(4, 1)
    target = rows[:, None].repeat(1, 3, 1)
    for u0, u1 in itertools.product((0.0, 0.25, 0.5, 0.75, 0.999), (0.0, 0.2499, 0.25, 0.9)):
        u = torch.tensor([[u0, u1, u1]]).repeat(4, 1)
        for draft, parents in [(None, None), (target[:, :2], None), (None, torch.tensor([-1, 0, 0])), (None, torch.tensor([-1, 0, 1]))]:
            args = [target, tokens, u, draft, parents]
            check_verdict(verify_draft(*[a if a is None else a.to(device) for a in args]), verify64(*args))
    # a draft that is above the target everywhere leaves no residual: the answer comes from the target's row
    draft = torch.full((1, 1, V), 0.5)
    args = [target[:1, :2], torch.tensor([[0, 0]]), torch.tensor([[0.6, 0.9]]), draft, None]
    out = verify_draft(*[a if a is None else a.to(device) for a in args])
    assert out.counts.tolist() == [0] and out.tokens.tolist() == [[2, -1]]


@pytest.mark.parametrize("device", DEVICES)
def test_verify_no_residual_over_a_large_vocabulary(device):
    V = 10_000
    g = torch.Generator().manual_seed(80)
    target = torch.softmax(torch.randn(2, 2, V, generator=g), -1)
    draft = target[:, :1] * 2
    for u0 in (0.0, 0.3, 0.9999):
        args = [target, torch.tensor([[0, 5], [0, 9999]]), torch.tensor([[u0, 0.9], [u0, 0.9]]), draft, None]
        check_verdict(verify_draft(*[a if a is None else a.to(device) for a in args]), verify64(*args))


@pytest.mark.parametrize("device", DEVICES)
def test_verify_views_and_empty(device):
    g = torch.Generator().manual_seed(81)
    B, T, V = 3, 4, 501
    wide = torch.softmax(torch.randn(B, 2 * T, V + 3, generator=g), -1)
    target = wide[:, ::2, 2:-1]
    draft = wide[:, 1:-2:2, 1:-2]
    tokens = torch.randint(0, V, (2 * B, T), generator=g)[::2]
    u = torch.rand(T, B, generator=g).double().t()
    for d in (draft, None):
        args = [target, tokens, u, d, None]
        check_verdict(verify_draft(*[a if a is None else a.to(device) for a in args]), verify64(*args))
    out = verify_draft(target[:0].to(device), tokens[:0].to(device), u[:0].to(device))
    assert out.tokens.shape == (0, T) and out.counts.shape == (0,)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1024, 300])
def test_verify_wide_trees(device, T):
    """All nodes are children of the root, a token twice among them, all but the last refused."""
    g = torch.Generator().manual_seed(T)
    V = 2000
    order = torch.randperm(V, generator=g)
    tokens = order[torch.arange(T) % (T - 100)].repeat(2, 1)  # the last 100 for the second time
    tokens[1, -1] = order[-1]
    parents = torch.zeros(T, dtype=torch.int64)
    parents[0] = -1
    target = torch.softmax(torch.randn(2, T, V, generator=g), -1)
    u = torch.full((2, T), 0.9)
    u[1, -1] = 0.0
    args = [target, tokens, u, None, parents]
    out = verify_draft(*[a if a is None else a.to(device) for a in args])
    assert out.counts.tolist() == [0, 1] and out.path[1, 1] == T - 1
    check_verdict(out, verify64(*args))


def test_verify_keeps_the_targets_distribution():
    """Over all drafts and numbers of a small vocabulary, the first token is distributed as the target's row."""
    g = torch.Generator().manual_seed(82)
    V, n = 4, 20000
    p, q = torch.softmax(torch.randn(V, generator=g), 0), torch.softmax(torch.randn(V, generator=g), 0)
    target = p.expand(n, 2, V)
    u = torch.rand(n, 4, generator=g)
    drawn = torch.multinomial(q, n, replacement=True, generator=g)
    tokens = torch.stack((torch.zeros(n, dtype=torch.long), drawn), 1)
    runs = [
        verify_draft(target, tokens, u[:, :2], draft_probs=q.expand(n, 1, V)),
        verify_draft(p.expand(n, 4, V), torch.tensor([0, 3, 1, 3]).expand(n, 4), u, parents=torch.tensor([-1, 0, 0, 0])),
    ]
    for out in runs:
        share = torch.bincount(out.tokens[:, 0], minlength=V) / n
        # five standard deviations of a share of n draws
        assert ((share - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all(), (share, p)


@pytest.mark.parametrize("device", DEVICES)
def test_verify_refuses(device):
    B, T, V = 2, 3, 10
    p = torch.full((B, T, V), 0.1, device=device)
    tokens, u = torch.zeros(B, T, dtype=torch.long, device=device), torch.zeros(B, T, device=device)
    parents = torch.tensor([-1, 0, 0], device=device)
    bad = [
        (p[0], tokens, u, None, None),
        (p, tokens.int(), u, None, None),
        (p, tokens[:, :2], u, None, None),
        (p, tokens, u.half(), None, None),
        (p, tokens, u[:1], None, None),
        (p, tokens, u, p, None),
        (p, tokens, u, p[:, :2].half(), None),
        (p, tokens, u, p[:, :2], parents),
        (p, tokens, u, None, parents.int()),
        (p, tokens, u, None, parents[:2]),
        (p, tokens, u, None, parents.expand(3, 3)),
        (p[:, :0], tokens[:, :0], u[:, :0], None, None),
        (p[..., :0], tokens, u, None, None),
    ]
    for args in bad:
        with pytest.raises(RuntimeError):
            verify_draft(*args)
    if device == "cuda":
        with pytest.raises(RuntimeError):
            verify_draft(p, tokens.cpu(), u)


# ---- together -------------------------------------------------------------------------------------------------------


def decode_step(cache, q, k, v, cos, sin, target, tokens, u, parents):
    """One step with a drafted tree: positions by depth, into the cache, attention, verification, the path kept."""
    mask = draft_tree_mask(parents)
    positions = cache.lengths.long()[:, None] + mask.sum(-1) - 1
    q, k = rotary_embedding(q, k, cos, sin, positions=positions)
    cache.append(k, v)
    out = cache_attention(q, cache, mask=mask)
    verdict = verify_draft(target, tokens, u, parents=parents)
    cache.keep(verdict.path)
    cache.advance(verdict.counts + 1)
    return (out, *verdict)


def step_inputs(device, T=7, V=3000, B=2, seed=90):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, h, T, 64, generator=g).to(BF16) for h in (8, 2, 2))
    target = torch.softmax(torch.randn(B, T, V, generator=g) * 3, -1)
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 3])
    tokens = target.topk(3, -1).indices[:, parents.clamp(min=0), torch.arange(T) % 3]
    return [t.to(device) for t in (q, k, v, target, tokens, torch.rand(B, T, generator=g), parents)]


@gpu
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
def test_a_step_of_all_matches_the_host(quant):
    caches, cos_sin = {}, rope_tables(600, 64)
    for device in ("cpu", "cuda"):
        caches[device] = filled_cache(2, 2, 500, 64, [300, 7], 7, BF16, quant, device)
    for seed in range(4):
        got = {}
        for device, cache in caches.items():
            q, k, v, target, tokens, u, parents = step_inputs(device, seed=seed)
            got[device] = decode_step(cache, q, k, v, *(t.to(device) for t in cos_sin), target, tokens, u, parents)
        for a, b in zip(got["cpu"][1:], got["cuda"][1:]):
            assert torch.equal(a, b.cpu())
        assert torch.equal(caches["cpu"].lengths, caches["cuda"].lengths.cpu())
        # the rotation's products may be fused on one side: a step of bf16, and for codes one of theirs. Random errors
        # of that size in the scores and the values: compared by their norm
        a, b = got["cpu"][0].double(), got["cuda"][0].cpu().double()
        assert (a - b).norm() <= 8 * half_step(BF16) * a.norm()


@gpu
@pytest.mark.parametrize("quant", ["int8", None])
def test_a_captured_step_replays(quant):
    """The same graph over a cache that grows, with eager work between, against an eager cache. Two graphs, in turn."""
    cos, sin = rope_tables(600, 64, device="cuda")
    eager = filled_cache(2, 2, 500, 64, [300, 7], 7, BF16, quant, "cuda")
    graphs = []
    for _ in range(2):
        cache = filled_cache(2, 2, 500, 64, [300, 7], 7, BF16, quant, "cuda")
        inputs = step_inputs("cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode_step(cache, *inputs[:3], cos, sin, *inputs[3:])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        cache.lengths.copy_(torch.tensor([300, 7]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = decode_step(cache, *inputs[:3], cos, sin, *inputs[3:])
        graphs.append((graph, cache, inputs, out))
    for seed in range(5):
        fresh = step_inputs("cuda", seed=seed)
        want = decode_step(eager, *fresh[:3], cos, sin, *fresh[3:])
        for graph, cache, inputs, out in graphs:
            for held, new in zip(inputs, fresh):
                held.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            assert torch.equal(cache.lengths, eager.lengths)


@gpu
def test_captured_rotary_gradient_replays():
    cos, sin = rope_tables(64, 32, device="cuda")
    q = randn(2, 4, 16, 32, dtype=BF16, device="cuda").requires_grad_()
    dq = randn(2, 4, 16, 32, seed=1, dtype=BF16, device="cuda")

    def step():
        return torch.autograd.grad(rotary_embedding(q, None, cos, sin), q, dq)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        dq.copy_(randn(2, 4, 16, 32, seed=10 + seed, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


@gpu
def test_other_streams():
    """Calls on a side stream, after waits as torch asks for, and twice at once on two caches."""
    cos, sin = rope_tables(600, 64, device="cuda")
    want_cache = filled_cache(2, 2, 500, 64, [300, 7], 7, BF16, "fp8", "cuda")
    inputs = step_inputs("cuda")
    want = decode_step(want_cache, *inputs[:3], cos, sin, *inputs[3:])
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches = [filled_cache(2, 2, 500, 64, [300, 7], 7, BF16, "fp8", "cuda") for _ in streams]
    results = []
    for stream, cache in zip(streams, caches):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            results.append(decode_step(cache, *inputs[:3], cos, sin, *inputs[3:]))
    torch.cuda.synchronize()
    for out in results:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@gpu
def test_rotary_second_gradient():
    """Of sum(w * grad): the rotation is its own gradient's gradient."""
    cos, sin = rope_tables(16, 8, device="cuda")
    q, k = randn(1, 2, 5, 8, device="cuda").requires_grad_(), randn(1, 1, 5, 8, seed=1, device="cuda").requires_grad_()
    dq, dk = randn(1, 2, 5, 8, seed=2, device="cuda").requires_grad_(), randn(1, 1, 5, 8, seed=3, device="cuda").requires_grad_()
    gq, gk = torch.autograd.grad(rotary_embedding(q, k, cos, sin), (q, k), (dq, dk), create_graph=True)
    w = randn(1, 2, 5, 8, seed=4, device="cuda")
    (second,) = torch.autograd.grad((gq * w).sum(), dq)
    check_rotated(second, w, cos, sin, None, False)


@pytest.mark.parametrize("device", DEVICES)
def test_cache_without_slots_gives_zeros(device):
    cache = KVCache(2, 1, 0, 32, dtype=BF16, device=device)
    mask = torch.zeros(3, 0, dtype=torch.bool, device=device)
    q = torch.ones(2, 2, 3, 32, dtype=BF16, device=device)
    assert not cache_attention(q, cache, mask=mask).any()
    with pytest.raises(RuntimeError):
        cache_attention(q, cache)


@gpu
@pytest.mark.parametrize("quant", [None, "int8"])
@pytest.mark.parametrize("T", [3, 50])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30])
def test_cache_attention_scales(quant, T, scale):
    cache = filled_cache(2, 1, 200, 64, [0, 100], T, BF16, quant, "cuda")
    q = randn(2, 2, T, 64, seed=73, dtype=BF16, device="cuda")
    check_attention(cache_attention(q, cache, scale=scale), q, cache, None, scale)


@gpu
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
@pytest.mark.parametrize("T", [5, 20, 70])
def test_cache_attention_odd_tokens_reach_those_that_see_them(quant, T):
    """A token with NaN among the new ones and one before them, for few and many rows, with splits."""
    cache = filled_cache(1, 1, 700, 64, [600], T, BF16, quant, "cuda")
    k, v = randn(1, 1, T, 64, seed=74, dtype=BF16, device="cuda"), randn(1, 1, T, 64, seed=75, dtype=BF16, device="cuda")
    v[0, 0, 3, 9] = math.nan
    cache.append(k, v)
    q = randn(1, 2, T, 64, seed=76, dtype=BF16, device="cuda")
    mask = (torch.rand(T, T, generator=torch.Generator().manual_seed(77)) < 0.5).cuda()
    out = cache_attention(q, cache, mask=mask)
    check_attention(out, q, cache, mask)
    assert torch.equal(torch.isnan(out[0, 0, :, 9]), mask[:, 3]) and torch.isfinite(out[0, :, ~mask[:, 3]]).all()
    # among those that stand: in a tile that all see, and in the last one before the new tokens
    for slot in (100, 599):
        cache.lengths.fill_(slot)
        cache.append(k[:, :, 3:4], v[:, :, 3:4])
        cache.lengths.fill_(600)
        assert torch.isnan(cache_attention(q, cache, mask=mask)[..., 9]).all()
        cache.lengths.fill_(slot)
        cache.append(k[:, :, 2:3], v[:, :, 2:3])
        cache.lengths.fill_(600)


@gpu
@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_cache_attention_infinite_values_among_the_standing(T, dtype):
    """Far from the new tokens, where no mask is: an infinity stays one, two of unlike signs and NaN are NaN."""
    cache = filled_cache(2, 1, 1200, 64, [1100, 300], T, dtype, None, "cuda")
    cache.v[:, :, 40, 1] = math.inf
    cache.v[:, :, 50, 2] = -math.inf
    cache.v[:, :, 60, 3] = math.nan
    cache.v[:, :, 70, 4] = math.inf
    cache.v[:, :, 200, 4] = -math.inf
    q = randn(2, 4, T, 64, seed=78, dtype=dtype, device="cuda")
    out = cache_attention(q, cache)
    check_attention(out, q, cache, None)
    assert (out[..., 1] == math.inf).all() and (out[..., 2] == -math.inf).all()
    assert torch.isnan(out[..., 3:5]).all() and torch.isfinite(out[..., 5:]).all() and torch.isfinite(out[..., 0]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_without_positions_in_the_tables(device):
    empty = torch.empty(0, 4, device=device)
    y = rotary_embedding(randn(1, 1, 2, 12, device=device), None, empty, empty, positions=torch.zeros(2, dtype=torch.long, device=device))
    assert torch.isnan(y[..., :8]).all() and torch.isfinite(y[..., 8:]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_cache_refuses_odd_lengths(device):
    with pytest.raises(ValueError):
        KVCache(2, 1, 8, 32, device=device, lengths=torch.zeros(4, dtype=torch.int32, device=device)[::2])
    cache = KVCache(2, 1, 8, 32, dtype=BF16, device=device)
    cache.lengths.copy_(torch.tensor([-5, 1000]))  # behind the ends: as the nearest length
    q = torch.ones(2, 1, 2, 32, dtype=BF16, device=device)
    check_attention(cache_attention(q, cache), q, cache, None)


def test_rope_scaling_refuses_what_it_does_not_know():
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    for more in ({"mscale": 1.0}, {"truncate": False}, {"rope_theta": 1e6}):
        with pytest.raises(ValueError, match=next(iter(more))):
            rope_frequencies(64, 1e4, {**yarn, **more})
    rope_frequencies(64, 1e4, {**yarn, "beta_fast": 16, "beta_slow": 2, "attention_factor": 1.0})


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("offset", [0, 3])
def test_append_of_the_caches_own_rows(device, offset):
    g = torch.Generator().manual_seed(5)
    cache = KVCache(2, 2, 300, 64, dtype=BF16, device=device)
    k, v = torch.randn(2, 2, 2, 300, 64, generator=g).to(BF16).to(device)
    cache.append(k, v)
    cache.append(cache.k[:, :, 1:280], cache.v[:, :, 1:280], offset=offset)
    for held, was in ((cache.k, k), (cache.v, v)):
        assert torch.equal(held[:, :, offset : offset + 279], was[:, :, 1:280])
        assert torch.equal(held[:, :, offset + 279 :], was[:, :, offset + 279 :])
        assert torch.equal(held[:, :, :offset], was[:, :, :offset])
