"""Serving operators where a value, a weight or a call is extreme: small weights, infinities, types, refusals."""

import math

import pytest
import torch
from torch.autograd import forward_ad

from accelerate_amd.models import LlamaConfig, LlamaForCausalLM
from accelerate_amd.ops import KVCache, cache_attention, rope_tables, rotary_embedding, verify_draft
from test_serving_generate import models, prompt

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- attention: weights far below the largest -----------------------------------------------------------------------


def sink_cache(B, H, n, D, quant, sink_value, gap, others):
    """n tokens, one of which (the 7th) has a score higher by `gap` powers of two than the others', which are alike; its
    value is `sink_value`, theirs are `others` [n, D]. Returns the cache, the last token not advanced over, and a query."""
    cache = KVCache(B, H, n, D, dtype=FP16, quant=quant, device="cuda")
    k, v = torch.zeros(1, 1, n, D, dtype=FP16), others.to(FP16).expand(1, 1, n, D).clone()
    k[..., 7, 0], v[..., 7, :] = 8.0, sink_value
    cache.append(k.expand(B, H, n, D).cuda(), v.expand(B, H, n, D).cuda())
    cache.lengths.fill_(n - 1)
    q = torch.zeros(B, H, 1, D, dtype=FP16)
    q[..., 0] = gap * math.log(2)
    return cache, q.cuda()


def check_weighted(out, q, cache, scale):
    """Against the definition in 64 bits, with what the cache holds."""
    n = cache.max_len
    k, v = (x[0, 0].double().cpu() for x in cache.read(dtype=FP32))
    s = k @ q[0, 0, 0].double().cpu() * scale
    p = torch.exp(s - s.max())
    total = p.sum()
    want, size = p @ v / total, p @ v.abs() / total
    # A score has one product that is not zero: it and its scales are rounded four times, its difference to the largest
    # once, its exponential to 2 steps (of 32 bits). A probability is held in 16 bits at least, and one below 2^-40 of
    # the largest may be lost. Sums of n terms are in 32 bits.
    score = 6 * half_step(FP32) * s.abs().max() + 4 * half_step(FP32)
    tolerance = (2**-16 * 1.01 + 2 * score + 2 * (n + 64) * half_step(FP32)) * size
    tolerance += n * 2.0**-40 * v.abs().max() / total
    tolerance += half_step(FP16) * 1.01 * want.abs() + 2.0**-25  # the result's own rounding
    got = out.double().cpu()
    assert torch.equal(got, got[:1, :1].expand_as(got))
    error = (got[0, 0, 0] - want).abs()
    assert (error <= tolerance).all(), (error / tolerance).max()


@gpu
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
@pytest.mark.parametrize("gap", [20.0, 24.5, 26.0, 30.0])
@pytest.mark.parametrize("B, n", [(1, 500), (1, 2000), (64, 1500)])
def test_weights_far_below_the_largest_count_in_fp16(quant, gap, B, n):
    """One token without a value takes nearly all the weight: the result is what the others' small weights sum to."""
    g = torch.Generator().manual_seed(1)
    cache, q = sink_cache(B, 4, n, 64, quant, 0.0, gap, (torch.rand(n, 64, generator=g) + 1) * 15000)
    check_weighted(cache_attention(q, cache, scale=0.125), q, cache, 0.125)


@gpu
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
@pytest.mark.parametrize("gap", [-12.0, -30.0])
def test_a_large_value_of_low_weight_leaves_the_others_their_bits_in_fp16(quant, gap):
    g = torch.Generator().manual_seed(2)
    cache, q = sink_cache(1, 4, 300, 64, quant, 30000.0, gap, torch.randn(300, 64, generator=g) * 0.01)
    check_weighted(cache_attention(q, cache, scale=0.125), q, cache, 0.125)


@gpu
@pytest.mark.parametrize("quant", [None, "int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n", [40, 1000])
def test_scores_beyond_whole_numbers_of_32_bits(quant, dtype, n):
    """Products of 2^24 and more, where 32 bits step by 2 to 32: the largest score has all the weight, and no more."""
    D, heads = 64, 32
    g = torch.Generator().manual_seed(4)
    cache = KVCache(1, 1, n, D, dtype=dtype, quant=quant, device="cuda")
    size = torch.full((n,), 0.5)
    size[n // 3], size[-1] = 1.0, 0.75  # scores lie 2^22 apart
    k = (1500 * size[:, None]).expand(n, D).to(dtype)
    v = torch.randn(n, D, generator=g).to(dtype)
    cache.append(k[None, None].cuda(), v[None, None].cuda())
    cache.lengths.fill_(n - 1)
    q = (1500 + 200 * torch.arange(heads))[:, None].expand(heads, D).to(dtype)[None, :, None]
    out = cache_attention(q.cuda(), cache)[0, :, 0].double().cpu()
    want = cache.read(dtype=FP32)[1][0, 0, n // 3].double().cpu().expand(heads, D)
    # the token's value times its weight over itself: 16 bits of the weight, a division, and the result's own rounding
    assert ((out - want).abs() <= (half_step(dtype) + 2**-16 + 4 * half_step(FP32)) * want.abs() + 2.0**-25).all()


# ---- attention: infinities ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B, H, max_len", [(1, 1, 300), (1, 1, 4096), (16, 4, 1300)])  # one workgroup a head; many splits; few
def test_an_infinite_value_of_no_weight_stays_infinite(device, B, H, max_len):
    """A token far behind has a score 184 powers of two above the others': their weights are zero in 32 bits."""
    n, D = max_len - 20, 64
    cache = KVCache(B, H, max_len, D, dtype=BF16, device=device)
    cache.v.fill_(1)
    cache.k[:, :, n - 100, 0] = 64.0
    cache.v[:, :, 3, 1], cache.v[:, :, 4, 2], cache.v[:, :, 5, 3] = math.inf, -math.inf, math.nan
    cache.v[:, :, 6, 4], cache.v[:, :, 140, 4] = math.inf, -math.inf
    cache.lengths.fill_(n - 1)
    q = torch.zeros(B, 2 * H, 1, D, dtype=BF16, device=device)
    q[:, ::2, :, 0] = 16.0  # every other head: 64 * 16 / 8 / ln 2
    out = cache_attention(q, cache).float().cpu()
    assert (out[..., 1] == math.inf).all() and (out[..., 2] == -math.inf).all() and torch.isnan(out[..., 3:5]).all()
    # the others are means of ones: sums of n terms in 32 bits, and the result's own rounding
    rest = out[..., [0, *range(5, D)]]
    assert ((rest - 1).abs() <= half_step(BF16) + 2 * (n + 64) * half_step(FP32)).all()


# ---- forward-mode derivatives ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["q", "k", "cos", "grad"])
def test_rotary_drops_no_tangent(device, which):
    """The rotation is linear: its tangent is that of the input, rotated, as on the host, or the call is refused."""
    cos, sin = rope_tables(6, 8, device=device)
    g = torch.Generator().manual_seed(3)
    q, k, dq = (torch.randn(1, 2, 6, 8, generator=g).to(device) for _ in range(3))
    t = torch.randn(1, 2, 6, 8, generator=g).to(device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(cos, torch.ones_like(cos)) if which == "cos" else forward_ad.make_dual({"q": q, "k": k, "grad": dq}[which], t)

        def call():
            if which == "grad":
                x = q.clone().requires_grad_()
                return torch.autograd.grad(rotary_embedding(x, None, cos, sin), x, dual)[0]
            y = rotary_embedding(dual if which == "q" else q, dual if which == "k" else k, dual if which == "cos" else cos, sin)
            return y[which == "k"]

        if device == "cuda":
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        else:
            assert forward_ad.unpack_dual(call()).tangent is not None


@pytest.mark.parametrize("device", DEVICES)
def test_the_cache_drops_no_tangent(device):
    cache = KVCache(1, 1, 8, 32, dtype=BF16, device=device)
    x = torch.ones(1, 1, 2, 32, dtype=BF16, device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x.clone())
        for call in (lambda: cache.append(dual, x), lambda: cache.append(x, dual), lambda: cache_attention(dual, cache)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        cache.append(x, x)
        cache_attention(x, cache)


# ---- generate -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
def test_an_int32_prompt_generates_what_an_int64_one_does(device):
    target, draft = models(device)
    ids = prompt(device)
    calls = [{}, {"cache_dtype": "int8"}, {"draft_model": draft}, {"draft_model": draft, "draft_widths": (2, 1)}]
    for kwargs in calls + [{"cache_dtype": "int8", "graph_decode": True}]:
        for n in (1, 4):
            want = target.generate(ids, max_new_tokens=n, **kwargs)
            got = target.generate(ids.int(), max_new_tokens=n, **kwargs)
            assert got.dtype == torch.int64 and torch.equal(got, want)


def test_generate_refuses_trees_beyond_what_is_verified():
    target, draft = models("cpu")
    ran = []
    for m in (target, draft):
        m.register_forward_hook(lambda *a: ran.append(1))
    for widths in ((32, 32), (1,) * 1024, (97, 97, 97, 97, 97, 97)):  # 1057, 1025 and some 10^12 nodes
        with pytest.raises(ValueError, match="1024"):
            target.generate(prompt("cpu"), max_new_tokens=4, draft_model=draft, draft_widths=widths)
    assert not ran


def test_generate_refuses_a_temperature_that_is_no_number():
    target, _ = models("cpu")
    with pytest.raises(ValueError, match="temperature"):
        target.generate(prompt("cpu"), max_new_tokens=2, temperature=math.nan)


def test_arguments_of_serving_caches_are_refused_without_them():
    """They were ignored: positions that are given would seem to be followed."""
    target, _ = models("cpu")
    ids = prompt("cpu", B=1)
    rope, positions = target.serving_rope(ids.device), torch.arange(9)[None] + 5
    mask = torch.ones(9, 9, dtype=torch.bool).tril()
    for kwargs in ({"positions": positions}, {"mask": mask}, {"offset": 1}, {"prefill": True}, {"rope": rope}):
        for caches in (None, target.make_kv_caches(1, 12, ids.device, torch.float32)):
            with pytest.raises(ValueError, match="make_serving_caches"):
                target(ids, kv_caches=caches, **kwargs)


@pytest.mark.parametrize("device", DEVICES)
def test_a_cast_model_serves_with_the_tables_that_it_is_given(device):
    config = LlamaConfig.tiny(num_hidden_layers=1, max_position_embeddings=300)
    model = LlamaForCausalLM(config).to(device=device, dtype=BF16)
    tables = rope_tables(300, config.hidden_size // config.num_attention_heads, config.rope_theta, device=device)
    rounded = model.serving_rope(torch.device(device))
    # the buffers hold what the cast left: half a step of bf16, and angles up to 300 that were rounded four times to 32 bits
    assert all((a - b).abs().max() <= 2**-9 + 300 * 4 * half_step(FP32) for a, b in zip(rounded, tables))
    model.rope_cos, model.rope_sin = tables
    for got, table in zip(model.serving_rope(torch.device(device)), tables):
        assert got.dtype == FP32 and torch.equal(got, table)
    ids = prompt(device)
    assert model.generate(ids, max_new_tokens=3, cache_dtype="int8").shape == (3, 12)


@pytest.mark.parametrize("device", DEVICES)
def test_an_fp32_model_generates_under_autocast(device):
    """Its caches are of the type that autocast gives the projections."""
    target, draft = models(device, dtype=FP32)
    ids = prompt(device)
    calls = [{"cache_dtype": "int8"}, {"draft_model": draft}, {"draft_model": draft, "draft_widths": (2, 2), "cache_dtype": "fp8"}]
    for kwargs in calls + [{"temperature": 1.0}, {"cache_dtype": "int8", "graph_decode": True}]:
        with torch.autocast(device, dtype=BF16):
            out = target.generate(ids, max_new_tokens=8, **kwargs)
        assert out.shape == (3, 17) and torch.equal(out[:, :9], ids)
        if "temperature" in kwargs:
            continue
        with torch.no_grad():
            logits = target(out)["logits"][:, 8:-1].float()
        best, got = logits.amax(-1), logits.gather(-1, out[:, 9:, None])[..., 0]
        # as in test_drafts_on_gpu_follow_the_model: the best token within the roundings of both ways through the model
        assert (best - got <= 0.1 * (best - logits.mean(-1))).all()


# ---- verification ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("before", [1, 70])
def test_a_refused_token_without_weight_takes_none_from_its_siblings(device, before):
    """NaN counts as no weight: the siblings after such a token are tested as if it had not been drafted."""
    V, T = 200, before + 3
    target = torch.zeros(2, T, V)
    target[:, :, :before] = math.nan
    target[:, :, 100], target[:, :, 101] = 0.25, 0.75
    tokens = torch.tensor([0, *range(before), 100, 101]).repeat(2, 1)
    parents = torch.tensor([-1] + [0] * (T - 1))
    u = torch.full((2, T), 0.9)
    u[0, -2] = 0.2  # below the 0.25 of token 100; the other sequence goes on to token 101 with 0.9 * 0.75
    out = verify_draft(target.to(device), tokens.to(device), u.to(device), parents=parents.to(device))
    assert out.counts.tolist() == [1, 1]
    assert out.tokens[:, 0].tolist() == [100, 101] and out.path[:, 1].tolist() == [T - 2, T - 1]
