"""LlamaForCausalLM.generate over a quantised cache, with drafted tokens, and with sampling."""

import pytest
import torch

from accelerate_amd.models import LlamaConfig, LlamaForCausalLM

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def models(device, dtype=None, **overrides):
    torch.manual_seed(0)
    config = dict(num_hidden_layers=2, vocab_size=97, max_position_embeddings=64, **overrides)
    target, draft = LlamaForCausalLM(LlamaConfig.tiny(**config)), LlamaForCausalLM(LlamaConfig.tiny(**config))
    with torch.no_grad():  # a draft that is right at times, and a target with clear choices
        for a, b in zip(draft.parameters(), target.parameters()):
            a.copy_(b + 0.3 * b.std() * torch.randn_like(b))
        for m in (target, draft):
            m.lm_head.weight.mul_(10)
    dtype = dtype or (torch.float32 if device == "cpu" else torch.bfloat16)
    return [m.eval().to(device=device, dtype=dtype) for m in (target, draft)]


def prompt(device, B=3, S=9):
    return torch.randint(0, 97, (B, S), generator=torch.Generator().manual_seed(1)).to(device)


@pytest.mark.parametrize("widths", [(1,), (1, 1, 1, 1), (3, 2), (2, 1, 2), (97,)])
def test_drafts_do_not_change_greedy_tokens(widths):
    target, draft = models("cpu")
    ids = prompt("cpu")
    for n in (1, 2, 13, 55):  # the last: to the end of the tables
        want = target.generate(ids, max_new_tokens=n)
        assert torch.equal(target.generate(ids, max_new_tokens=n, draft_model=draft, draft_widths=widths), want)
        assert torch.equal(target.generate(ids, max_new_tokens=n, draft_model=target, draft_widths=widths), want)


@gpu
@pytest.mark.parametrize("widths", [(1, 1, 1, 1), (3, 2)])
@pytest.mark.parametrize("cache_dtype", [None, "int8", "fp8"])
def test_drafts_on_gpu_follow_the_model(widths, cache_dtype):
    """Each new token is the best, within bf16's steps, after the ones before it by the same model without a cache."""
    target, draft = models("cuda")
    ids = prompt("cuda")
    out = target.generate(ids, max_new_tokens=20, draft_model=draft, draft_widths=widths, cache_dtype=cache_dtype)
    assert out.shape == (3, 29) and torch.equal(out[:, :9], ids)
    with torch.no_grad():
        logits = target(out)["logits"][:, 8:-1].float()
    best, got = logits.amax(-1), logits.gather(-1, out[:, 9:, None])[..., 0]
    spread = best - logits.mean(-1)
    # roundings of the two ways through the model, and of keys and values to 8 bits (a step of 2^-4 in e4m3)
    assert (best - got <= 0.1 * spread).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_dtype", ["int8", "fp8"])
def test_quantised_cache_stays_close(device, cache_dtype):
    target, _ = models(device)
    ids = prompt(device)
    out = target.generate(ids, max_new_tokens=12, cache_dtype=cache_dtype)
    assert torch.equal(out, target.generate(ids, max_new_tokens=12, cache_dtype=cache_dtype))
    caches = target.make_serving_caches(3, 21, ids.device, target.lm_head.weight.dtype, cache_dtype)
    with torch.no_grad():
        target(out[:, :9], kv_caches=caches, prefill=True)
        caches[0].advance(9)
        logits = []
        for i in range(9, 20):
            logits.append(target(out[:, i : i + 1], kv_caches=caches)["logits"])
            caches[0].advance(1)
        whole = target(out[:, :20])["logits"][:, 9:].float()
    logits = torch.cat(logits, 1).float()
    # a relative step of 2^-4 for e4m3, of 2^-8 of the largest for int8, in keys and values of two layers
    assert (logits - whole).norm() <= (0.15 if cache_dtype == "fp8" else 0.05) * whole.norm()


@pytest.mark.parametrize("device", DEVICES)
def test_sampling_follows_its_numbers(device):
    target, draft = models(device)
    ids = prompt(device, B=2)

    def run(seed, **kwargs):
        g = torch.Generator(device=device).manual_seed(seed)
        return target.generate(ids, max_new_tokens=10, temperature=1.5, generator=g, **kwargs)

    for kwargs in ({}, {"draft_model": draft}, {"draft_model": draft, "draft_widths": (2, 2)}, {"cache_dtype": "int8"}):
        a = run(3, **kwargs)
        assert a.shape == (2, 19) and (a >= 0).all() and (a < 97).all()
        assert torch.equal(a, run(3, **kwargs))
        assert not torch.equal(a, run(4, **kwargs))


def test_sampled_drafts_keep_the_distribution():
    """The first two new tokens of many samples, with and without a draft, against the model's own probabilities."""
    torch.manual_seed(0)
    config = dict(num_hidden_layers=1, vocab_size=5, hidden_size=32, intermediate_size=32, num_attention_heads=2,
                  num_key_value_heads=1, max_position_embeddings=32)
    target, draft = LlamaForCausalLM(LlamaConfig.tiny(**config)).eval(), LlamaForCausalLM(LlamaConfig.tiny(**config)).eval()
    for m in (target, draft):
        m.lm_head.weight.data.mul_(40)
    n = 4000
    ids = torch.tensor([[1, 2, 3]]).expand(n, 3).contiguous()
    with torch.no_grad():
        first = torch.softmax(target(ids[:1])["logits"][0, -1], -1)
        rest = [torch.softmax(target(torch.tensor([[1, 2, 3, t]]))["logits"][0, -1], -1) for t in range(5)]
    want = (first[:, None] * torch.stack(rest)).flatten()
    for widths in ((1, 1), (2, 1), (3, 2)):
        out = target.generate(ids, max_new_tokens=2, draft_model=draft, draft_widths=widths, temperature=1.0,
                              generator=torch.Generator().manual_seed(5))
        share = torch.bincount(out[:, 3] * 5 + out[:, 4], minlength=25) / n
        # five standard deviations of a share of n draws, and one draw
        assert ((share - want).abs() <= 5 * (want * (1 - want) / n).sqrt() + 1 / n).all()


@gpu
def test_graph_decode_over_a_quantised_cache_matches_eager():
    target, _ = models("cuda")
    ids = prompt("cuda")
    for n in (1, 2, 15):
        eager = target.generate(ids, max_new_tokens=n, cache_dtype="int8")
        graphed = target.generate(ids, max_new_tokens=n, cache_dtype="int8", graph_decode=True)
        assert torch.equal(eager, graphed)


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 16},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 16},
])
def test_scaled_positions_reach_both_paths(scaling):
    target, draft = models("cpu", rope_scaling=scaling)
    plain, _ = models("cpu")
    ids = prompt("cpu")
    want = target.generate(ids, max_new_tokens=20)
    assert torch.equal(target.generate(ids, max_new_tokens=20, draft_model=draft), want)
    with torch.no_grad():
        assert not torch.allclose(target(ids)["logits"], plain(ids)["logits"])


def test_generate_refuses():
    target, draft = models("cpu")
    torch.manual_seed(2)
    other = LlamaForCausalLM(LlamaConfig.tiny(num_hidden_layers=1, vocab_size=98, max_position_embeddings=64))
    short = LlamaForCausalLM(LlamaConfig.tiny(num_hidden_layers=1, vocab_size=97, max_position_embeddings=16))
    ids = prompt("cpu")
    for kwargs in (
        {"cache_dtype": "int4"},
        {"temperature": -1.0},
        {"draft_model": other},
        {"draft_model": short},
        {"draft_model": draft, "draft_widths": ()},
        {"draft_model": draft, "draft_widths": (2, 0)},
        {"draft_model": draft, "draft_widths": (98,)},
        {"draft_model": draft, "max_new_tokens": 56},
        {"draft_model": draft, "max_new_tokens": 0},
        {"draft_model": draft, "graph_decode": True},
        {"cache_dtype": "int8", "temperature": 1.0, "graph_decode": True},
    ):
        with pytest.raises(ValueError):
            target.generate(ids, **{"max_new_tokens": 8, **kwargs})


@gpu
def test_graph_decode_with_tables_left_on_the_host():
    """A model that was built on the GPU has its rotary tables on the host still."""
    target, _ = models("cuda")
    ids = prompt("cuda")
    want = target.generate(ids, max_new_tokens=6, cache_dtype="int8")
    target.rope_cos, target.rope_sin = target.rope_cos.cpu(), target.rope_sin.cpu()
    for graph_decode in (False, True):
        assert torch.equal(target.generate(ids, max_new_tokens=6, cache_dtype="int8", graph_decode=graph_decode), want)
