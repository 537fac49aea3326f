"""The operators of serving with drafted tokens over a cache: what is measured of them.

Four operators that one decoding step of a language model calls in turn: rotary positions, the cache that holds keys and
values in 8 (or 16) bits, attention of a few tokens over that cache, and the verification of drafted tokens.

Where ``own`` is false ``run`` computes them in elementary torch operations; where it is true it makes the framework's calls.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INT8_MAX = 127.0
FP8_MAX = 448.0
THETA = 500000.0
# tables made for contexts longer than the model was trained on
SCALINGS = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {
        "rope_type": "llama3",
        "factor": 8.0,
        "low_freq_factor": 1.0,
        "high_freq_factor": 4.0,
        "original_max_position_embeddings": 8192,
    },
    "yarn": {
        "rope_type": "yarn",
        "factor": 16.0,
        "beta_fast": 32.0,
        "beta_slow": 1.0,
        "original_max_position_embeddings": 8192,
    },
}


def listed():
    return [
        # one token of one request, far into a long context: latency alone
        rope_case("rope_decode_1", 1, 1, 32, 8, 128, 128, False, "bf16", "ragged", "llama3", False),
        # a training step of the 8B configuration at its full length, with the gradients of both inputs
        rope_case("rope_train_8b", 2, 8192, 32, 8, 128, 128, False, "bf16", "start", "none", True),
        # a partly rotated head with neighbouring pairs, an odd length, drafted tokens that share positions
        rope_case("rope_partial_odd", 3, 1537, 20, 20, 96, 48, True, "fp32", "ragged", "yarn", True),
        # a decoding step of 64 requests writes one token each behind caches of unlike lengths
        cache_case("cache_step_int8", 64, 8, 1, 128, 4096, "int8", "bf16"),
        # the prompt of four requests goes into the cache and comes back for the chunk that follows it
        cache_case("cache_prompt_fp8", 4, 8, 7001, 128, 8192, "fp8", "bf16"),
        cache_case("cache_prompt_int8_fp16", 2, 20, 1000, 64, 1024, "int8", "fp16"),
        # one request, a short context, a 16-bit cache: latency alone
        attention_case("attend_decode_short", 1, 32, 8, 1, 128, 300, 512, "same", "bf16", "chain"),
        # a decoding step of a busy server: 32 requests of the 70B configuration, an int8 cache
        attention_case("attend_decode_batch", 32, 64, 8, 1, 128, 16000, 16384, "int8", "bf16", "chain"),
        # one request with a very long context
        attention_case("attend_decode_long", 1, 32, 8, 1, 128, 130001, 131072, "same", "bf16", "chain"),
        # trees of drafted tokens for some requests
        attention_case("attend_tree_fp8", 8, 32, 8, 27, 128, 4000, 4224, "fp8", "bf16", "tree"),
        # chains of five sampled drafts, with the probabilities that they were drawn from
        verify_case("verify_chain_8b", 8, 6, 128256, "chain", True, "fp32"),
        # trees of a draft's best tokens, the small vocabulary of an odd size
        verify_case("verify_tree_gpt2", 2, 22, 50257, "tree", False, "fp32"),
    ]


def rope_case(name, batch, seq, q_heads, k_heads, head_dim, rotary_dim, interleaved, dtype, positions, scaling, backward):
    return dict(name=name, op="rope", batch=batch, seq=seq, q_heads=q_heads, k_heads=k_heads, head_dim=head_dim,
                rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype, positions=positions, scaling=scaling,
                backward=backward)


def cache_case(name, batch, heads, tokens, head_dim, max_len, kind, dtype):
    return dict(name=name, op="cache", batch=batch, heads=heads, tokens=tokens, head_dim=head_dim, max_len=max_len,
                kind=kind, dtype=dtype)


def attention_case(name, batch, q_heads, kv_heads, tokens, head_dim, context, max_len, kind, dtype, mask):
    return dict(name=name, op="attention", batch=batch, q_heads=q_heads, kv_heads=kv_heads, tokens=tokens,
                head_dim=head_dim, context=context, max_len=max_len, kind=kind, dtype=dtype, mask=mask)


def verify_case(name, batch, nodes, vocab, shape, draft_probs, dtype):
    return dict(name=name, op="verify", batch=batch, nodes=nodes, vocab=vocab, shape=shape, draft_probs=draft_probs,
                dtype=dtype)


def draw(rng):
    def spread(low, high):  # even over the logarithm
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    while True:
        op = rng.choice(["rope", "cache", "attention", "attention", "verify"])
        if op == "rope":
            head_dim = rng.choice([32, 64, 80, 96, 128, 256])
            k_heads = rng.choice([1, 2, 4, 8, 20])
            case = rope_case(None, spread(1, 16), spread(1, 8192), k_heads * rng.choice([1, 2, 4, 8]), k_heads, head_dim,
                             rng.choice([head_dim, head_dim, head_dim // 2]), rng.random() < 0.5,
                             rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["start", "ragged"]),
                             rng.choice(sorted(SCALINGS)), rng.random() < 0.5)
        elif op == "cache":
            tokens = spread(1, 8192)
            case = cache_case(None, spread(1, 64), rng.choice([1, 2, 4, 8, 20]), tokens, rng.choice([32, 64, 128, 256]),
                              tokens + spread(1, 4096), rng.choice(["int8", "fp8", "same"]),
                              rng.choice(["bf16", "bf16", "fp16"]))
        elif op == "attention":
            kv_heads, context, tokens = rng.choice([1, 2, 4, 8, 20]), spread(1, 131072), spread(1, 64)
            if rng.random() < 0.5:
                tokens = 1
            case = attention_case(None, spread(1, 64), kv_heads * rng.choice([1, 2, 4, 8]), kv_heads, tokens,
                                  rng.choice([32, 64, 128, 128, 256]), context, context + tokens + spread(1, 4096),
                                  rng.choice(["int8", "fp8", "same"]), rng.choice(["bf16", "bf16", "fp16"]),
                                  rng.choice(["chain", "tree"]))
        else:
            shape = rng.choice(["chain", "tree"])
            case = verify_case(None, spread(1, 32), spread(2, 32), rng.choice([32000, 50257, 128256, spread(100, 128256)]),
                               shape, shape == "chain" and rng.random() < 0.7, rng.choice(["fp32", "fp32", "bf16"]))
        del case["name"]
        w = work(case)
        if w["bytes"] <= 8.0e8 and w["flops"] <= 4.0e10 and _footprint(case) <= 8e9:
            return case


def _footprint(case):
    """Bytes of a state and of the plain form's intermediates, roughly."""
    if case["op"] == "rope":
        return 40 * case["batch"] * case["seq"] * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
    if case["op"] == "cache":
        return 24 * case["batch"] * case["max_len"] * case["heads"] * case["head_dim"]
    if case["op"] == "attention":
        slots = case["batch"] * case["max_len"]
        return slots * (12 * case["kv_heads"] * case["head_dim"] + 12 * case["q_heads"] * case["tokens"])
    return 16 * case["batch"] * case["nodes"] * case["vocab"]


def work(case):
    if case["op"] == "rope":
        tokens = case["batch"] * case["seq"]
        values = tokens * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        passes = 2 if case["backward"] else 1
        table = (tokens if case["positions"] == "ragged" else case["seq"]) * case["rotary_dim"] * 4
        return {"bytes": passes * (2 * values * DTYPES[case["dtype"]].itemsize + table), "flops": passes * 3 * values}
    if case["op"] == "cache":  # written (read in 16 bits, written in 8 with a scale a row) and read back
        rows = 2 * case["batch"] * case["heads"] * case["tokens"]
        held = case["head_dim"] * (2 if case["kind"] == "same" else 1) + (0 if case["kind"] == "same" else 4)
        return {"bytes": rows * 2 * (case["head_dim"] * 2 + held), "flops": rows * case["head_dim"] * 4}
    if case["op"] == "attention":
        slots = sum(_lengths(case)) + case["batch"] * case["tokens"]
        held = case["head_dim"] * (2 if case["kind"] == "same" else 1) + (0 if case["kind"] == "same" else 4)
        rows = case["batch"] * case["q_heads"] * case["tokens"]
        return {"bytes": 2 * slots * case["kv_heads"] * held + 2 * rows * case["head_dim"] * 2,
                "flops": 4 * slots * case["q_heads"] * case["tokens"] * case["head_dim"]}
    # one row of probabilities a sequence, and with the draft's own a second one; a value for each drafted token
    rows = case["batch"] * (2 if case["draft_probs"] else 1)
    size = DTYPES[case["dtype"]].itemsize
    return {"bytes": rows * case["vocab"] * size + case["batch"] * case["nodes"] * (16 + 2 * size),
            "flops": rows * case["vocab"] * 2}


def _lengths(case):
    """Tokens in the cache before the new ones: the first sequence has the case's context, the others down to half of it."""
    n = case["batch"]
    return [case["context"] - (case["context"] * i) // (2 * n) for i in range(n)]


# ---- inputs ---------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"rope": _prepare_rope, "cache": _prepare_cache, "attention": _prepare_attention,
             "verify": _prepare_verify}[case["op"]](case, g)
    state["case"] = case
    return state


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _prepare_rope(case, g):
    B, S, D, dtype = case["batch"], case["seq"], case["head_dim"], DTYPES[case["dtype"]]
    max_pos = 131072 if case["positions"] == "ragged" else S
    state = {
        "q": _normal(g, B, S, case["q_heads"] * D, dtype=dtype),  # as the projections give them
        "k": _normal(g, B, S, case["k_heads"] * D, dtype=dtype),
        "positions": None,
    }
    if case["positions"] == "ragged":
        start = torch.randint(0, max_pos - S, (B, 1), generator=g, device="cuda")
        state["positions"] = start + torch.arange(S, device="cuda") // 2  # pairs of siblings share a position
    if case["backward"]:
        state["dq"] = _normal(g, B, case["q_heads"], S, D, dtype=dtype)
        state["dk"] = _normal(g, B, case["k_heads"], S, D, dtype=dtype)
    scaling = SCALINGS[case["scaling"]]
    if own:
        from accelerate_amd.ops import rope_tables

        state["cos"], state["sin"] = rope_tables(max_pos, case["rotary_dim"], theta=THETA, scaling=scaling, device="cuda")
    else:
        freq, factor = _plain_frequencies(case["rotary_dim"], scaling)
        angle = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * freq[None]
        state["cos"], state["sin"] = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    return state


def _plain_frequencies(rotary_dim, scaling):
    pair = torch.arange(0, rotary_dim, 2, device="cuda", dtype=torch.float64)
    freq, factor = THETA ** (-pair / rotary_dim), 1.0
    if scaling is None:
        return freq, factor
    s = scaling["factor"]
    if scaling["rope_type"] == "linear":
        return freq / s, factor
    trained = scaling["original_max_position_embeddings"]
    if scaling["rope_type"] == "llama3":  # slow pairs are slowed by the factor, fast ones kept, a ramp between
        turns = trained * freq / (2 * math.pi)
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return freq * (keep + (1 - keep) / s), factor

    def index(turns):  # the pair that turns so often over the trained length
        return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(THETA))

    low = max(math.floor(index(scaling["beta_fast"])), 0)
    high = min(math.ceil(index(scaling["beta_slow"])), rotary_dim - 1)
    ramp = ((pair / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
    return freq * ((1 - ramp) + ramp / s), 0.1 * math.log(s) + 1.0


def _prepare_cache(case, g):
    B, H, T, D, dtype = case["batch"], case["heads"], case["tokens"], case["head_dim"], DTYPES[case["dtype"]]
    room = case["max_len"] - T
    channel = torch.exp(_normal(g, H * D))  # some channels are much larger than others, as keys have them
    state = {
        "k": (_normal(g, B, T, H * D) * channel).to(dtype),
        "v": _normal(g, B, T, H * D, dtype=dtype),
        "lengths": torch.randint(0, room + 1, (B,), generator=g, device="cuda", dtype=torch.int32),
    }
    if own:
        from accelerate_amd.ops import KVCache

        cache = KVCache(B, H, case["max_len"], D, dtype=dtype, quant=None if case["kind"] == "same" else case["kind"],
                        device="cuda")
        cache.lengths.copy_(state["lengths"])
        state["cache"] = cache
    else:
        held = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "same": dtype}[case["kind"]]
        for name in ("k", "v"):
            state["held_" + name] = torch.zeros(B, H, case["max_len"], D, device="cuda", dtype=held)
            state["scale_" + name] = torch.zeros(B, H, case["max_len"], device="cuda")
    return state


def _prepare_attention(case, g):
    B, H, L, D, dtype = case["batch"], case["kv_heads"], case["max_len"], case["head_dim"], DTYPES[case["dtype"]]
    T, kind = case["tokens"], case["kind"]
    state = {"q": _normal(g, B, T, case["q_heads"] * D, dtype=dtype),
             "lengths": torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)}
    for name in ("k", "v"):
        if kind == "same":
            state[name] = _normal(g, B, H, L, D, dtype=dtype)
        else:
            size = _normal(g, B, H, L).abs() * 0.3 + 0.7  # some tokens are larger than others
            if kind == "int8":
                state[name] = torch.empty(B, H, L, D, device="cuda", dtype=torch.int8).random_(-127, 128, generator=g)
                state["scale_" + name] = size * (1.7 / INT8_MAX)
            else:
                state[name] = _normal(g, B, H, L, D, dtype=torch.bfloat16).mul_(60).clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
                state["scale_" + name] = torch.exp2(torch.round(torch.log2(size / 60)))
    state["mask"] = None
    if case["mask"] == "tree":  # every drafted token sees the one that it follows, and what that one sees
        parent = _parents(g, B, T)
        state["mask"] = _ancestors(parent)
    if own:
        from accelerate_amd.ops import KVCache

        cache = KVCache(B, H, L, D, dtype=dtype, quant=None if kind == "same" else kind, device="cuda")
        cache.lengths.copy_(state["lengths"])
        for name in ("k", "v"):
            getattr(cache, name).copy_(state.pop(name))
            if kind != "same":
                getattr(cache, name + "_scale").copy_(state.pop("scale_" + name))
        state["cache"] = cache
    return state


def _parents(g, batch, nodes):
    """Random trees: node 0 is the root, a later node follows one of those before it, mostly a near one."""
    at = torch.arange(nodes, device="cuda")
    back = 1 + (torch.rand(batch, nodes, generator=g, device="cuda") ** 2 * torch.clamp(at, max=6)).long()
    return torch.where(at[None] == 0, -1, (at[None] - back).clamp(min=0))


def _ancestors(parent):
    """[B, T, T]: whether j is i or one that i follows."""
    nodes = parent.shape[1]
    at = torch.arange(nodes, device=parent.device)
    reach = ((parent[:, :, None] == at) | (at[:, None] == at)).double()
    return torch.linalg.matrix_power(reach, nodes) > 0  # the ways from i to j in that many steps, some of which stay


def _prepare_verify(case, g):
    B, T, V, dtype = case["batch"], case["nodes"], case["vocab"], DTYPES[case["dtype"]]
    logits = _normal(g, B, T, V) * 2.5
    state = {"target": torch.softmax(logits, -1).to(dtype), "draft": None, "parents": None,
             "uniforms": torch.rand(B, T, generator=g, device="cuda")}
    drafted = logits + _normal(g, B, T, V) * 0.4  # a draft that is mostly right
    if case["shape"] == "chain":
        probs = torch.softmax(drafted[:, :-1], -1).to(dtype)
        if case["draft_probs"]:
            pick = torch.multinomial(probs.float().reshape(-1, V), 1, generator=g).view(B, T - 1)
            state["draft"] = probs
        else:
            pick = probs.argmax(-1)
    else:  # the draft's best tokens after the node that each one follows, the next best for the next sibling
        parent = _parents(g, B, T)
        order = ((parent[:, :, None] == parent[:, None, :]).tril(-1)).sum(-1)[:, 1:]  # how many siblings came before
        best = drafted.topk(min(T, V), -1).indices
        rows = torch.gather(best, 1, parent[:, 1:, None].expand(-1, -1, best.shape[-1]))
        pick = torch.gather(rows, 2, order[..., None])[..., 0]
        state["parents"] = parent
    state["tokens"] = torch.cat([torch.zeros(B, 1, dtype=torch.long, device="cuda"), pick], 1)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------


def run(state):
    return {"rope": _run_rope, "cache": _run_cache, "attention": _run_attention, "verify": _run_verify}[state["case"]["op"]](state)


def _heads(x, head_dim):
    return x.view(x.shape[0], x.shape[1], -1, head_dim).transpose(1, 2)


def _run_rope(state):
    case = state["case"]
    D, interleaved = case["head_dim"], case["interleaved"]
    if own:
        from accelerate_amd.ops import rotary_embedding

        q, k = _heads(state["q"], D), _heads(state["k"], D)
        if not case["backward"]:
            return rotary_embedding(q, k, state["cos"], state["sin"], positions=state["positions"], interleaved=interleaved)
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = rotary_embedding(q, k, state["cos"], state["sin"], positions=state["positions"], interleaved=interleaved)
        return (*out, *torch.autograd.grad(out, (q, k), (state["dq"], state["dk"])))
    cos, sin = state["cos"], state["sin"]
    if state["positions"] is None:
        cos, sin = cos[None, None, : case["seq"]], sin[None, None, : case["seq"]]
    else:
        cos, sin = cos[state["positions"]][:, None], sin[state["positions"]][:, None]
    q, k = _heads(state["q"], D), _heads(state["k"], D)
    out = [_plain_rotate(x, cos, sin, case["rotary_dim"], interleaved) for x in (q, k)]
    if case["backward"]:  # the rotation's transpose turns back
        out += [_plain_rotate(x, cos, -sin, case["rotary_dim"], interleaved) for x in (state["dq"], state["dk"])]
    return tuple(out)


def _plain_rotate(x, cos, sin, rotary_dim, interleaved):
    wide = x.float()
    turned, rest = wide[..., :rotary_dim], wide[..., rotary_dim:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., : rotary_dim // 2], turned[..., rotary_dim // 2 :]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _run_cache(state):
    case = state["case"]
    T, D = case["tokens"], case["head_dim"]
    k, v = _heads(state["k"], D), _heads(state["v"], D)
    if own:
        cache = state["cache"]
        cache.append(k, v)
        return cache.read(start=cache.lengths, length=T)
    slot = state["lengths"].long()[:, None] + torch.arange(T, device="cuda")  # [B, T]
    b = torch.arange(case["batch"], device="cuda")[:, None]
    out = []
    for name, x in (("k", k), ("v", v)):
        held, scales = state["held_" + name], state["scale_" + name]
        code, scale = _plain_quantise(x, case["kind"])
        held[b, :, slot] = code.transpose(1, 2)
        back = held[b, :, slot].transpose(1, 2)
        if case["kind"] != "same":
            scales[b, :, slot] = scale.transpose(1, 2)
            back = back.float() * scales[b, :, slot].transpose(1, 2)[..., None]
        out.append(back.to(x.dtype))
    return tuple(out)


def _plain_quantise(x, kind):
    if kind == "same":
        return x, None
    wide = x.float()
    most = wide.abs().amax(-1)
    if kind == "int8":  # the quotient in 64 bits: 32 would move values that lie next to a border
        scale = most / INT8_MAX
        code = torch.round(wide.double() / torch.where(scale > 0, scale, 1.0)[..., None].double())
        return code.to(torch.int8), scale
    mantissa, exponent = torch.frexp(most / FP8_MAX)  # the least power of two that is not less
    scale = torch.where(most > 0, torch.ldexp(torch.ones_like(most), exponent - (mantissa == 0.5).int()), 0.0)
    code = wide / torch.where(scale > 0, scale, 1.0)[..., None]  # exact, by a power of two
    return code.to(torch.float8_e4m3fn), scale


def _run_attention(state):
    case = state["case"]
    q = _heads(state["q"], case["head_dim"])
    if own:
        from accelerate_amd.ops import cache_attention

        return cache_attention(q, state["cache"], mask=state["mask"])
    B, Hq, T, D = q.shape
    H, L = case["kv_heads"], case["max_len"]
    k, v = state["k"].float(), state["v"].float()
    if case["kind"] != "same":
        k, v = k * state["scale_k"][..., None], v * state["scale_v"][..., None]
    scores = torch.matmul(q.float().reshape(B, H, -1, D), k.transpose(-1, -2)).view(B, Hq, T, L) / math.sqrt(D)
    seen = _seen(case, state["lengths"], state["mask"])
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p.view(B, H, -1, L), v).view(B, Hq, T, D).to(q.dtype)


def _seen(case, lengths, mask):
    """[B, T, L]: the slots that each new token sees: all before the new ones, and of those what the mask says."""
    T = case["tokens"]
    at = torch.arange(case["max_len"], device="cuda") - lengths.long()[:, None]  # [B, L], counted from the first new one
    i = torch.arange(T, device="cuda")
    if mask is None:
        return at[:, None] <= i[None, :, None]
    new = torch.gather(mask, 2, at.clamp(0, T - 1)[:, None].expand(-1, T, -1))
    return (at < 0)[:, None] | (((at >= 0) & (at < T))[:, None] & new)


def _run_verify(state):
    if own:
        from accelerate_amd.ops import verify_draft

        out = verify_draft(state["target"], state["tokens"], state["uniforms"], draft_probs=state["draft"],
                           parents=state["parents"])
        return out.tokens, out.counts, out.path
    target, tokens, u = state["target"], state["tokens"], state["uniforms"].double()
    B, T, V = target.shape
    at = torch.arange(T, device="cuda")
    parent = state["parents"]
    if parent is None:
        parent = (at - 1).expand(B, T)
    before = parent.clamp(min=0)
    b = torch.arange(B, device="cuda")[:, None]
    p = target[b, before, tokens].double()
    if state["draft"] is not None:
        q = torch.nn.functional.pad(state["draft"], (0, 0, 0, 1))[b, before, tokens].double()
        taken = u * q < p
    else:  # a draft that was certain: what its rejected siblings held is gone
        sibling = (parent[:, :, None] == parent[:, None, :]) & (at[:, None] > at)
        left = 1 - (sibling * p[:, None, :]).sum(-1)
        taken = u * left < p
        taken &= ~(sibling & taken[:, None, :]).any(-1)
    taken[:, 0] = True
    on_path = ~(_ancestors(parent) & ~taken[:, None, :]).any(-1)  # all that it follows were taken too
    counts = on_path.sum(-1) - 1
    order = torch.where(on_path, at, T + at).argsort(-1)
    valid = at <= counts[:, None]
    path = torch.where(valid, order, -1)
    last = torch.gather(order, 1, counts[:, None])[:, 0]
    b = b[:, 0]
    weight = target[b, last].double()
    if state["draft"] is not None:
        row = torch.nn.functional.pad(state["draft"], (0, 0, 0, 1))[b, last].double()  # nothing was drafted after the last
        weight = (weight - row).clamp(min=0)
    else:
        gone = (parent == last[:, None]) & (at > 0)
        weight = weight.scatter_reduce(1, tokens, torch.where(gone, 0.0, math.inf).double(), "amin")
    total = weight.cumsum(-1)
    final = (total <= u[:, :1] * total[:, -1:]).sum(-1)
    accepted = torch.nn.functional.pad(torch.gather(tokens, 1, order)[:, 1:], (0, 1), value=-1)
    out = torch.where(at < counts[:, None], accepted, torch.where(at == counts[:, None], final[:, None], -1))
    return out, counts, path


# ---- in 64 bits -----------------------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "cache": _exact_cache, "attention": _exact_attention, "verify": _exact_verify}[case["op"]](case, state)


def _exact_rope(case, state):
    """As products of complex numbers, the angles from the formulas."""
    R, D, scaling = case["rotary_dim"], case["head_dim"], SCALINGS[case["scaling"]]
    freq, factor = [], 1.0
    for i in range(R // 2):
        f = THETA ** (-2.0 * i / R)
        if scaling is None:
            pass
        elif scaling["rope_type"] == "linear":
            f /= scaling["factor"]
        elif scaling["rope_type"] == "llama3":
            wave, trained = 2 * math.pi / f, scaling["original_max_position_embeddings"]
            if wave > trained / scaling["low_freq_factor"]:
                f /= scaling["factor"]
            elif wave > trained / scaling["high_freq_factor"]:
                smooth = (trained / wave - scaling["low_freq_factor"]) / (scaling["high_freq_factor"] - scaling["low_freq_factor"])
                f = (1 - smooth) * f / scaling["factor"] + smooth * f
        else:
            trained, s = scaling["original_max_position_embeddings"], scaling["factor"]
            ends = [R * math.log(trained / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (scaling["beta_fast"], scaling["beta_slow"])]
            low, high = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), R - 1)
            slow = min(max((i - low) / (high - low if high > low else 0.001), 0.0), 1.0)
            f = f / s * slow + f * (1 - slow)
            factor = 0.1 * math.log(s) + 1.0
        freq.append(f)
    freq = torch.tensor(freq, device="cuda", dtype=torch.float64)
    positions = state["positions"] if state["positions"] is not None else torch.arange(case["seq"], device="cuda")[None]
    turn = torch.polar(torch.full((), factor, device="cuda", dtype=torch.float64), positions.double()[..., None] * freq)[:, None]
    inputs = [_heads(state["q"], D), _heads(state["k"], D)] + ([state["dq"], state["dk"]] if case["backward"] else [])
    out = []
    for n, x in enumerate(inputs):
        x = x.double().contiguous()
        pairs = x[..., :R].unflatten(-1, (R // 2, 2)) if case["interleaved"] else x[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * (turn if n < 2 else turn.conj()))
        x[..., :R] = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        out.append(x)
    return tuple(out)


def _exact_cache(case, state):
    out = []
    for name in ("k", "v"):
        x = _heads(state[name], case["head_dim"]).double().contiguous()
        if case["kind"] == "int8":
            scale = (x.abs().amax(-1, keepdim=True) / 127.0).float().double()  # the scale is held in 32 bits
            x = torch.where(scale > 0, torch.round(x / scale) * scale, 0.0)
        elif case["kind"] == "fp8":  # steps of an eighth of the value's power of two, and no finer than 2^-9
            most = x.abs().amax(-1, keepdim=True)
            fraction, exponent = torch.frexp(most / 448.0)
            scale = torch.exp2(torch.where(fraction == 0.5, exponent - 1, exponent).double())
            y = x / torch.where(most > 0, scale, 1.0)
            step = torch.exp2(torch.frexp(y.abs().clamp(min=2.0**-6)).exponent.double() - 4)
            x = torch.round(y / step) * step * scale
        out.append(x)
    return tuple(out)


def _exact_attention(case, state):
    """Sequence by sequence, over what is seen alone."""
    D, T, rep = case["head_dim"], case["tokens"], case["q_heads"] // case["kv_heads"]
    q = _heads(state["q"], D).double()
    result = torch.empty_like(q)
    for b, n in enumerate(_lengths(case)):
        k, v = (state[name][b, :, : n + T].double() for name in ("k", "v"))
        if case["kind"] != "same":
            k, v = k * state["scale_k"][b, :, : n + T, None].double(), v * state["scale_v"][b, :, : n + T, None].double()
        seen = torch.ones(T, n + T, device="cuda", dtype=torch.bool)
        seen[:, n:] = torch.ones(T, T, device="cuda", dtype=torch.bool).tril() if state["mask"] is None else state["mask"][b]
        s = torch.einsum("hrtd,hld->hrtl", q[b].unflatten(0, (-1, rep)), k) * D**-0.5
        s = torch.where(seen, s, -math.inf)
        s = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
        result[b] = torch.einsum("hrtl,hld->hrtd", s, v).flatten(0, 1)
    return result


def _exact_verify(case, state):
    """The walk, step by step, on the host."""
    B, T, V = state["target"].shape
    tokens, u = state["tokens"].tolist(), state["uniforms"].double().tolist()
    parents = state["parents"].tolist() if state["parents"] is not None else [list(range(-1, T - 1))] * B
    out = np.full((B, T), -1), np.zeros(B, dtype=np.int64), np.full((B, T), -1)
    for b in range(B):
        node, path, said, mass, gone, refused = 0, [0], [], 1.0, [], False
        row = state["target"][b, 0].double().cpu().numpy()
        for i in range(1, T):
            if parents[b][i] != node:
                continue
            x = tokens[b][i]
            if state["draft"] is not None:
                if refused:
                    break
                took = u[b][i] * float(state["draft"][b, node, x].double()) < row[x]
                refused = not took
            else:
                took = u[b][i] * mass < row[x] and x not in gone
            if took:
                node, mass, gone = i, 1.0, []
                row = state["target"][b, i].double().cpu().numpy()
                path.append(i)
                said.append(x)
            elif x not in gone:
                mass -= row[x]
                gone.append(x)
        if refused:
            row = np.maximum(row - state["draft"][b, node].double().cpu().numpy(), 0.0)
        elif state["draft"] is None:
            row = row.copy()
            row[gone] = 0.0
        total = np.cumsum(row)
        said.append(int(np.searchsorted(total, u[b][0] * total[-1], side="right")))
        out[0][b, : len(said)], out[1][b], out[2][b, : len(path)] = said, len(path) - 1, path
    return tuple(torch.from_numpy(x) for x in out)
