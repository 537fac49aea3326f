"""Verification of drafted tokens against a target's probabilities, from given random numbers.

Node 0 of a sequence is the last token that stands, a node i > 0 is a drafted token that follows its parent, and
``target_probs[:, i]`` is the target's distribution of the token after node i. The tokens that come out are distributed
as if the target had been sampled token by token, whatever was drafted.

On a GPU the kernels are those of ``ops/csrc/verify_kernels.hip``; on a CPU the walk runs on the host.
"""

from typing import NamedTuple, Optional

import torch

from . import _load_extension

MAX_NODES = 1024  # of a draft, root included


class DraftVerdict(NamedTuple):
    """What of a draft stands. ``counts`` [B]: drafted tokens that were taken. ``tokens`` [B, T]: these, then the
    target's own next token, then -1. ``path`` [B, T]: the nodes that were taken, with the root, then -1. All int64."""

    tokens: torch.Tensor
    counts: torch.Tensor
    path: torch.Tensor


def verify_draft(
    target_probs: torch.Tensor,
    tokens: torch.Tensor,
    uniforms: torch.Tensor,
    draft_probs: Optional[torch.Tensor] = None,
    parents: Optional[torch.Tensor] = None,
) -> DraftVerdict:
    """Walk from the root over drafted tokens that are taken, then draw the token that follows.

    ``target_probs`` [B, T, V] (fp32, bf16 or fp16), ``tokens`` int64 [B, T] (node 0's is not read), ``uniforms`` fp32 or
    fp64 [B, T] in [0, 1): number i > 0 tests node i, number 0 draws the last token. With a parent's target row p and
    u = uniforms[b, i], a child with token x is

    - of a draft that was drawn from ``draft_probs`` [B, T - 1, V] (row i - 1 for node i; a chain only): taken iff
      u q(x) < p(x); after a refusal the last token is drawn from max(p - q, 0);
    - of a draft without probabilities, a chain or, with ``parents`` int64 [T] or [B, T], a tree: taken iff u r < p(x),
      where r is 1 less the p of its siblings that were refused before it (in the order of the nodes); if none is
      taken the last token is drawn from p without them.

    A node whose token is outside the vocabulary, or whose parent is not a node before it, is no draft: a chain ends
    before it, a tree goes without it, so shorter drafts are padded with token or parent -1. The last token is the first
    whose cumulative weight exceeds uniforms[b, 0] times the sum. If no weight is left it is drawn from p as it is; it is
    0 if that has none either. NaN counts as no weight. Comparisons and sums are in 64 bits.
    """
    if target_probs.is_cuda:
        ext = _load_extension(required=True)
        return DraftVerdict(*ext.verify_draft(target_probs, tokens, uniforms, draft_probs, parents))

    def need(ok, message):
        if not ok:
            raise RuntimeError(f"verify_draft: {message}")

    need(target_probs.dim() == 3 and target_probs.is_floating_point(), "target_probs must be a [B, T, V] tensor")
    B, T, V = target_probs.shape
    need(1 <= T <= MAX_NODES, f"1 to {MAX_NODES} nodes, got {T}")
    need(V >= 1, "an empty vocabulary")
    need(
        draft_probs is None or parents is None,
        "draft_probs are for chains; the tokens of a tree are taken as certain drafts",
    )
    need(tokens.dtype == torch.int64 and tokens.shape == (B, T), "tokens must be int64 [B, T]")
    need(
        uniforms.dtype in (torch.float32, torch.float64) and uniforms.shape == (B, T),
        "uniforms must be float32 or float64 [B, T]",
    )
    need(
        draft_probs is None or (draft_probs.dtype == target_probs.dtype and draft_probs.shape == (B, T - 1, V)),
        "draft_probs must be [B, T - 1, V] of target_probs' type",
    )
    need(
        parents is None
        or (parents.dtype == torch.int64 and (parents.shape == (T,) or parents.shape in ((B, T), (1, T)))),
        "parents must be int64 [T] or [B, T]",
    )
    follows = torch.arange(-1, T - 1) if parents is None else parents
    follows, ids, u = follows.expand(B, T).tolist(), tokens.tolist(), uniforms.double().tolist()
    out, counts, path = torch.full((B, T), -1), torch.zeros(B, dtype=torch.int64), torch.full((B, T), -1)
    for b in range(B):
        node, taken, refused, left = 0, [0], [], 1.0
        less = None
        for i in range(1, T):
            x, parent = ids[b][i], follows[b][i]
            if not (0 <= x < V and 0 <= parent < i):
                if parents is None:
                    break
                continue
            if parent != node or x in refused:
                continue
            p = float(target_probs[b, node, x].double())
            if draft_probs is not None:
                if u[b][i] * float(draft_probs[b, node, x].double()) < p:
                    node = i
                    taken.append(i)
                    continue
                less = draft_probs[b, node].double()
                break
            if u[b][i] * left < p:
                node, refused, left = i, [], 1.0
                taken.append(i)
            else:
                left -= p if p > 0 else 0.0  # NaN too
                refused.append(x)
        row = target_probs[b, node].double()
        row = torch.where(row > 0, row, 0.0)
        weight = row.clone()
        if less is not None:
            weight = target_probs[b, node].double() - less
            weight = torch.where(weight > 0, weight, 0.0)
        weight[refused] = 0.0
        if not (weight > 0).any():
            weight = row
        total = weight.cumsum(0)
        passed = (total > max(u[b][0], 0.0) * total[-1]).nonzero()
        some = weight.nonzero()
        last = int(passed[0]) if len(passed) else int(some[-1]) if len(some) else 0
        n = len(taken) - 1
        out[b, : n + 1] = torch.tensor([ids[b][i] for i in taken[1:]] + [last])
        path[b, : n + 1] = torch.tensor(taken)
        counts[b] = n
    return DraftVerdict(out, counts, path)
