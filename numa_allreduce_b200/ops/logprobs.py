"""Log-probabilities of given tokens, with entropy and top alternatives."""

from __future__ import annotations

from typing import NamedTuple, Sequence

import torch
import torch.distributed as dist

from . import _ext
from .errors import after_launch


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` gives for each row of logits (fp32, token ids int64).

    All of it lies in one allocation, which lives as long as any part: clone
    what is to be kept alone.
    """

    logprob: torch.Tensor       # [rows]: of the given token, -inf if it is not in this part of the vocabulary
    entropy: torch.Tensor       # [rows]: of the distribution, in nats
    lse: torch.Tensor           # [rows]: log of the sum of exp(logits)
    top_logprobs: torch.Tensor  # [rows, top_k], falling
    top_tokens: torch.Tensor    # [rows, top_k]
    top_logits: torch.Tensor    # [rows, top_k]: the logits themselves, by which shards are merged


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0, vocab_start: int = 0) -> TokenLogprobs:
    """Log-softmax of ``logits[rows, vocabulary]`` at ``tokens``, and its entropy and ``top_k`` largest entries.

    One launch and one pass over the logits (fp32, fp16 or bf16; rows may be
    further apart than the vocabulary), sums in fp32. The few parts of a row
    that can hold its largest entries are read again for them, and a row whose
    maximum is above 2^24 or below -2^23 (fp16: below -50000) is summed again.
    ``top_k`` is at most 32;
    equal logits rank by the lowest token id. Entries of -inf (masked tokens)
    have probability 0. A row that holds NaN or +inf, or only -inf, gives NaN
    (``lse`` of the last is -inf); NaN ranks as -inf.

    ``logits`` may be one shard of the vocabulary, with column 0 the token
    ``vocab_start``: the result is that of the shard alone, and
    :func:`join_token_logprobs` makes the whole vocabulary's from all shards.
    For inference: logits that require a gradient, or carry a forward-mode
    tangent, are refused, and so are tensors that are not plain memory (fake,
    batched or wrapped ones).
    """
    native = _ext.native()
    r = TokenLogprobs._make(native.token_logprobs(logits, tokens, top_k, vocab_start))
    if native.check_requested():
        after_launch(logits.device)
    return r


def join_token_logprobs(shards: Sequence[TokenLogprobs]) -> TokenLogprobs:
    """The results of every vocabulary shard (in order of the shards, for the
    same tokens and top_k) as those of the whole vocabulary."""
    if not shards:
        raise ValueError("join_token_logprobs needs at least one shard")
    part = torch.stack([s.lse for s in shards])  # [shards, rows]
    lse = part.logsumexp(0)
    shift = part - lse  # log of a shard's probability
    weight = shift.exp()
    # a shard whose tokens are all masked has no distribution of its own (NaN): it adds nothing
    masked = (part == -torch.inf) & (lse != -torch.inf)
    entropy = torch.where(masked, 0, weight * (torch.stack([s.entropy for s in shards]) - shift)).sum(0)
    logprob = torch.where(masked, -torch.inf, torch.stack([s.logprob for s in shards]) + shift).amax(0)
    top = torch.cat([torch.where(m[:, None], -torch.inf, s.top_logprobs + d[:, None])
                     for s, d, m in zip(shards, shift, masked)], -1)
    ids = torch.cat([s.top_tokens for s in shards], -1)
    raw = torch.cat([s.top_logits for s in shards], -1)
    k = shards[0].top_logprobs.shape[1]
    # by the logits, which are exact (NaN as -inf); stable: equal ones keep the order of the token ids
    order = raw.nan_to_num(nan=-torch.inf, posinf=torch.inf, neginf=-torch.inf)
    order = order.argsort(dim=-1, descending=True, stable=True)[:, :k]
    return TokenLogprobs(logprob, entropy, lse, top.gather(-1, order), ids.gather(-1, order), raw.gather(-1, order))


def gather_token_logprobs(shard: TokenLogprobs, group=None) -> TokenLogprobs:
    """:func:`join_token_logprobs` over the ranks of a process group, each with
    its shard of the vocabulary in rank order: one all-gather of
    ``12 + 16 top_k`` bytes per row (for fp32). Every rank gets the whole
    vocabulary's result."""
    rows, k = shard.top_logprobs.shape
    if rows == 0:
        return shard
    dtype = shard.lse.dtype
    # as whole numbers of the floats' width: an id keeps its bits (in one or two of them), and so does a NaN
    word = torch.int64 if dtype == torch.float64 else torch.int32
    fields = (torch.stack([shard.logprob, shard.entropy, shard.lse], -1), shard.top_logprobs, shard.top_logits,
              shard.top_tokens)
    mine = torch.cat([t.contiguous().view(word) for t in fields], -1)
    world = dist.get_world_size(group)
    parts = torch.empty(world * rows, mine.shape[1], dtype=word, device=mine.device)
    dist.all_gather_into_tensor(parts, mine, group=group)

    def result(p: torch.Tensor) -> TokenLogprobs:
        logprob, entropy, lse = p[:, :3].contiguous().view(dtype).unbind(-1)
        top, raw = (p[:, 3 + i * k:3 + (i + 1) * k].contiguous().view(dtype) for i in range(2))
        ids = torch.empty(rows, k, dtype=torch.int64, device=p.device)
        ids.view(word).copy_(p[:, 3 + 2 * k:])
        return TokenLogprobs(logprob, entropy, lse, top, ids, raw)

    return join_token_logprobs([result(p) for p in parts.view(world, rows, mine.shape[1])])
