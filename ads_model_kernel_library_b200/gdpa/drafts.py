"""Drafted tokens: a cheaper model, or a look into the text, proposes several at once, the target reads them in one step of the paged cache
(:meth:`.paged.PagedKVCache.step` with more than one token a request), and its probabilities decide how many of them stay."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops, paged

__all__ = ["verify_draft_tokens"]


def verify_draft_tokens(
    target_probs: torch.Tensor,
    draft_probs: Optional[torch.Tensor],
    draft_tokens: torch.Tensor,
    query_offset: torch.Tensor,
    draft_offset: torch.Tensor,
    accept_uniform: torch.Tensor,
    sample_uniform: torch.Tensor,
    max_drafts: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accept drafts and draw the next token so that what comes out is distributed as the target's own tokens.

    Request ``b`` has the drafts ``draft_tokens[draft_offset[b]:draft_offset[b + 1]]``, ``n`` of them (at most ``max_drafts``), and the rows
    ``query_offset[b]:query_offset[b + 1]`` of ``target_probs`` ``[rows, vocabulary]`` (fp32 or bf16): row ``j`` is the target's distribution of
    draft ``j``, row ``n`` that of the token after them, so a step has one row more than drafts (its first query is the last token that was known).
    Without a row more, that many drafts are not looked at, nor are those past ``max_drafts``: they count as neither accepted nor refused, so a caller that
    has stored more than ``max_drafts`` takes the others out of the cache itself.  A request without rows takes no part.  ``draft_probs`` ``[drafts, vocabulary]`` are the
    distributions that the drafts were drawn from, ``None`` for drafts that were not drawn at all.

    Draft ``j`` is accepted if ``accept_uniform[j] * draft_probs[j, token] < target_probs[j, token]`` and all before it are (``None``: the factor is
    1; a token outside the vocabulary never is).  Then one more is drawn: after a refused draft from ``max(target - draft, 0)`` (``None``:
    the target without that token; where nothing is left, the target), after the last from its row of the target: the first token at which the partial
    sum exceeds ``sample_uniform[b]`` times the total.  Probabilities need not add up to 1; those that are not positive finite numbers count as 0.
    Sums are in 64 bits.

    Returns ``(tokens, accepted, refused)``: ``[B, max_drafts + 1]`` of the drafts' type, the accepted drafts, the drawn token (-1 if the row has no
    probability at all) and -1 behind them; int32 ``[B]`` each, the numbers of accepted and refused drafts.  ``refused`` is what
    :func:`~.paged.drop_cached_tokens` takes out of the cache.  Nothing synchronises with the host; there are no gradients.
    """
    if ops._validate_offsets and not torch.compiler.is_compiling():
        ops._check_offsets("query_offset", query_offset, target_probs.shape[0], False)
        ops._check_offsets("draft_offset", draft_offset, draft_tokens.shape[0], False)
    return (paged._operators or paged._load()).verify(target_probs, draft_probs, draft_tokens, query_offset, draft_offset, accept_uniform, sample_uniform, max_drafts)
