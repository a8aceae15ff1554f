"""Beam search on the device: the selection over beams and vocabulary, and the reordering of the states that
follow the beams (reference counterpart: the greedy / sampling step of examples/deepseek_v32/inference/generate.py).

Neither synchronises with the host: a whole step, model included, can be captured into a graph."""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from tilelang import _native


def beam_select(logits: torch.Tensor, scores: torch.Tensor, take: Optional[int] = None,
                finished: Optional[torch.Tensor] = None,
                eos_id: int = -1) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``take`` best continuations of every sequence's beams (default: as many as beams, at most 64).

    logits [batch, beams, vocab] or [batch * beams, vocab] (fp32, bf16, fp16; at most 64 beams and 2^20 tokens),
    scores float32 [batch, beams] (the beams' sums of log probabilities; -inf for a beam that is not in use).  The
    value of token t after beam k is

        scores[k] + logits[k, t] - logsumexp(logits[k])

    in float64 but for the logsumexp, which float32 exponentials and sums give on the device (off by less than
    2^-19), and the largest come first, ties by the lowest ``k * vocab + t``. One beam's tokens are always in the
    order of their logits; between two beams, values that are closer than that may come in either order. A beam of
    ``finished`` [batch, beams] (bool) has one continuation, ``eos_id``, with its score as it is. Not-a-number
    values count as -inf, so a beam whose logits hold not-a-numbers or +inf, or whose score is not finite, comes
    last.

    Returns (scores float32, parents int64, tokens int64), each [batch, take]."""
    return _native.ops().beam_select(logits, scores, scores.shape[-1] if take is None else take, finished, eos_id)


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor, length: Optional[int] = None) -> None:
    """``state[b, k] <- state[b, parents[b, k]]`` in place for every state, without a copy of any.

    Each state is [batch * beams, ...] of any type; parents int64 [batch, beams] within a sequence (a parent outside
    0 .. beams - 1 leaves its beam as it is; at most 32 beams).  ``length``: only the first ``length`` entries of
    the states' second dimension move (the filled part of a cache).  What moves of a row must be contiguous and at
    most 2^36 - 1024 bytes, and no two states may share memory."""
    _native.ops().reorder_states(states, parents, length)
