"""A beam search's selection over beams and vocabulary.

    chosen = beam.select(logits, scores, ended=ended, end_word=eos)      # logits [requests, beams, words], scores [requests, beams]
    chosen.scores, chosen.beams, chosen.words                            # [requests, count], the best first

Log-probabilities, sums with the beams' scores and the selection in one or two launches that read the logits once.  KvCache.fork moves the pages of a
cache to the beams that go on.  The selection is a TorchScript operator as well, torch.ops.functs.beam_select.  GPU tensors only, and no backward pass.
"""
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _C  # noqa: F401  (registers the operators)
from ._lib import C

MAX_BEAMS, MAX_COUNT, MAX_WORDS = C["FX_BEAM_MAX_BEAMS"], C["FX_BEAM_MAX_COUNT"], C["FX_BEAM_MAX_WORDS"]


class Chosen(NamedTuple):
    """scores float32, beams int32 (which of its request's beams each continues; -1: none), words int64 (-1: none), all [requests, count]."""
    scores: Tensor
    beams: Tensor
    words: Tensor


def select(logits: Tensor, scores: Tensor, count: int = 0, ended: Optional[Tensor] = None, end_word: int = -1) -> Chosen:
    """The `count` (0: as many as beams) best of scores[b, k] + log_softmax(logits[b, k])[w] of each request b, best first; equal ones in the order of beams,
    then of words.  logits float32, float16 or bfloat16 [requests, beams, words], scores float32 [requests, beams].  A masked word's logit is -infinity
    (a finite mask gives such words their small probability, and takes a millisecond where fewer words than `count` are left of a large vocabulary); a beam
    that does not exist yet (all but one behind a prompt) has the score -infinity.  Beams with ended[b, k] (bool) keep their score and continue with
    `end_word` alone.  Places for which there is no candidate: -infinity, -1, -1.  include/fxhip.h has every rule."""
    return Chosen(*torch.ops.functs.beam_select(logits, scores, count, ended, end_word))


def first_scores(requests: int, beams: int, device="cuda") -> Tensor:
    """Scores to start with: the first beam of each request is there, the others are not."""
    scores = torch.full((requests, beams), float("-inf"), device=device)
    scores[:, 0] = 0.0
    return scores
