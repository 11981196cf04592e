"""Rotary positions: the frequencies that a head's columns turn with, and the rotation.

    frequencies, magnitude = rotary.frequencies(64, device="cuda")        # once
    x = rotary.rotary(x, positions, frequencies, magnitude)               # queries and keys, in every layer

Of a head's columns the first 2 * len(frequencies) turn, pair i of a token at position p by the angle p * frequencies[i]; pairs are
columns i and i + len(frequencies), or 2 i and 2 i + 1 (interleaved).  Both run on one product's queries and keys at once, as
qkv[:, :heads].  KvCache.append turns the keys that it stores by itself.

The rotation is a TorchScript operator as well, torch.ops.functs.rotary.  GPU tensors only.
"""
import math
from typing import Tuple

import torch
from torch import Tensor

from . import _C  # noqa: F401  (registers the operators)
from . import _lib
from ._lib import C

STRETCHES = ("linear", "base", "parts", "bands")


def frequencies(columns: int, base: float = 10000.0, stretch: float = 1.0, how: str = "linear", length: int = 4096, fast: float = 32.0, slow: float = 1.0,
                device="cuda") -> Tuple[Tensor, float]:
    """float64 [columns / 2] frequencies base ** (-2 i / columns), and the magnitude to turn with.  For contexts `stretch` times as long as
    the `length` tokens that a model has seen:
      linear  all divided by `stretch`
      base    the base times stretch ** (columns / (columns - 2)): the slowest one is divided by `stretch`, the fastest stays
      parts   those of more than `fast` turns in `length` tokens stay, those of fewer than `slow` are divided, in between a straight line over i;
              the magnitude is 0.1 ln(stretch) + 1
      bands   the same with the straight line over the number of turns; the magnitude stays 1 (fast 4, slow 1 are usual)"""
    if columns < 2 or columns % 2 != 0:
        raise _lib.FxError(C["FX_E_INVALID"], "columns turn in pairs: an even number of them, got %s" % columns)
    if how not in STRETCHES:
        raise _lib.FxError(C["FX_E_INVALID"], "how must be one of %s, got %r" % (STRETCHES, how))
    if not (math.isfinite(base) and base > 1.0 and math.isfinite(stretch) and stretch >= 1.0 and length >= 1 and 0.0 < slow < fast):
        raise _lib.FxError(C["FX_E_INVALID"], "base is more than 1, stretch and length 1 at least, and slow positive and less than fast")
    if how == "base" and stretch > 1.0:
        if columns == 2:
            raise _lib.FxError(C["FX_E_INVALID"], "one pair has no slowest and fastest frequency: how='base' takes 4 columns at least")
        base = base * stretch ** (columns / (columns - 2))
    i = torch.arange(columns // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / columns)
    magnitude = 1.0
    if stretch > 1.0 and how == "linear":
        f = f / stretch
    elif stretch > 1.0 and how == "parts":
        # the (fractional) i at which a frequency makes so many turns
        at = lambda turns: columns * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), columns - 1)
        divided = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        f = f * (1.0 - divided) + f / stretch * divided
        magnitude = 0.1 * math.log(stretch) + 1.0
    elif stretch > 1.0 and how == "bands":
        whole = ((length * f / (2.0 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f * whole + f / stretch * (1.0 - whole)
    return f.to(device), magnitude


def rotary(x: Tensor, positions: Tensor, frequencies: Tensor, magnitude: float = 1.0, interleaved: bool = False) -> Tensor:
    """x [tokens, heads, depth] or [batch, tokens, heads, depth] (float32, float16 or bfloat16, any strides) turned; positions int32 or int64
    [tokens], or [batch, tokens]; frequencies float64 or float32.  Has a backward pass (for x), which may be differentiated again.
    Forward and backward passes may be captured into a graph.  Refused are a captured backward pass that comes to a tensor which is in a living graph of the default
    stream, and a captured call on a leaf that requires a gradient and is in a living graph of another stream: drop that graph's results before."""
    return torch.ops.functs.rotary(x, positions, frequencies, magnitude, interleaved)
