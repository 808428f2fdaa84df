"""The end of a decode step: one token per row of logits, on the GPU (zs_sample), so
that a step from request lengths to tokens can be captured in a CUDA graph."""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import paged


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
           top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
           min_p: Union[float, torch.Tensor] = 0.0, out: Optional[torch.Tensor] = None,
           err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Tokens int64 [B] for logits [B, V] (bf16, fp16 or float32, V up to 2**20) and random
    numbers u float32 [B] in [0, 1).

    With w_i = exp((x_i - max x) / temperature), and the tokens in the order of x, largest
    first and equal ones by index: the first top_k are kept (0: all), of these the shortest
    beginning whose weights reach top_p of theirs, of these the ones with w_i >= min_p; the
    first token in any case. The result is the first token, by index, at which the running
    sum of the kept weights passes u times their sum. It does not depend on the batch or on
    an order of sums. temperature 0 takes the first of the largest.

    A setting is a number, or a tensor with one for each row (float32; top_k: int32). A
    number is taken in 64 bits, so a top_p of 0.95 may end a row's kept tokens one token from
    where the float32 nearest to 0.95 does. A number outside its range is refused; a tensor's
    counts as the nearest end (a top_k below 0 as 0), NaN as off (temperature: as 0), u
    outside its own likewise, and an infinite temperature makes all weights 1. A logit of
    -inf is never chosen. A row with a NaN, or of -inf alone, gives -1 and sets bit
    8 in err (int32 [1])."""
    return (paged._native or paged._load()).sample(logits, u, temperature, top_k, top_p, min_p, out, err)
