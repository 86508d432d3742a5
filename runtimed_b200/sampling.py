"""Sampling from logits: temperature, top-k, top-p and min-p with given random numbers
(``rtd_sample``), the counterpart of ``rtd_argmax`` for generation that is not greedy
(crates/runtimed-model/src/decode/sample.rs:11-18 has the greedy pick alone)."""
from __future__ import annotations

from typing import Optional

import torch

from ._torch import binding

MAX_VOCAB = 1 << 19


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 ids [T], one drawn from each row of logits [T, V] (V at most MAX_VOCAB) by the
    random numbers u [T] (f32 in [0, 1)).  The filters are tensors [T] on the same device
    (f32; top_k int32) or None; they apply in the order top-k, top-p over what is left,
    min-p, all at the row's temperature.  A temperature of 0 or a top_k of 1 takes the
    largest logit, as argmax."""
    return binding.sample(logits, u, temperature, top_k, top_p, min_p, out)
