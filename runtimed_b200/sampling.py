"""Sampling from logits: temperature, top-k, top-p and min-p with given random numbers
(``rtd_sample``), the counterpart of ``rtd_argmax`` for generation that is not greedy
(crates/runtimed-model/src/decode/sample.rs:11-18 has the greedy pick alone)."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .errors import ConfigError, ShapeError
from .weights import _DT, Context, _raise

MAX_VOCAB = 1 << 19

_stream = torch._C._cuda_getCurrentRawStream


def _per_row(name: str, t: Optional[torch.Tensor], dtype: torch.dtype, rows: int, dev: torch.device):
    if t is None:
        return None
    if t.dtype != dtype or t.device != dev or not t.is_contiguous():
        raise ConfigError(f"{name}: a contiguous {dtype} tensor on {dev} is wanted, got {t.dtype} on {t.device}")
    if tuple(t.shape) != (rows,):
        raise ShapeError(name, [rows], list(t.shape))
    return t.data_ptr()


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 ids [T], one drawn from each row of logits [T, V] by the random numbers u [T]
    (f32 in [0, 1)).  The filters are tensors [T] on the same device (f32; top_k int32) or
    None; they apply in the order top-k, top-p over what is left, min-p, all at the row's
    temperature.  A temperature of 0 or a top_k of 1 takes the largest logit, as argmax."""
    if logits.dim() != 2:
        raise ShapeError("logits", [-1, -1], list(logits.shape))
    dev = logits.device
    if dev.type != "cuda" or logits.dtype not in _DT:
        raise ConfigError(f"logits: {logits.dtype} on {dev} (f32, f16 or bf16 on a CUDA device)")
    rows, vocab = logits.shape
    ld = logits.stride(0) if rows > 1 else vocab
    if logits.stride(1) != 1 and vocab > 1 or ld < vocab:
        raise ConfigError(f"logits: strides {logits.stride()} (rows must be dense)")
    if not 0 < vocab <= MAX_VOCAB:
        raise ConfigError(f"logits: {vocab} entries a row (1 to {MAX_VOCAB})")
    if out is None:
        out = torch.empty((rows,), dtype=torch.int32, device=dev)
    f32 = torch.float32
    ctx = Context.for_device(dev)
    st = _lib.lib().rtd_sample(ctx.handle, logits.data_ptr(), _DT[logits.dtype], ld, rows, vocab,
                               _per_row("temperature", temperature, f32, rows, dev),
                               _per_row("top_k", top_k, torch.int32, rows, dev),
                               _per_row("top_p", top_p, f32, rows, dev), _per_row("min_p", min_p, f32, rows, dev),
                               _per_row("u", u, f32, rows, dev), _per_row("out", out, torch.int32, rows, dev),
                               _stream(dev.index))
    if st:
        _raise(st, ctx.handle)
    return out
