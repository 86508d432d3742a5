"""The paged KV cache held in 4 bits: device-side block tables, the quantising append,
attention over the pages and a reader.

Torch-level entry points of ``rtd_kv_plan``, ``rtd_rope_kv4_append``, ``rtd_attention_kv4``
and ``rtd_kv4_read`` (``include/rtd.h`` states the format and the rules).  Each runs on the
current stream of its tensors' device, allocates nothing but the outputs it returns, and
may be captured in a CUDA graph.  ``BlockTables`` keeps the state that ``plan`` works on.

What only the device can see (a block id outside the pool, a length beyond its bound, an
exhausted pool) is reported by ``Context.check_device_status``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import numpy as np
import torch

from . import _lib
from .errors import ConfigError, ShapeError
from .weights import _DT, Context, _raise

BLOCK = 16   # tokens of a page
GROUP = 32   # dims that share a step and a minimum
HEAD_DIMS = (32, 64, 96, 128)
MAX_SEQS = 8192

_stream = torch._C._cuda_getCurrentRawStream


def page_bytes(head_dim: int) -> int:
    """Bytes of one page: 16 tokens of one kv head, K and V."""
    if head_dim not in HEAD_DIMS:
        raise ConfigError(f"4-bit KV cache: head_dim {head_dim} (32, 64, 96 or 128)")
    return 20 * head_dim


def alloc_pages(num_blocks: int, n_kv: int, head_dim: int, device="cuda:0") -> torch.Tensor:
    """An empty pool: uint8 [num_blocks, n_kv, page_bytes(head_dim)]."""
    return torch.zeros((int(num_blocks), int(n_kv), page_bytes(head_dim)), dtype=torch.uint8, device=device)


def rope_frequencies(rot_dim: int, theta: float, device="cuda:0") -> torch.Tensor:
    """theta^(-2i / rot_dim), f64 [rot_dim / 2]: ``append``'s inv_freq for plain NeoX rope."""
    i = np.arange(rot_dim // 2, dtype=np.float64)
    return torch.from_numpy(float(theta) ** (-2.0 * i / max(1, rot_dim))).to(device)


def _ints(name: str, t: torch.Tensor, dev: torch.device, *shape) -> int:
    """The address of a dense int32 tensor of `shape` on `dev`."""
    if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
        raise ConfigError(f"{name}: a contiguous int32 tensor on {dev} is wanted, got {t.dtype} on {t.device}")
    if tuple(t.shape) != shape:
        raise ShapeError(name, list(shape), list(t.shape))
    return t.data_ptr()


def _pool(pages: torch.Tensor, head_dim: int) -> Tuple[int, int]:
    """(blocks, kv heads) of a pool of pages."""
    if pages.dtype != torch.uint8 or pages.dim() != 3 or not pages.is_contiguous() or not pages.is_cuda:
        raise ConfigError("pages: a contiguous uint8 CUDA tensor [blocks, n_kv, page bytes] is wanted")
    if pages.shape[2] != page_bytes(head_dim):
        raise ShapeError("pages", [-1, -1, page_bytes(head_dim)], list(pages.shape))
    return pages.shape[0], pages.shape[1]


def _heads(name: str, x: torch.Tensor, dev: torch.device, head_dim: int) -> int:
    """Elements between the tokens of x [T, heads, head_dim], whose heads lie side by side."""
    if x.dim() != 3 or x.shape[2] != head_dim:
        raise ShapeError(name, [-1, -1, head_dim], list(x.shape))
    if x.device != dev:
        raise ConfigError(f"{name}: on {x.device}, the pages on {dev}")
    if x.dtype not in _DT:
        raise ConfigError(f"{name}: {x.dtype} (f32, f16 or bf16)")
    t, h, _ = x.shape
    st, sh, sd = x.stride()
    if sd != 1 or (h > 1 and sh != head_dim) or (t > 1 and st < h * head_dim):
        raise ConfigError(f"{name}: strides {x.stride()} (a token's heads must lie side by side, tokens apart)")
    return st if t > 1 else h * head_dim


def plan(want: torch.Tensor, length: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
         free_count: torch.Tensor, max_tokens: Optional[int] = None, out=None):
    """Bring every sequence from ``length`` to ``want`` tokens: blocks move between ``table``
    [S, max_blocks] and the stack ``free_list`` / ``free_count``, all updated in place.

    With ``max_tokens`` (or ``out``, four buffers to reuse) the new tokens are listed:
    (q_start [S + 1], tok_seq, tok_pos, tok_slot [max_tokens]), -1 behind the last token."""
    dev = table.device
    if not table.is_cuda:
        raise ConfigError(f"table: on {dev}, a CUDA device is wanted")
    if table.dim() != 2:
        raise ShapeError("table", [-1, -1], list(table.shape))
    s, most = table.shape
    if out is None and max_tokens is not None:
        n = int(max_tokens)
        out = (torch.empty((s + 1,), dtype=torch.int32, device=dev),
               *torch.empty((3, n), dtype=torch.int32, device=dev).unbind(0))
    n, lists = 0, (None, None, None, None)
    if out is not None:
        n = out[1].shape[0]
        lists = (_ints("q_start", out[0], dev, s + 1), _ints("tok_seq", out[1], dev, n),
                 _ints("tok_pos", out[2], dev, n), _ints("tok_slot", out[3], dev, n))
    ctx = Context.for_device(dev)
    st = _lib.lib().rtd_kv_plan(ctx.handle, _ints("want", want, dev, s), s, _ints("length", length, dev, s),
                                _ints("table", table, dev, s, most), most,
                                _ints("free_list", free_list, dev, free_list.numel()),
                                _ints("free_count", free_count, dev, 1), free_list.numel(), *lists, n,
                                _stream(dev.index))
    if st:
        _raise(st, ctx.handle)
    return out


def append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, inv_freq: torch.Tensor, tok_pos: torch.Tensor,
           tok_slot: torch.Tensor, pages: torch.Tensor, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate q [T, n_head, D] and k [T, n_kv, D] by tok_pos * inv_freq (the first
    2 * len(inv_freq) dims), quantise k and v into the pages at tok_slot (negative: left
    out) and return the rotated queries, f32 [T, n_head, D]."""
    d = q.shape[-1]
    blocks, n_kv = _pool(pages, d)
    dev = pages.device
    ldq, ldk, ldv = _heads("q", q, dev, d), _heads("k", k, dev, d), _heads("v", v, dev, d)
    t, n_head = q.shape[0], q.shape[1]
    if k.shape[0] != t or v.shape[0] != t or k.shape[1] != n_kv or v.shape[1] != n_kv:
        raise ShapeError("k / v", [t, n_kv, d], list(k.shape if k.shape[:2] != (t, n_kv) else v.shape))
    if not (q.dtype == k.dtype == v.dtype):
        raise ConfigError(f"q, k and v of one type are wanted, got {q.dtype}, {k.dtype}, {v.dtype}")
    if inv_freq.dtype != torch.float64 or inv_freq.device != dev or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ConfigError("inv_freq: a contiguous f64 vector on the pages' device is wanted")
    if q_out is None:
        q_out = torch.empty((t, n_head, d), dtype=torch.float32, device=dev)
    elif tuple(q_out.shape) != (t, n_head, d) or q_out.dtype != torch.float32 or not q_out.is_contiguous() or q_out.device != dev:
        raise ShapeError("q_out", [t, n_head, d], list(q_out.shape))
    ctx = Context.for_device(dev)
    st = _lib.lib().rtd_rope_kv4_append(ctx.handle, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv,
                                        _DT[q.dtype], t, n_head, n_kv, d, 2 * inv_freq.shape[0], inv_freq.data_ptr(),
                                        _ints("tok_pos", tok_pos, dev, t), _ints("tok_slot", tok_slot, dev, t),
                                        pages.data_ptr(), blocks, q_out.data_ptr(), _stream(dev.index))
    if st:
        _raise(st, ctx.handle)
    return q_out


def read(pages: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float32):
    """(k, v) [n, n_kv, D]: the values held in int32 ``slots`` (zeros where negative)."""
    d = pages.shape[-1] // 20
    blocks, n_kv = _pool(pages, d)
    dev = pages.device
    if dtype not in _DT:
        raise ConfigError(f"read: {dtype} (f32, f16 or bf16)")
    n = slots.shape[0]
    k, v = torch.empty((2, n, n_kv, d), dtype=dtype, device=dev).unbind(0)
    ctx = Context.for_device(dev)
    st = _lib.lib().rtd_kv4_read(ctx.handle, _ints("slots", slots, dev, n), n, n_kv, d, pages.data_ptr(), blocks,
                                 k.data_ptr(), v.data_ptr(), _DT[dtype], _stream(dev.index))
    if st:
        _raise(st, ctx.handle)
    return k, v


def attention(q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor,
              max_q: int, max_ctx: int, scale: Optional[float] = None, out_dtype: torch.dtype = torch.float32,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """o [T, n_head, D]: causal GQA of q [T, n_head, D] over the pages.  Sequence s (row s of
    ``table``) has the queries q_start[s] .. q_start[s + 1] - 1, at the last positions of
    its ctx_len[s] tokens.  ``max_q`` and ``max_ctx`` bound the queries and the length of
    any sequence.  Rows of no sequence are left as they were in ``out``."""
    d = q.shape[-1]
    blocks, n_kv = _pool(pages, d)
    dev = pages.device
    ldq = _heads("q", q, dev, d)
    t, n_head = q.shape[0], q.shape[1]
    if table.dim() != 2:
        raise ShapeError("table", [-1, -1], list(table.shape))
    s, most = table.shape
    if out is None:
        out = torch.empty((t, n_head, d), dtype=out_dtype, device=dev)
    if out.shape != q.shape:
        raise ShapeError("out", list(q.shape), list(out.shape))
    ldo = _heads("out", out, dev, d)
    ctx = Context.for_device(dev)
    st = _lib.lib().rtd_attention_kv4(ctx.handle, q.data_ptr(), _DT[q.dtype], ldq, t, n_head, n_kv, d,
                                      1.0 / math.sqrt(d) if scale is None else scale,
                                      _ints("q_start", q_start, dev, s + 1), _ints("ctx_len", ctx_len, dev, s), s,
                                      _ints("table", table, dev, s, most), most, max_q, max_ctx, pages.data_ptr(),
                                      blocks, out.data_ptr(), _DT[out.dtype], ldo, _stream(dev.index))
    if st:
        if st == _lib.RTD_ERR_SHAPE:
            msg = _lib.lib().rtd_last_error(ctx.handle)
            raise ConfigError(msg.decode() if msg else "rtd_attention_kv4: shape")
        _raise(st, ctx.handle)
    return out
