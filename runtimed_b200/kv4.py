"""The paged KV cache held in 4 bits: device-side block tables, the quantising append,
attention over the pages and a reader.

Torch-level entry points of ``rtd_kv_plan``, ``rtd_rope_kv4_append``, ``rtd_attention_kv4``
and ``rtd_kv4_read`` (``include/rtd.h`` states the format and the rules).  Each runs on the
current stream of its tensors' device, allocates nothing but the outputs it returns, and
may be captured in a CUDA graph.  ``attention`` works in its device's context: calls on two
streams of a device, replayed graphs among them, must not overlap.  ``BlockTables`` keeps the state that ``plan`` works on.

What only the device can see (a block id outside the pool, a length beyond its bound, an
exhausted pool) is reported by ``Context.check_device_status``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import numpy as np
import torch

from ._torch import binding
from .errors import ConfigError
from .weights import _DT

BLOCK = 16   # tokens of a page
GROUP = 32   # dims that share a step and a minimum
HEAD_DIMS = (32, 64, 96, 128)
MAX_SEQS = 8192


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


def plan(want: torch.Tensor, length: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
         free_count: torch.Tensor, max_tokens: Optional[int] = None,
         out: Optional[Tuple[torch.Tensor, ...]] = None) -> Optional[Tuple[torch.Tensor, ...]]:
    """Bring every sequence from ``length`` to ``want`` tokens: blocks move between ``table``
    [S, max_blocks] and the stack ``free_list`` / ``free_count``, all int32 and updated in
    place (`rtd_kv_plan`; at most MAX_SEQS sequences).

    With ``max_tokens`` (or ``out``, four buffers to reuse) the new tokens are listed:
    (q_start [S + 1], tok_seq, tok_pos, tok_slot [max_tokens]), -1 behind the last token."""
    return binding.plan(want, length, table, free_list, free_count, max_tokens, out)


def append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, inv_freq: torch.Tensor, tok_pos: torch.Tensor,
           tok_slot: torch.Tensor, pages: torch.Tensor, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate q [T, n_head, D] and k [T, n_kv, D] by tok_pos * inv_freq (the first
    2 * len(inv_freq) dims), quantise k and v into the pages at tok_slot (negative: left
    out) and return the rotated queries, f32 [T, n_head, D]."""
    return binding.append(q, k, v, inv_freq, tok_pos, tok_slot, pages, q_out)


def read(pages: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [n, n_kv, D]: the values held in int32 ``slots`` (zeros where negative)."""
    return binding.read(pages, slots, _code(dtype))


def attention(q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor,
              max_q: int, max_ctx: int, scale: Optional[float] = None, out_dtype: torch.dtype = torch.float32,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """o [T, n_head, D]: causal GQA of q [T, n_head, D] over the pages.  Sequence s (row s of
    ``table``) has the queries q_start[s] .. q_start[s + 1] - 1, at the last positions of
    its ctx_len[s] tokens.  ``max_q`` and ``max_ctx`` bound the queries and the length of
    any sequence; ``scale`` is 1 / sqrt(D) where it is None.  Rows of no sequence are left as
    they were in ``out``."""
    return binding.attention(q, pages, table, q_start, ctx_len, max_q, max_ctx, scale, _code(out_dtype), out)


def _code(dtype: torch.dtype) -> int:
    code = _DT.get(dtype)
    if code is None:
        raise ConfigError(f"{dtype} (f32, f16 or bf16)")
    return code


class BlockTables:
    """Device-side bookkeeping of a paged cache: lengths, block table and free stack, and the
    token lists of a step, in buffers of their own (a step may be captured in a CUDA graph).

    ``from_cache`` takes over the state of a host-side ``PagedKvCache`` and ``into`` gives it
    back; between the two the host's copy is stale."""

    def __init__(self, max_seqs: int, max_blocks: int, num_blocks: int, max_tokens: int, device="cuda:0"):
        if not 0 < max_seqs <= MAX_SEQS:
            raise ConfigError(f"block tables of {max_seqs} sequences (1 to {MAX_SEQS})")
        i32 = dict(dtype=torch.int32, device=device)
        self.length = torch.zeros((max_seqs,), **i32)
        self.table = torch.zeros((max_seqs, max_blocks), **i32)
        self.free_list = torch.arange(num_blocks - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), num_blocks, **i32)
        self.q_start = torch.zeros((max_seqs + 1,), **i32)
        self.tok_seq, self.tok_pos, self.tok_slot = (torch.full((max_tokens,), -1, **i32) for _ in range(3))

    def step(self, want: torch.Tensor) -> None:
        """Sequences to ``want`` tokens (int32 [max_seqs]); the new tokens into q_start / tok_*."""
        plan(want, self.length, self.table, self.free_list, self.free_count,
             out=(self.q_start, self.tok_seq, self.tok_pos, self.tok_slot))

    def set_lengths(self, want: torch.Tensor) -> None:
        """The same without token lists (a rollback, a release)."""
        plan(want, self.length, self.table, self.free_list, self.free_count)

    @classmethod
    def from_cache(cls, cache, max_tokens: int) -> "BlockTables":
        t = cls(cache.max_seqs, cache.max_blocks, cache.num_blocks, max_tokens, cache.device)
        length = np.zeros(cache.max_seqs, np.int32)
        for s, n in cache.lengths.items():
            length[s] = n
        free = np.zeros(cache.num_blocks, np.int32)
        free[:len(cache._free)] = cache._free
        t.length.copy_(torch.from_numpy(length))
        t.table.copy_(torch.from_numpy(cache._host_table))
        t.free_list.copy_(torch.from_numpy(free))
        t.free_count.fill_(len(cache._free))
        return t

    def into(self, cache) -> None:
        """The state back to the host's cache (waits for the device)."""
        length, table = self.length.cpu().numpy(), self.table.cpu().numpy()
        cache._free = self.free_list[:int(self.free_count)].tolist()
        cache._host_table[:] = table
        cache._blocks = {s: table[s, :-(-int(n) // BLOCK)].tolist() for s, n in enumerate(length) if n}
        cache.lengths = {s: int(n) for s, n in enumerate(length) if n}
        cache._dirty = True
