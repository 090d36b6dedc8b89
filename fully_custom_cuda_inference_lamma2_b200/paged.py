"""Paged KV cache: pages of a shared pool instead of an arena row range per sequence.

KVArena (arena.py) reserves every sequence's capacity for its whole life, in fp16. Here a
sequence holds as many pages of `page_size` tokens as its rows need, taken from one pool,
and the pool may hold e4m3 codes with one power-of-two scale for each page and kv head
(float8_e8m0fnu), half the bytes of fp16:

  k/v          [L, num_pages, Hkv, page_size, D]   fp16 or float8_e4m3fn
  k/v_scales   [L, num_pages, Hkv]                 float8_e8m0fnu (e4m3 only)
  page_table   [B, max_pages] int32                the same pages in every layer
  seq_lens     [B] int32                           rows cached, read and moved on the device

Pages are given out on the host (reserve / release) before the calls that fill them; the
calls themselves (paged_append, paged_decode, paged_prefill) read the table and the
lengths on the device, so they are capturable and one graph serves every length.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import attn_varlen


class PagedKVCache:
    """Pools of `num_pages` pages for `layers` layers, and the page table of B sequences.

    max_tokens / max_seqlen: the most new tokens of one call, and of one sequence in it (a decode
    step has B and 1); max_kv_tokens: the most keys of all sequences in a paged_prefill of more
    than 64 query rows per kv head (default: what the pool holds)."""

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, *, num_pages: int, page_size: int = 64,
                 max_pages: Optional[int] = None, q_heads: Optional[int] = None, dtype=torch.float8_e4m3fn,
                 max_tokens: Optional[int] = None, max_seqlen: int = 1, max_kv_tokens: Optional[int] = None, device=None):
        if dtype not in (torch.float16, torch.float8_e4m3fn):
            raise ValueError("the paged cache holds float16 or float8_e4m3fn")
        if page_size not in (16, 32, 64, 128) or page_size * head_dim > 16384:
            raise ValueError("page_size must be 16, 32, 64 or 128, and page_size * head_dim at most 16384")
        if layers <= 0 or batch <= 0 or kv_heads <= 0 or num_pages <= 0:
            raise ValueError("layers, batch, kv_heads and num_pages must be positive")
        self.layers, self.batch, self.kv_heads, self.head_dim = layers, batch, kv_heads, head_dim
        self.q_heads = q_heads if q_heads is not None else kv_heads
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.max_pages = int(max_pages) if max_pages is not None else self.num_pages
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        shape = (layers, self.num_pages, kv_heads, self.page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=self.device)
        self.v = torch.empty(shape, dtype=dtype, device=self.device)
        self.k_scales = self.v_scales = None
        if dtype == torch.float8_e4m3fn:
            self.k_scales = torch.empty(shape[:3], dtype=torch.float8_e8m0fnu, device=self.device)
            self.v_scales = torch.empty(shape[:3], dtype=torch.float8_e8m0fnu, device=self.device)
        self.page_table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=self.device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=self.device)
        max_tokens = max(batch, int(max_tokens)) if max_tokens is not None else batch * max_seqlen
        if max_kv_tokens is None:
            max_kv_tokens = self.num_pages * self.page_size if max_seqlen > 1 else 0
        self.workspace = attn_varlen.make_paged_workspace(batch, self.q_heads, kv_heads, head_dim, max_tokens,
                                                          int(max_seqlen), int(max_kv_tokens), self.device)
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(batch)]

    def layer(self, l: int):
        """(k, v, k_scales, v_scales) views of layer l in the layout that the attn_varlen.paged_* calls take."""
        return self.k[l], self.v[l], None if self.k_scales is None else self.k_scales[l], \
            None if self.v_scales is None else self.v_scales[l]

    def pages_of(self, seq: int) -> List[int]:
        """The pages that sequence `seq` holds, in order."""
        return list(self._pages[seq])

    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, seq: int, tokens: int) -> None:
        """Give sequence `seq` the pages for `tokens` rows in all (it keeps the ones that it has).

        On the current stream, which the calls that use the pages follow. Raises RuntimeError, and changes
        nothing, when the pool or the table's row has too few."""
        have = self._pages[seq]
        need = -(-int(tokens) // self.page_size) - len(have)
        if need <= 0:
            return
        if len(have) + need > self.max_pages:
            raise RuntimeError(f"sequence {seq}: {tokens} tokens need more than {self.max_pages} pages")
        if need > len(self._free):
            raise RuntimeError(f"sequence {seq}: {need} pages needed, {len(self._free)} free")
        new = self._free[:-need - 1:-1]
        self.page_table[seq, len(have):len(have) + need] = torch.tensor(new, dtype=torch.int32).to(self.device)
        del self._free[-need:]
        have.extend(new)

    def release(self, seq: int) -> None:
        """Take back the pages of sequence `seq` and set its length to 0, on the current stream."""
        self._free.extend(reversed(self._pages[seq]))
        self._pages[seq] = []
        self.page_table[seq].fill_(-1)
        self.seq_lens[seq].zero_()

    def read_error(self, clear: bool = True) -> int:
        """The device error word (bit 0 capacity, 1 timeout, 3 page outside the pool, 4 a scale byte
        that no append makes, in a long chunk); synchronises."""
        return attn_varlen.paged_read_error(self.workspace, clear)


def paged_append(cache: PagedKVCache, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, *,
                 q: Optional[torch.Tensor] = None, q_rot_out: Optional[torch.Tensor] = None,
                 cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: int = -1, advance: bool = False,
                 rope_theta: float = 10000.0, rotary_dim: int = -1) -> None:
    """RoPE on k_new (and q) at positions T_b + i, and append of (k_rot, v_new) to `layer`'s pages. One token per
    sequence ([B, H, D]), or ragged rows with cu_seqlens_q and max_seqlen_q."""
    k, v, ks, vs = cache.layer(layer)
    attn_varlen.paged_append(k_new, v_new, k, v, cache.page_table, cache.seq_lens, k_scales=ks, v_scales=vs, q=q,
                             q_rot_out=q_rot_out, cu_seqlens_q=cu_seqlens_q, max_seqlen_q=max_seqlen_q,
                             rope_theta=rope_theta, rotary_dim=rotary_dim, advance=advance, workspace=cache.workspace)


def paged_decode(cache: PagedKVCache, layer: int, q: torch.Tensor, out: torch.Tensor, *,
                 k_new: Optional[torch.Tensor] = None, v_new: Optional[torch.Tensor] = None, advance: bool = False,
                 scale: Optional[float] = None, rope_theta: float = 10000.0, rotary_dim: int = -1,
                 q_rot_out: Optional[torch.Tensor] = None, prefetch_kv: bool = False) -> torch.Tensor:
    """One decode step of `layer`: RoPE + append at T_b (when k_new is given) and split-KV attention over all keys of
    each sequence, in one launch on the current stream, without allocation or host sync.

    prefetch_kv: read the lengths, the page table and the cached rows before waiting for the previous kernel on the
    stream (FCCI_PAGED_PREFETCH_KV). Only when no kernel that may still be running writes them, e.g. right after the
    projection that produced q/k_new/v_new, or in a chain of layers' steps whose first has it not set and of which only
    the last advances."""
    k, v, ks, vs = cache.layer(layer)
    attn_varlen.paged_decode(q, k, v, out, cache.page_table, cache.seq_lens, k_scales=ks, v_scales=vs, k_new=k_new,
                             v_new=v_new, scale=-1.0 if scale is None else float(scale), rope_theta=rope_theta,
                             rotary_dim=rotary_dim, advance=advance, q_rot_out=q_rot_out, workspace=cache.workspace,
                             prefetch_kv=prefetch_kv)
    return out


def paged_prefill(cache: PagedKVCache, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                  out: torch.Tensor, cu_seqlens_q: torch.Tensor, max_seqlen_q: int, *, advance: bool = False,
                  scale: Optional[float] = None, rope_theta: float = 10000.0, rotary_dim: int = -1) -> torch.Tensor:
    """Prompts or chunks of `layer`: RoPE + append of n_b new tokens at T_b, causal attention of token i over keys
    0 .. T_b + i. Rows behind cu_seqlens_q[B] are left as they were."""
    k, v, ks, vs = cache.layer(layer)
    attn_varlen.paged_prefill(q, k_new, v_new, k, v, out, cache.page_table, cache.seq_lens, cu_seqlens_q, max_seqlen_q,
                              k_scales=ks, v_scales=vs, scale=-1.0 if scale is None else float(scale),
                              rope_theta=rope_theta, rotary_dim=rotary_dim, advance=advance, workspace=cache.workspace)
    return out
