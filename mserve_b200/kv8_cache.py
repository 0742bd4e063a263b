"""An HBM-resident KV cache in 8 bits for a fixed batch of sequences.

Beside the offload engine (engine.OffloadKV: 16-bit KV in host memory, selected rows over the host link)
for sequences that fit HBM at one byte per value: K and V of every layer in 8-bit pages with a
power-of-two scale per (page, KV head) and the pages' key bounds (ops.Kv8Pages), one int32 page table
[B, max_pages] shared by all layers.  No counterpart in the reference.

A decode step, per layer: the step's tokens are appended (mskv_kv8_append), then either the whole cache is
attended (mskv_kv8_attention) or, with ``top_blocks``, every page is scored from its bounds
(mskv_kv8_block_score), the best pages and the last ones are selected per (sequence, KV head)
(mskv_topk) and attention runs over those.  No host synchronisation: ``begin_step`` sends the step's
lengths through pinned staging, so the per-layer calls can be captured once in a CUDA graph and replayed
while the cache grows.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Union

import numpy as np
import torch

from . import ops


class PagedKV8:
    """8-bit paged KV of num_layers layers for `batch` sequences of up to `capacity` tokens.

    q_heads, kv_heads, head_dim: the model's (this rank's share, when heads are sharded); page_size: tokens
    per page; cache_dtype: torch.float8_e4m3fn or torch.float8_e5m2.  top_blocks > 0: attention over the
    top_blocks best pages and the last recent_blocks (at least 1) of every (sequence, KV head), the pages of
    the query's own positions always among the last; 0: over the whole cache.
    """

    def __init__(self, num_layers: int, batch: int, q_heads: int, kv_heads: int, head_dim: int, capacity: int, *,
                 top_blocks: int = 0, recent_blocks: int = 1, page_size: int = 16,
                 cache_dtype: torch.dtype = torch.float8_e4m3fn, device: Optional[torch.device] = None):
        if num_layers <= 0:
            raise ValueError("num_layers must be positive")
        if batch <= 0 or kv_heads <= 0 or q_heads <= 0 or q_heads % kv_heads:
            raise ValueError("q_heads must be a positive multiple of kv_heads, batch positive")
        ops.check_kv8_layout(page_size, head_dim, cache_dtype)
        if capacity <= 0:
            raise ValueError("capacity must be positive")
        if top_blocks < 0 or (top_blocks > 0 and recent_blocks < 1):
            raise ValueError("top_blocks must be >= 0, and recent_blocks >= 1 with it")
        self.device = ops._norm(device if device is not None else "cuda")
        self.L, self.B, self.Hq, self.Hkv, self.D = num_layers, batch, q_heads, kv_heads, head_dim
        self.C, self.page_size = int(capacity), int(page_size)
        self.top_blocks, self.recent_blocks = int(top_blocks), int(recent_blocks)
        self.max_pages = (self.C + page_size - 1) // page_size
        self.num_pages = batch * self.max_pages
        self.pages: List[ops.Kv8Pages] = [
            ops.kv8_pages(self.num_pages, kv_heads, head_dim, page_size=page_size, dtype=cache_dtype, device=self.device,
                          bounds=top_blocks > 0)
            for _ in range(num_layers)]
        self._free = list(range(self.num_pages - 1, -1, -1))
        self.page_table_h = np.full((batch, self.max_pages), -1, dtype=np.int32)
        self.page_table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=self.device)
        self.len_h = np.zeros(batch, dtype=np.int64)
        # the step's state on the device: lengths before it, tokens it appends, lengths and blocks after it
        self._state = torch.zeros(4, batch, dtype=torch.int32, device=self.device)
        self.tok0, self.n_new, self.lens, self.held = self._state.unbind(0)
        self._most_new = 0                          # tokens that the step appends to one sequence, at most
        self._idx = self._counts = None             # of the last selection, for inspection

    # ------------------------------------------------------------------ lengths and pages
    def begin_step(self, n_new: Union[int, Sequence[int]] = 1) -> None:
        """Room for n_new tokens of every sequence (an int, or one number each; 0 leaves a sequence as it is).

        Maps the pages they need and sets the device-side lengths, through pinned staging copies on the current
        stream; the host waits for nothing.  append_layer then writes each layer's rows and decode_layer attends
        over the grown cache.  Not to be captured (a replay would send the captured step's lengths again).
        """
        self._not_captured()
        given = np.asarray(n_new)
        if given.dtype.kind not in "iu" or given.shape not in ((), (self.B,)):
            raise ValueError(f"n_new must be an integer or one for each of the {self.B} sequences")
        n_new = np.broadcast_to(given.astype(np.int64), (self.B,))
        if (n_new < 0).any():
            raise ValueError("n_new must not be negative")
        new_len = self.len_h + n_new
        if (new_len > self.C).any():
            raise ValueError(f"a step exceeds the capacity of {self.C} tokens per sequence")
        # a page for every position up to the new lengths: batch * max_pages of them exist, so one is always free
        mapped = False
        for b in range(self.B):
            for p in range(int(self.len_h[b]) // self.page_size, -(-int(new_len[b]) // self.page_size)):
                if self.page_table_h[b, p] < 0:
                    self.page_table_h[b, p] = self._free.pop()
                    mapped = True
        self._send(self.len_h, n_new, new_len, mapped)
        self.len_h = new_len

    def reset(self, b: int) -> None:
        """Empties sequence b: its pages are free for others from the next step on.

        Called between steps: a step that is under way loses the rows it has not appended yet.
        """
        if not 0 <= b < self.B:
            raise ValueError(f"no sequence {b}")
        self._not_captured()
        row = self.page_table_h[b]
        self._free.extend(int(p) for p in row[row >= 0])
        row[:] = -1
        self.len_h = self.len_h.copy()
        self.len_h[b] = 0
        self._send(self.len_h, np.zeros(self.B, dtype=np.int64), self.len_h, True)

    def _not_captured(self) -> None:
        with torch.cuda.device(self.device.index):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("begin_step and reset belong between a captured step's replays, not into the capture")

    def _send(self, old: np.ndarray, n_new: np.ndarray, new: np.ndarray, table: bool) -> None:
        self._most_new = int(n_new.max())

        def send(to: torch.Tensor, values: np.ndarray) -> None:
            # pinned memory of this copy's own: torch's allocator hands it out again when the copy is done
            to.copy_(torch.from_numpy(values.astype(np.int32)).pin_memory(), non_blocking=True)

        with torch.cuda.device(self.device.index):
            if table:
                send(self.page_table, self.page_table_h)
            send(self._state, np.stack([old, n_new, new, -(-new // self.page_size)]))

    # ------------------------------------------------------------------ a layer of the step
    def append_layer(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """The step's rows [B, Hkv, n, D] of one layer (n at least every sequence's n_new; fp32, fp16 or bf16).

        A captured call writes n rows at most: its replays are for steps of up to n tokens.
        """
        if k_new.dim() != 4 or k_new.shape[:2] != (self.B, self.Hkv) or k_new.shape[3] != self.D:
            raise ValueError(f"k_new must be [B={self.B}, Hkv={self.Hkv}, n, D={self.D}]")
        if k_new.shape[2] < self._most_new:
            raise ValueError(f"the step appends up to {self._most_new} tokens, k_new holds {k_new.shape[2]}")
        ops.kv8_append(self.pages[layer], self.page_table, k_new, v_new, tok0=self.tok0, counts=self.n_new)

    def _recent(self, positions: int) -> int:
        """Last pages that are always attended: recent_blocks, and those of the last `positions` tokens wherever they end in a page."""
        return max(self.recent_blocks, 1 - (1 - positions) // self.page_size)

    def _check_q(self, q: torch.Tensor) -> None:
        if q.dim() not in (3, 4) or q.shape[:2] != (self.B, self.Hq) or q.shape[-1] != self.D:
            raise ValueError(f"q must be [B={self.B}, Hq={self.Hq}, (Q,) D={self.D}], got {list(q.shape)}")

    def select(self, layer: int, q: torch.Tensor):
        """Pages for q [B, Hq, D] or [B, Hq, Q, D]: (indices [B, Hkv, top + recent], ascending, counts [B, Hkv]), the caller's own.

        The best top_blocks are those of the last position's scores; the last pages are recent_blocks, or as many as the Q
        positions' own tokens can lie in (two, where Q > 1) if that is more, so every position attends to itself.
        """
        self._check_q(q)
        recent = self._recent(q.shape[2] if q.dim() == 4 else 1)
        rows, dev = self.B * self.Hkv, self.device
        scores = torch.empty(rows, self.max_pages, dtype=torch.float32, device=dev)
        self._idx = torch.empty(rows, self.top_blocks + recent, dtype=torch.int32, device=dev)
        self._counts = torch.empty(rows, dtype=torch.int32, device=dev)
        ops.kv8_block_score(q, self.pages[layer], self.page_table, lens=self.lens, max_blocks=self.max_pages,
                            out=scores.view(self.B, self.Hkv, self.max_pages))
        with torch.cuda.device(dev.index):          # ops.topk launches on the current device
            ops.topk(scores, top_k=self.top_blocks, recent=recent, len_=self.held, len_scalar=self.max_pages,
                     sel_per_batch=self.Hkv, out=self._idx, counts=self._counts)
        return self._idx.view(self.B, self.Hkv, -1), self._counts.view(self.B, self.Hkv)

    def decode_layer(self, layer: int, q: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                     t_bound: Optional[int] = None) -> torch.Tensor:
        """Attention of the last Q tokens over one layer's cache: q [B, Hq, Q, D] (or [B, Hq, D]) -> [B, Hq, Q, D].

        Position i of a sequence of length n sees the tokens below n - Q + 1 + i.  t_bound: the length bound
        that the kernel is launched for, from the longest sequence's length to the capacity (the default, which
        stays valid in a captured step while the cache grows; a smaller one does up to that length).
        """
        if q.dim() == 3:
            q = q.unsqueeze(2)
        if t_bound is not None and not int(self.len_h.max()) <= t_bound <= self.C:
            raise ValueError(f"t_bound {t_bound} must lie in [{int(self.len_h.max())}, {self.C}]")
        if self.top_blocks:
            idx, counts = self.select(layer, q)
            return ops.kv8_attention(q, self.pages[layer], self.page_table, lens=self.lens, blocks=idx, counts=counts, out=out)
        self._check_q(q)
        return ops.kv8_attention(q, self.pages[layer], self.page_table, lens=self.lens,
                                 max_tokens=self.C if t_bound is None else t_bound, out=out)

    def step_layer(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, *,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """append_layer and decode_layer: one layer of a decode step."""
        self.append_layer(layer, k_new, v_new)
        return self.decode_layer(layer, q, out=out)
