"""Host-side page allocator for a paged KV cache.

Same contract as the reference's ``PagedKVCache`` and ``PAGE_SIZE``
(fskernels/paged_attn/paged_kv_cache.py:6-154): pools
[num_layers, num_pages, num_kv_heads, 16, head_dim], a device block table
[max_seqs, max_blocks_per_seq] int32 with -1 for unallocated entries, a free
list, ``allocate_sequence``/``free_sequence``/``append_kv``/
``get_block_table_tensor``/``get_seq_lens_tensor`` and the
``pages_used``/``pages_free`` counters.

Differences: the logical->physical map is mirrored on the host, so neither
``append_kv`` nor ``free_sequence`` reads the device block table back (the
reference calls ``.item()`` per appended token, paged_kv_cache.py:126);
``from_config`` honours a ``dtype`` argument (the reference hard-wires
bfloat16, :80); pools may be float8_e4m3fn; sequences can share the pages of a
common prefix (``fork_sequence``, counted references); a step can append any
number of tokens per sequence with the position rotation on the way
(``begin_chunk``, ``append_qkv_batch``).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List

import torch

from .. import _native as N

PAGE_SIZE = 16


@dataclass
class PagedKVCache:
    num_layers: int
    num_pages: int
    max_seqs: int
    max_blocks_per_seq: int
    num_kv_heads: int
    head_dim: int
    dtype: torch.dtype
    device: str

    def __post_init__(self):
        shape = (self.num_layers, self.num_pages, self.num_kv_heads, PAGE_SIZE, self.head_dim)
        self.k_pool = torch.zeros(shape, dtype=self.dtype, device=self.device)
        self.v_pool = torch.zeros_like(self.k_pool)
        if self.k_pool.is_cuda:
            N.status_word(self.k_pool.device)  # made here: a captured step may be the first to name it
        self.block_table = torch.full((self.max_seqs, self.max_blocks_per_seq), -1, dtype=torch.int32,
                                      device=self.device)
        self._seq_lens: List[int] = [0] * self.max_seqs
        self._active: List[bool] = [False] * self.max_seqs
        self._pages: List[List[int]] = [[] for _ in range(self.max_seqs)]
        # popped from the end: lowest page indices are handed out last, as in the reference
        self._free_pages: List[int] = list(range(self.num_pages))
        # e4m3 pools store x / scale; fixed per-tensor scales (set_fp8_scales)
        self.k_scale = torch.ones((), dtype=torch.float32, device=self.device)
        self.v_scale = torch.ones((), dtype=torch.float32, device=self.device)
        self._step_ids: List[int] = []
        self._step_counts: List[int] = []
        self._step_bt = None
        self._step_pos = None
        self._step_seq = None  # block-table row of each token (None: token t is row t)
        self._step_last = -1   # the step's largest position
        self._page_refs: Dict[int, int] = {}  # holders of the pages that have more than one
        self._shared_runs: Dict[tuple, int] = {}  # shared_prefix_pages by sequences, until the next fork or free

    @classmethod
    def from_config(cls, config, num_pages: int = 4096, max_seqs: int = 16, max_blocks_per_seq: int = 512,
                    device: str = "cuda", dtype: torch.dtype = torch.bfloat16) -> "PagedKVCache":
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        return cls(num_layers=config.num_hidden_layers, num_pages=num_pages, max_seqs=max_seqs,
                   max_blocks_per_seq=max_blocks_per_seq, num_kv_heads=config.num_key_value_heads,
                   head_dim=head_dim, dtype=dtype, device=device)

    def allocate_sequence(self) -> int:
        for sid in range(self.max_seqs):
            if not self._active[sid]:
                self._active[sid] = True
                self._seq_lens[sid] = 0
                self._pages[sid] = []
                return sid
        raise RuntimeError("All sequence slots are occupied")

    def free_sequence(self, seq_id: int) -> None:
        pages = self._pages[seq_id]
        self._shared_runs.clear()
        if pages:
            self.block_table[seq_id, : len(pages)] = -1
            self._free_pages.extend(p for p in pages if self._release(p))
        self._pages[seq_id] = []
        self._active[seq_id] = False
        self._seq_lens[seq_id] = 0

    def _release(self, page: int) -> bool:
        """Give up one holder of a page; True when it was the last one."""
        n = self._page_refs.get(page, 1)
        if n <= 2:
            self._page_refs.pop(page, None)
        else:
            self._page_refs[page] = n - 1
        return n == 1

    def fork_sequence(self, seq_id: int, num_tokens: int) -> int:
        """A new sequence that begins with tokens 0 .. num_tokens - 1 of
        ``seq_id`` by sharing their pages (no copy).  ``num_tokens`` fills whole
        pages, so that neither sequence writes to a shared one: append the rest
        of a prompt to each.  A shared page returns to the pool with its last
        holder."""
        n = int(num_tokens)
        if not 0 <= seq_id < self.max_seqs or not self._active[seq_id]:
            raise ValueError("fork_sequence needs an active sequence")
        if n <= 0 or n % PAGE_SIZE or n > self._seq_lens[seq_id]:
            raise ValueError(f"num_tokens must be a positive multiple of {PAGE_SIZE} up to the sequence's length")
        new = self.allocate_sequence()
        self._shared_runs.clear()
        pages = self._pages[seq_id][: n // PAGE_SIZE]
        for p in pages:
            self._page_refs[p] = self._page_refs.get(p, 1) + 1
        self._pages[new] = list(pages)
        self._seq_lens[new] = n
        self.block_table[new, : len(pages)] = self.block_table[seq_id, : len(pages)]
        return new

    def shared_prefix_pages(self, seq_ids: List[int]) -> int:
        """Leading pages that all of ``seq_ids`` hold in common and have filled."""
        if len(seq_ids) < 2:
            return self._seq_lens[seq_ids[0]] // PAGE_SIZE if seq_ids else 0
        # Only forks make common pages, and those are full: what a set of
        # sequences shares changes with a fork or a free, not with a step.
        key = tuple(seq_ids)
        n = self._shared_runs.get(key)
        if n is None:
            rows = [self._pages[s] for s in seq_ids]
            n, first = min(len(r) for r in rows), rows[0]
            for r in rows[1:]:
                if r is not first and r[:n] != first[:n]:
                    n = next(i for i in range(n) if r[i] != first[i])
            if seq_ids.count(seq_ids[0]) == len(seq_ids):
                return min(n, self._seq_lens[seq_ids[0]] // PAGE_SIZE)  # one sequence, several times
            self._shared_runs[key] = n
        return n

    def _alloc_page(self) -> int:
        if not self._free_pages:
            raise RuntimeError("Out of KV pages")
        return self._free_pages.pop()

    def append_kv(self, seq_id: int, layer_idx: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Append one token's K/V ([1, KV_H, 1, D]) to a sequence of one layer."""
        pos = self._seq_lens[seq_id]
        page_idx, off = divmod(pos, PAGE_SIZE)
        pages = self._pages[seq_id]
        if page_idx == len(pages):
            if page_idx >= self.max_blocks_per_seq:
                raise RuntimeError("sequence exceeds max_blocks_per_seq")
            pp = self._alloc_page()
            pages.append(pp)
            self.block_table[seq_id, page_idx] = pp
        pp = pages[page_idx]
        self.k_pool[layer_idx, pp, :, off, :] = k[0, :, 0, :]
        self.v_pool[layer_idx, pp, :, off, :] = v[0, :, 0, :]
        self._seq_lens[seq_id] = pos + 1

    def write_prefill(self, seq_id: int, layer_idx: int, k: torch.Tensor, v: torch.Tensor, reserve: int = 0) -> None:
        """Write a prompt's K/V ([KV_H, T, D]) as tokens 0..T-1 of one layer of
        a sequence, with one indexed copy per pool (the reference appends the
        prompt token by token, benchmarks/run_hf_triton_fp8_paged.py:113-117).
        Pages are allocated on the host for max(T, reserve) tokens, so a
        caller can fix the block table for the decode steps that follow.
        The sequence length becomes T (the same T for every layer).  A sequence
        that shares pages (``fork_sequence``) is refused."""
        if k.dim() != 3 or k.shape != v.shape or k.shape[0] != self.num_kv_heads or k.shape[2] != self.head_dim:
            raise ValueError("k / v must be [num_kv_heads, T, head_dim]")
        T = int(k.shape[1])
        pages = self._pages[seq_id]
        # An empty prompt too: the tokens after it would go to the first page.
        # Who holds a page holds those before it, so the first one tells.
        if pages and pages[0] in self._page_refs:
            raise RuntimeError("write_prefill would overwrite pages shared with another sequence")
        need = (max(T, int(reserve)) + PAGE_SIZE - 1) // PAGE_SIZE
        if need > self.max_blocks_per_seq:
            raise RuntimeError("sequence exceeds max_blocks_per_seq")
        if need > len(pages):
            new = [self._alloc_page() for _ in range(need - len(pages))]
            first = len(pages)
            pages.extend(new)
            self.block_table[seq_id, first:need] = torch.tensor(new, dtype=torch.int32).to(self.device)
        if T > 0:
            tok = torch.arange(T)
            phys = torch.tensor(pages, dtype=torch.long)[tok // PAGE_SIZE].to(self.device)
            slot = (tok % PAGE_SIZE).to(self.device)
            kt, vt = k.transpose(0, 1), v.transpose(0, 1)  # [T, KV_H, D]
            if self.dtype == torch.float8_e4m3fn:
                kt = (kt.float() / self.k_scale).clamp(-448.0, 448.0).to(self.dtype)
                vt = (vt.float() / self.v_scale).clamp(-448.0, 448.0).to(self.dtype)
            self.k_pool[layer_idx][phys, :, slot, :] = kt.to(self.dtype)
            self.v_pool[layer_idx][phys, :, slot, :] = vt.to(self.dtype)
        self._seq_lens[seq_id] = T

    def set_fp8_scales(self, k_scale, v_scale) -> None:
        """Per-tensor scales of an e4m3 pool (value = e4m3 x scale), e.g. amax / 448
        of calibration K/V."""
        self.k_scale.fill_(float(k_scale))
        self.v_scale.fill_(float(v_scale))

    # ---------------------------------------------------------- batched decode step
    def begin_step(self, seq_ids: List[int]):
        """Reserve the slot of one new token for each sequence in ``seq_ids``:
        pages are allocated on the host (no device read-back) and the new
        block-table entries are written with one host-to-device copy.  Returns
        (block_table [B, max_blocks], positions [B]) device tensors for
        ``append_kv_batch`` and the decode call."""
        rows, cols, vals = [], [], []
        for sid in seq_ids:
            pos = self._seq_lens[sid]
            page_idx = pos // PAGE_SIZE
            pages = self._pages[sid]
            if page_idx == len(pages):
                if page_idx >= self.max_blocks_per_seq:
                    raise RuntimeError("sequence exceeds max_blocks_per_seq")
                pp = self._alloc_page()
                pages.append(pp)
                rows.append(sid)
                cols.append(page_idx)
                vals.append(pp)
        if rows:
            upd = torch.tensor([rows, cols, vals], dtype=torch.int64).to(self.device, non_blocking=True)
            self.block_table[upd[0], upd[1]] = upd[2].to(torch.int32)
        self._step_ids = list(seq_ids)
        self._step_counts = [1] * len(seq_ids)
        self._step_seq = None
        self._step_last = max((self._seq_lens[s] for s in seq_ids), default=-1)
        self._step_bt = self.get_block_table_tensor(self._step_ids)
        self._step_pos = self.get_seq_lens_tensor(self._step_ids)
        return self._step_bt, self._step_pos, self._step_pos + 1

    def begin_chunk(self, seq_ids: List[int], counts: List[int]):
        """Reserve the slots of ``counts[i]`` new tokens for each (distinct)
        sequence ``seq_ids[i]``: prompt chunks, or several tokens of a step.
        Returns (block_table [B, max_blocks], positions [T], block-table row of
        each token [T]), device tensors; the tokens of a sequence follow one
        another, sequences in order.  Append with ``append_qkv_batch``, commit
        with ``end_step``."""
        counts = [int(c) for c in counts]
        if len(counts) != len(seq_ids) or any(c < 0 for c in counts):
            raise ValueError("counts must have one non-negative entry per sequence")
        if len(set(seq_ids)) != len(seq_ids):
            raise ValueError("begin_chunk takes each sequence once")
        need = [(self._seq_lens[s] + c + PAGE_SIZE - 1) // PAGE_SIZE for s, c in zip(seq_ids, counts)]
        if any(n > self.max_blocks_per_seq for n in need):
            raise RuntimeError("sequence exceeds max_blocks_per_seq")
        if sum(max(n - len(self._pages[s]), 0) for s, n in zip(seq_ids, need)) > len(self._free_pages):
            raise RuntimeError("Out of KV pages")
        rows, cols, vals, pos, seq = [], [], [], [], []
        for i, (s, c, n) in enumerate(zip(seq_ids, counts, need)):
            pages = self._pages[s]
            while len(pages) < n:
                rows.append(s)
                cols.append(len(pages))
                vals.append(self._alloc_page())
                pages.append(vals[-1])
            first = self._seq_lens[s]
            pos.extend(range(first, first + c))
            seq.extend([i] * c)
        if rows:
            upd = torch.tensor([rows, cols, vals], dtype=torch.int64).to(self.device, non_blocking=True)
            self.block_table[upd[0], upd[1]] = upd[2].to(torch.int32)
        self._step_ids, self._step_counts = list(seq_ids), counts
        self._step_last = max((self._seq_lens[s] + c - 1 for s, c in zip(seq_ids, counts) if c), default=-1)
        self._step_bt = self.get_block_table_tensor(self._step_ids)
        place = torch.tensor([pos, seq], dtype=torch.int32).to(self.device, non_blocking=True)
        self._step_pos, self._step_seq = place[0], place[1]
        return self._step_bt, self._step_pos, self._step_seq

    def append_qkv_batch(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos, sin, *, q_weight=None,
                         k_weight=None, eps: float = 1e-6, interleaved: bool = False, q_out=None, k_out=None, status=None):
        """Norm and rotate this step's q and k and write k and v into layer
        ``layer_idx`` with one kernel: q [T, Q_H, D], k / v [T, KV_H, D] of the
        tokens of ``begin_step`` (T = B) or ``begin_chunk``; the other arguments
        are those of ``paged_kv_append_rope``.  A step that goes past the rows of
        cos / sin is refused; what the kernel finds is in ``read_status()``, or in
        ``status``.  Returns the rotated q."""
        from .paged_append_rope import paged_kv_append_rope
        if self._step_pos is None:
            raise RuntimeError("call begin_step() or begin_chunk() before append_qkv_batch()")
        if cos is not None and self._step_last >= cos.shape[0]:
            raise ValueError(f"position {self._step_last} of this step is past the {cos.shape[0]} rows of cos / sin")
        if status is None and self.k_pool.is_cuda:
            status = N.status_word(self.k_pool.device)
        e4m3 = self.dtype == torch.float8_e4m3fn
        return paged_kv_append_rope(q, k, v, self.k_pool[layer_idx], self.v_pool[layer_idx], self._step_bt, self._step_pos,
                                    cos, sin, seq_ids=self._step_seq, q_weight=q_weight, k_weight=k_weight, eps=eps,
                                    interleaved=interleaved, scale_k=self.k_scale if e4m3 else None,
                                    scale_v=self.v_scale if e4m3 else None, q_out=q_out, k_out=k_out, status=status)

    def append_kv_batch(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Write this step's K/V ([B, KV_H, 128] or [B, KV_H, 1, 128]) of every
        sequence of ``begin_step`` into layer ``layer_idx`` with one kernel."""
        from .paged_append import paged_kv_append
        if self._step_pos is None or self._step_seq is not None:
            raise RuntimeError("call begin_step() before append_kv_batch()")
        paged_kv_append(k, v, self.k_pool[layer_idx], self.v_pool[layer_idx], self._step_bt, self._step_pos,
                        scale_k=self.k_scale, scale_v=self.v_scale)

    def end_step(self) -> torch.Tensor:
        """Commit the step: every sequence grows by its tokens (one each after
        ``begin_step``, ``counts`` after ``begin_chunk``).
        Returns the new lengths [B] (device) for the next decode call."""
        for sid, count in zip(self._step_ids, self._step_counts):
            self._seq_lens[sid] += count
        lens = self.get_seq_lens_tensor(self._step_ids)
        self._step_ids, self._step_counts = [], []
        self._step_bt = self._step_pos = self._step_seq = None
        return lens

    def seq_len(self, seq_id: int) -> int:
        return self._seq_lens[seq_id]

    def get_block_table_tensor(self, active_seq_ids: List[int]) -> torch.Tensor:
        idx = torch.tensor(active_seq_ids, dtype=torch.long, device=self.device)
        return self.block_table[idx]

    def get_seq_lens_tensor(self, active_seq_ids: List[int]) -> torch.Tensor:
        return torch.tensor([self._seq_lens[s] for s in active_seq_ids], dtype=torch.int32, device=self.device)

    @property
    def pages_used(self) -> int:
        return self.num_pages - len(self._free_pages)

    @property
    def pages_free(self) -> int:
        return len(self._free_pages)

    def __repr__(self) -> str:
        return (f"PagedKVCache(pages={self.num_pages}, used={self.pages_used}, "
                f"seqs={sum(self._active)}/{self.max_seqs})")
