"""Paged decode of a batch whose sequences share a prefix.

Requests behind one system prompt or document, or samples of one prompt, hold
the same leading pages (``PagedKVCache.fork_sequence``).  ``paged_flash_decode``
reads them once per sequence; ``paged_flash_decode_shared_prefix`` reads them
once for the batch and does the prefix's share as a matrix product on the
tensor cores, joining each sequence's own tokens by log-sum-exp.  The result is
that of ``paged_flash_decode`` over the whole tables up to rounding.
"""
from __future__ import annotations

import torch

from .. import _native as N
from .. import _ops
from ..gqa_decode import HEAD_DIMS, _check_idx, _check_sink
from ..gqa_decode_hf import _scale_ptr


def shared_prefix_pays(batch: int, prefix_len: int) -> bool:
    """Whether reading a prefix once for the batch beats ``paged_flash_decode``
    over the whole tables, which reads it per sequence.  Device times with 8 KV
    heads, head dim 128, tails of 64, pools within L2, whole tables against shared
    prefix: 16-bit pools, 32 query heads, 2 x 2048 tokens 14.8 / 14.0 us, 2 x 4096
    17.2 / 16.0, 16 x 2048 26.3 / 16.4, 32 x 16384 266 / 40; e4m3 pools 2 x 4096
    18.8 / 17.0, 16 x 2048 22.5 / 17.4, 32 x 16384 168 / 41 (2 x 16384 loses: 26.6
    / 28.6); head dim 64, 2 x 4096 14.4 / 14.9, 8 x 2048 15.4 / 13.4.  A call takes
    19 us on the host, one of ``paged_flash_decode`` 24."""
    return batch >= 2 and (batch - 1) * prefix_len >= 4096


def paged_flash_decode_shared_prefix(q, k_pool, v_pool, prefix_table, prefix_len, block_table, seq_lens, page_size, *,
                                     s_aux=None, scale_q=None, scale_k=None, scale_v=None, out_dtype=None, out=None):
    """out[b, qh] = attention of q[b, qh] over the prefix's tokens 0 ..
    prefix_len - 1 followed by sequence b's own 0 .. seq_lens[b] - 1.

    q [B, Q_H, D]; pools [num_pages, KV_H, 16, D] (types as
    ``paged_flash_decode``); prefix_table [n] int32 pages of the prefix;
    prefix_len an int or an int32 device tensor of one entry (read on the
    device, so a captured graph follows it); block_table [B, max_blocks] int32
    pages of the own tokens alone, seq_lens [B] int32 their counts (0: prefix
    only).  A column slice ``table[:, n:]`` of the full tables serves as
    block_table.  The keyword arguments are those of ``paged_flash_decode``.

    The scratch is allocated per call: calls on several streams, and several
    captured graphs, do not share it.  Bad pages are masked and reported by
    ``read_status()``."""
    if q.dim() != 3 or k_pool.dim() != 4 or v_pool.dim() != 4:
        raise ValueError("q must be [B, Q_H, D] and pools [num_pages, KV_H, page_size, D]")
    if not q.is_cuda:
        raise ValueError("paged_flash_decode_shared_prefix runs on CUDA tensors only")
    dev = q.device
    if k_pool.device != dev or v_pool.device != dev:
        raise ValueError("q and the pools must be on the same device")
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
        raise ValueError("k_pool and v_pool must match in shape and dtype")
    B, QH, D = q.shape
    _, KVH, PS, D2 = k_pool.shape
    if int(page_size) != PS or PS != 16:
        raise ValueError(f"page_size must be 16 and match the pool (pool has {PS})")
    if D not in HEAD_DIMS or D2 != D or (D != 128 and k_pool.element_size() == 1):
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} (128 for an e4m3 pool) and match the pools")
    if KVH == 0 or QH == 0 or QH % KVH:
        raise ValueError("q heads must be a multiple of the pools' KV heads")
    e4m3 = N.dtype_code(k_pool.dtype) == N.FK_DTYPE_E4M3
    N.dtype_code(q.dtype)
    if not e4m3 and q.dtype != k_pool.dtype:
        raise TypeError("q must have the pools' dtype for 16-bit pools")
    if torch.is_grad_enabled() and q.requires_grad:
        raise ValueError("paged_flash_decode_shared_prefix has no backward pass; call it under torch.no_grad()")
    if out_dtype is None:
        out_dtype = q.dtype if q.dtype != torch.float8_e4m3fn else torch.float16
    if out_dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("out_dtype must be float16 or bfloat16")
    if q.stride()[2] != 1:
        q = q.contiguous()
    if k_pool.stride()[3] != 1:
        k_pool = k_pool.contiguous()
    if v_pool.stride()[3] != 1:
        v_pool = v_pool.contiguous()
    if prefix_table.dim() != 1:
        raise ValueError("prefix_table must be [n]")
    prefix_table = _check_idx(prefix_table, "prefix_table", dev)
    host_len = 0
    if torch.is_tensor(prefix_len):
        if prefix_len.numel() != 1:
            raise ValueError("prefix_len must have one entry")
        prefix_len = _check_idx(prefix_len, "prefix_len", dev)
    else:
        host_len, prefix_len = int(prefix_len), None
        if host_len < 0 or host_len > 16 * prefix_table.shape[0]:
            raise ValueError("prefix_len must be 0 .. 16 * len(prefix_table)")
    if block_table.dim() != 2 or block_table.shape[0] < B:
        raise ValueError("block_table must be [B, max_blocks]")
    bt = block_table
    if bt.device != dev:
        raise ValueError("block_table must be on q's device")
    if bt.dtype != torch.int32 or (bt.stride()[1] != 1 and bt.shape[1] > 1):
        bt = bt.to(torch.int32).contiguous()
    lens = _check_idx(seq_lens, "seq_lens", dev)
    if lens.numel() < B:
        raise ValueError("seq_lens must have one entry per sequence")
    s_aux = _check_sink(s_aux, QH, dev)
    sq = _scale_ptr(scale_q, dev) if q.dtype == torch.float8_e4m3fn else None
    sk = _scale_ptr(scale_k, dev) if e4m3 else None
    sv = _scale_ptr(scale_v, dev) if e4m3 else None
    if out is None:
        if q.dtype == out_dtype:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)  # 1.4 us; empty 3.4
        else:
            out = torch.empty(B, QH, D, dtype=out_dtype, device=dev)
    elif out.shape != (B, QH, D) or out.dtype != out_dtype or out.stride(-1) != 1 or out.device != dev:
        raise ValueError("out must be [B, Q_H, D] of out_dtype on q's device with unit inner stride")
    _ops.shared_prefix(q, k_pool, v_pool, prefix_table, prefix_len, host_len, bt, lens, s_aux, sq, sk, sv, out)
    return out
