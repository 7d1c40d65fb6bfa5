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


def _estimates(batch, prefix_len, own_len, q_heads, kv_heads, head_dim, e4m3):
    """(us of ``paged_flash_decode`` over the whole tables, us with the prefix
    shared), from what each spends its time on; the factors are fitted to the
    1170 sizes of ``shared_prefix_pays``.

    Whole tables: a launch, every sequence's elements, and the merge of an item's
    segments, short and many where sequences are few.  Items of four heads, and
    of query chunks, start at more.  Shared: three launches (the own part's is
    longer where tails fill a page at most, four of which go to one CTA); the own
    elements; an SM's share of the prefix in tiles, which starts late where the
    own part is on every SM; the join of a row's records."""
    sms = 148
    group = max(q_heads // kv_heads, 1)
    chunks = -(-group // 8)
    quads = e4m3 and kv_heads % 4 == 0 and 4 < group <= 8
    items = kv_heads * (chunks + 1) // 2 if chunks > 1 else kv_heads // (4 if quads else 1 + (kv_heads % 2 == 0))
    elements = 2e-6 * batch * kv_heads * head_dim  # one token of every sequence, in millions
    segments = min(2 * sms / (batch * items), (prefix_len + own_len) / 64)
    whole = ((25.5 if quads else 20.5 if chunks > 1 else 11.5 if head_dim > 64 else 10.5)
             + (0.2 if head_dim > 64 else 0.28) * elements * (prefix_len + own_len)
             + (0.5 if quads else 0.15 if e4m3 else 0.08) * segments)
    tiles, row_tiles = -(-prefix_len // 128), -(-batch * group // 128)
    pairs, odd = divmod(row_tiles, 2)
    granules = kv_heads * (pairs * tiles + odd * ((tiles + 1) // 2))
    share = -(-granules // sms)
    records = min(granules, sms) / (kv_heads * (pairs + odd)) * (2 if row_tiles == 1 else 1)
    busy = min(1.0, batch * items * ((own_len + 15) // 16) / (4 * sms))
    shared = (9.5 + (3 if chunks > 1 else 0) + (0 if own_len > 16 else 8.5 if chunks > 1 else 1.8)
              + 0.34 * elements * own_len + busy * (1.9 + 3.75 * min(share, 4))
              + (5 if e4m3 else 2.75) * share + 0.11 * records)
    return whole, shared


def shared_prefix_pays(batch: int, prefix_len: int, own_len: int = 64, *, q_heads: int = 32, kv_heads: int = 8,
                       head_dim: int = 128, kv_dtype=torch.float16) -> bool:
    """Whether reading a prefix once for the batch beats ``paged_flash_decode``
    over the whole tables, which reads it per sequence: ``own_len`` tokens of its
    own a sequence (the mean), heads and pools as given.

    Both were measured on the device at 1170 sizes: 1 to 8 KV heads, groups of 1
    to 16, head dims 64 and 128, f16 and e4m3 pools, 2 to 128 sequences, prefixes
    of 128 to 65536 tokens, tails up to 2000, pools past L2 where they can be.  At
    400 others (drawn of the same ranges) the rule takes a way that is over 10 %
    slower 21 times, 1.3 % on average; 4096 prefix tokens saved as the rule: 84
    times, 5.2 %.  In us, whole tables / shared, tails of 64: 8 KV heads, 32 query
    heads, f16: 2 x 1024 tokens 13.8 / 13.6, 2 x 16384 31.6 / 26.8, 16 x 2048 27.4 /
    16.7, 64 x 16384 523 / 48; e4m3 2 x 16384 28.2 / 30.5; head dim 64 2 x 4096 15.2 /
    15.9.  One KV head, 8 query heads: 4 x 16384 21.4 / 25.9.  Tails of 1000 want a
    longer prefix: 8 KV heads, f16, 4 x 4096 22.5 / 32.0, 16 x 4096 49.6 / 39.4."""
    if batch < 2 or prefix_len <= 0:
        return False
    whole, shared = _estimates(batch, prefix_len, own_len, q_heads, kv_heads, head_dim, kv_dtype == torch.float8_e4m3fn)
    return shared < whole


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
