"""Paged KV append with the position rotation (and per-head norms) on the way.

``paged_kv_append_rope`` does in one kernel what a layer does between its q / k
/ v projection and ``paged_flash_decode``: norm and rotate q and k, write the
rotated k and the v of every token into their pages (quantised for e4m3 pools),
return the rotated q.  It takes one token per sequence (a decode step) or any
number (prompt chunks), reads positions on the device and is CUDA-graph
capturable, as ``paged_kv_append``.
"""
from __future__ import annotations

import torch

from .. import _native as N
from .. import _ops
from ..gqa_decode import _check_idx
from ..gqa_decode_hf import _scale_ptr
from ..qk_norm_rope import _check_heads, _check_no_grad, _check_out, _check_status, _check_table, _check_weight


def paged_kv_append_rope(q, k, v, k_pool, v_pool, block_table, positions, cos, sin, *, seq_ids=None, q_weight=None,
                         k_weight=None, eps: float = 1e-6, interleaved: bool = False, scale_k=None, scale_v=None,
                         q_out=None, k_out=None, status=None):
    """q [T, Q_H, D], k / v [T, KV_H, D] float16/bfloat16 (a decode step's
    [B, H, 1, D] too); pools [num_pages, KV_H, 16, D] of the same dtype or
    float8_e4m3fn (then ``scale_k`` / ``scale_v``); block_table [B, max_blocks]
    int32; positions [T] int32; ``seq_ids`` [T] int32 names each token's
    block-table row (default: token t is row t).  cos, sin, the norm weights,
    ``eps`` and ``interleaved`` as in ``qk_norm_rope``.

    The rotated k and v as it is go to slot ``positions[t] % 16`` of page
    ``block_table[seq, positions[t] // 16]``; no two tokens of a call may share a
    slot.  ``k_out`` also gets the rotated k (a prompt's attention reads it).
    A position outside the tables (FK_STATUS_BAD_POSITION: rows zeroed) or a page
    outside the pool (FK_STATUS_BAD_PAGE) appends nothing and sets the bit in
    ``status``, if given.  Returns the rotated q [T, Q_H, D]."""
    if q.dim() == 4 and k.dim() == 4 and v.dim() == 4 and q.shape[2] == k.shape[2] == v.shape[2] == 1:
        q, k, v = q.squeeze(2), k.squeeze(2), v.squeeze(2)
    T, D, dev = _check_heads(q, k, "paged_kv_append_rope")
    shape, dt = k.shape, k.dtype
    if v.shape != shape or v.dtype != dt or v.device != dev:
        raise ValueError("v must match k in shape, dtype and device")
    _check_no_grad("paged_kv_append_rope", q, k, v, q_weight, k_weight)
    pool, pdt = k_pool.shape, k_pool.dtype
    if len(pool) != 4 or pool != v_pool.shape or pool[1] != shape[1] or pool[2] != 16 or pool[3] != D:
        raise ValueError("pools must be [num_pages, KV_H, 16, D] with the heads and head dim of k")
    if v_pool.dtype != pdt or k_pool.device != dev or v_pool.device != dev:
        raise ValueError("the pools must have one dtype and be on q's device")
    if k_pool.stride()[3] != 1 or v_pool.stride()[3] != 1:
        raise ValueError("the pools must have unit inner stride")
    pool_code = N.dtype_code(pdt)
    if pool_code != N.FK_DTYPE_E4M3 and pdt != dt:
        raise TypeError("a 16-bit pool must have the dtype of k and v")
    bt = block_table
    if bt.dim() != 2 or bt.device != dev:
        raise ValueError("block_table must be [B, max_blocks] on q's device")
    if bt.dtype != torch.int32 or bt.stride()[1] != 1:
        bt = bt.to(torch.int32).contiguous()
    positions = _check_idx(positions, "positions", dev)
    if seq_ids is not None:
        seq_ids = _check_idx(seq_ids, "seq_ids", dev)
        if seq_ids.numel() != T:
            raise ValueError("seq_ids must have one entry per token")
    elif bt.shape[0] < T:
        raise ValueError("block_table must have a row per token (or pass seq_ids)")
    if positions.numel() != T:
        raise ValueError("positions must have one entry per token")
    _check_table(cos, sin, D, dev)
    q_weight = _check_weight(q_weight, "q_weight", D, dev)
    k_weight = _check_weight(k_weight, "k_weight", D, dev)
    sk = sv = None
    if pool_code == N.FK_DTYPE_E4M3:
        if scale_k is None or scale_v is None:
            raise ValueError("an e4m3 pool needs scale_k and scale_v")
        sk, sv = _scale_ptr(scale_k, dev), _scale_ptr(scale_v, dev)
    q_out = _check_out(q_out, q, "q_out")
    if k_out is not None:
        k_out = _check_out(k_out, k, "k_out")
    _check_status(status, dev)
    _ops.rope(q, k, v, cos, sin, positions, seq_ids, bt, q_weight, k_weight, float(eps), bool(interleaved), sk, sv, q_out, k_out,
              k_pool, v_pool, status)
    return q_out
