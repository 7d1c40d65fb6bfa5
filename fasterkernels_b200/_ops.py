"""The C-ABI launches of the decode entry points, and their registration as
``torch.library`` custom ops so that ``torch.compile`` traces a model through
them without a graph break.

The reference's entry points are user Triton kernels, which ``torch.compile``
traces (fskernels/triton/triton_gqa_decode.py:126-155); a ``ctypes`` call is
opaque to it.  Each launcher below takes checked, laid-out tensors and writes
``out`` (declared as mutated; the fake implementation does nothing, since the
output is preallocated by the caller).  Eager calls go straight to the
launcher (no dispatcher overhead on the hot path); calls made while
``torch.compile`` is tracing go through ``torch.ops.fasterkernels_b200.*``.
Both run the same kernel with the same arguments, so the results are
bit-identical.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _native as N


def _scale(x):
    return N.ptr(x) if x is not None else None


# ---------------------------------------------------------------- launchers
def varlen_launch(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, s_aux: Optional[torch.Tensor],
                  out: torch.Tensor) -> None:
    dev = q.device
    B, QH, D = q.shape
    T, KVH, _ = k.shape
    code = N.dtype_code(q.dtype)
    ws = N.workspace(dev, B, QH, KVH, code)
    rc = N.lib().fk_flash_decode_gqa_varlen(
        N.ptr(q), N.ptr(k), N.ptr(v), N.ptr(cu), N.ptr(s_aux), N.ptr(out),
        B, QH, KVH, D, T, code,
        q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0), out.stride(1),
        N.ptr(ws), ws.numel(), N.stream_of(dev))
    N.check(rc, "fk_flash_decode_gqa_varlen")


def dense_launch(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                 starts: Optional[torch.Tensor], s_aux: Optional[torch.Tensor], scale_q: Optional[torch.Tensor],
                 scale_k: Optional[torch.Tensor], scale_v: Optional[torch.Tensor], out: torch.Tensor) -> None:
    dev = q.device
    B, QH, D = q.shape
    _, KVH, S, _ = k_cache.shape
    kv_code = N.dtype_code(k_cache.dtype)
    ws = N.workspace(dev, B, QH, KVH, kv_code)
    rc = N.lib().fk_flash_decode_gqa_hf_dense(
        N.ptr(q), N.ptr(k_cache), N.ptr(v_cache), N.ptr(lens), N.ptr(starts), N.ptr(s_aux), N.ptr(out),
        B, QH, KVH, D, S, N.dtype_code(q.dtype), kv_code, N.dtype_code(out.dtype),
        _scale(scale_q), _scale(scale_k), _scale(scale_v),
        q.stride(0), q.stride(1), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
        v_cache.stride(0), v_cache.stride(1), v_cache.stride(2), out.stride(0), out.stride(1),
        N.ptr(ws), ws.numel(), N.stream_of(dev))
    N.check(rc, "fk_flash_decode_gqa_hf_dense")


def paged_launch(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, bt: torch.Tensor, lens: torch.Tensor,
                 s_aux: Optional[torch.Tensor], scale_q: Optional[torch.Tensor], scale_k: Optional[torch.Tensor],
                 scale_v: Optional[torch.Tensor], out: torch.Tensor) -> None:
    dev = q.device
    B, QH, D = q.shape
    P, KVH, PS, _ = k_pool.shape
    kv_code = N.dtype_code(k_pool.dtype)
    ws = N.workspace(dev, B, QH, KVH, kv_code)
    rc = N.lib().fk_paged_flash_decode(
        N.ptr(q), N.ptr(k_pool), N.ptr(v_pool), N.ptr(bt), N.ptr(lens), N.ptr(s_aux), N.ptr(out),
        B, QH, KVH, D, P, PS, bt.shape[1], N.dtype_code(q.dtype), kv_code, N.dtype_code(out.dtype),
        _scale(scale_q), _scale(scale_k), _scale(scale_v),
        q.stride(0), q.stride(1), k_pool.stride(0), k_pool.stride(1), k_pool.stride(2),
        v_pool.stride(0), v_pool.stride(1), v_pool.stride(2), bt.stride(0), out.stride(0), out.stride(1),
        N.ptr(ws), ws.numel(), N.stream_of(dev))
    N.check(rc, "fk_paged_flash_decode")


def append_launch(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                  bt: torch.Tensor, positions: torch.Tensor, increment: bool, scale_k: Optional[torch.Tensor],
                  scale_v: Optional[torch.Tensor], status: Optional[torch.Tensor]) -> None:
    B, KVH, D = k_new.shape
    rc = N.lib().fk_paged_kv_append(
        N.ptr(k_new), N.ptr(v_new), N.dtype_code(k_new.dtype), N.ptr(k_pool), N.ptr(v_pool),
        N.dtype_code(k_pool.dtype), N.ptr(bt), N.ptr(positions), 1 if increment else 0, _scale(scale_k),
        _scale(scale_v), N.ptr(status), B, KVH, D, k_pool.shape[0], bt.shape[1], k_new.stride(0), k_new.stride(1),
        v_new.stride(0), v_new.stride(1), k_pool.stride(0), k_pool.stride(1), k_pool.stride(2), v_pool.stride(0),
        v_pool.stride(1), v_pool.stride(2), bt.stride(0), N.stream_of(k_new.device))
    N.check(rc, "fk_paged_kv_append")


_ROPE_ARGS = struct.Struct("17Q34qd")  # fk_rope_args of include/fk_decode.h
_WIDE_CODES = {torch.float16: N.FK_DTYPE_F16, torch.bfloat16: N.FK_DTYPE_BF16, torch.float32: N.FK_DTYPE_F32}


def _addr(t):
    return 0 if t is None else t.data_ptr()


def _rows16(t):
    """t, or a copy whose rows start on 16-byte boundaries."""
    if t is None:
        return None
    e = t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * e % 16 == 0 for s in t.stride()[:-1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def rope_launch(q: torch.Tensor, k: torch.Tensor, v: Optional[torch.Tensor], cos: Optional[torch.Tensor],
                sin: Optional[torch.Tensor], positions: Optional[torch.Tensor], seq_ids: Optional[torch.Tensor],
                bt: Optional[torch.Tensor], q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                eps: float, interleaved: bool, scale_k: Optional[torch.Tensor], scale_v: Optional[torch.Tensor],
                q_out: torch.Tensor, k_out: Optional[torch.Tensor], k_pool: Optional[torch.Tensor],
                v_pool: Optional[torch.Tensor], status: Optional[torch.Tensor]) -> None:
    T, QH, D = q.shape
    if T == 0:
        return
    _, KH, _ = k.shape
    q_t, q_h, q_d = q.stride()
    k_t, k_h, k_d = k.stride()
    qo_t, qo_h, _ = q_out.stride()
    ko_t = ko_h = R = max_pos = cos_row = sin_row = table = 0
    inner = q_d == 1 == k_d
    if k_out is not None:
        ko_t, ko_h, _ = k_out.stride()
    if cos is not None:
        (max_pos, R), table = cos.shape, _WIDE_CODES[cos.dtype]
        cos_row, c_d = cos.stride()
        sin_row, s_d = sin.stride()
        inner = inner and c_d == 1 == s_d
    v_t = v_h = kp_p = kp_h = kp_s = vp_p = vp_h = vp_s = pool_code = bt_b = bt_rows = blocks = pages = 0
    if k_pool is not None:
        v_t, v_h, v_d = v.stride()
        inner = inner and v_d == 1
        kp_p, kp_h, kp_s, _ = k_pool.stride()
        vp_p, vp_h, vp_s, _ = v_pool.stride()
        pool_code, pages = N.dtype_code(k_pool.dtype), k_pool.shape[0]
        bt_rows, blocks = bt.shape
        bt_b, _ = bt.stride()
    qw = kw = 0
    if q_weight is not None:
        qw = _WIDE_CODES[q_weight.dtype]
    if k_weight is not None:
        kw = _WIDE_CODES[k_weight.dtype]
    if inner:
        args = _ROPE_ARGS.pack(
            *[0 if t is None else t.data_ptr()
              for t in (q, k, v, q_out, k_out, k_pool, v_pool, cos, sin, positions, seq_ids, bt, q_weight, k_weight, scale_k,
                        scale_v, status)], q_t, q_h, k_t, k_h, v_t, v_h, qo_t, qo_h, ko_t, ko_h, kp_p, kp_h, kp_s, vp_p, vp_h,
            vp_s, cos_row, sin_row, bt_b, T, QH, KH, D, 2 * R, interleaved, max_pos, bt_rows, blocks, pages,
            N.dtype_code(q.dtype), pool_code, table, qw, kw, eps)
        rc = N.lib().fk_qk_norm_rope(args, N.raw_stream(q.device.index))
        if rc == 0:
            return
    # rows the kernel cannot read in 16-byte pieces: copies of those inputs
    ins = (q, k, v, cos, sin, q_weight, k_weight)
    fit = tuple(_rows16(t) for t in ins)
    if all(a is b for a, b in zip(ins, fit)):
        N.check(rc, "fk_qk_norm_rope")
    q, k, v, cos, sin, q_weight, k_weight = fit
    rope_launch(q, k, v, cos, sin, positions, seq_ids, bt, q_weight, k_weight, eps, interleaved, scale_k, scale_v, q_out,
                k_out, k_pool, v_pool, status)


_PREFIX_ARGS = struct.Struct("13Q22q")  # fk_prefix_args of include/fk_decode.h
_prefix_ws = {}


def shared_prefix_launch(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, prefix_table: torch.Tensor,
                         prefix_len: Optional[torch.Tensor], prefix_len_host: int, bt: torch.Tensor, lens: torch.Tensor,
                         s_aux: Optional[torch.Tensor], scale_q: Optional[torch.Tensor],
                         scale_k: Optional[torch.Tensor], scale_v: Optional[torch.Tensor], out: torch.Tensor) -> None:
    dev = q.device
    B, QH, D = q.shape
    if B == 0:
        return
    P, KVH, _, _ = k_pool.shape
    kv_code = N.dtype_code(k_pool.dtype)
    lib = N.lib()
    key = (dev.index, B, QH, KVH, D, kv_code)
    status = N.status_word(dev)
    like = _prefix_ws.get(key)
    if like is None:
        need = int(lib.fk_shared_prefix_workspace_bytes(*key))
        if need == 0:
            raise RuntimeError(f"fk_shared_prefix_workspace_bytes failed: {N.last_error()}")
        # a view without memory of its own: empty_like of it takes 1.4 us, empty 3.4
        like = _prefix_ws[key] = status.view(torch.uint8)[:1].expand(need)
    # scratch of this call alone (torch's allocator reuses it in stream order;
    # in a captured graph it belongs to the graph's pool), so calls on other
    # streams and other graphs never share it
    ws = torch.empty_like(like, memory_format=torch.contiguous_format)
    qs, ks, vs, os = q.stride(), k_pool.stride(), v_pool.stride(), out.stride()
    args = _PREFIX_ARGS.pack(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), prefix_table.data_ptr(), _addr(prefix_len), bt.data_ptr(),
        lens.data_ptr(), _addr(s_aux), out.data_ptr(), _addr(scale_q), _addr(scale_k), _addr(scale_v), status.data_ptr(),
        prefix_len_host, prefix_table.shape[0], B, QH, KVH, D, P, bt.shape[1], N.dtype_code(q.dtype), kv_code,
        N.dtype_code(out.dtype), qs[0], qs[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], bt.stride()[0], os[0], os[1])
    N.check(lib.fk_paged_shared_prefix_decode(args, ws.data_ptr(), ws.numel(), N.raw_stream(dev.index)),
            "fk_paged_shared_prefix_decode")


# ---------------------------------------------------------------- custom ops
_LIB = "fasterkernels_b200"


@torch.library.custom_op(f"{_LIB}::varlen_decode", mutates_args=("out",), device_types="cuda")
def _varlen_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, s_aux: Optional[torch.Tensor],
               out: torch.Tensor) -> None:
    varlen_launch(q, k, v, cu, s_aux, out)


@torch.library.custom_op(f"{_LIB}::dense_decode", mutates_args=("out",), device_types="cuda")
def _dense_op(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
              starts: Optional[torch.Tensor], s_aux: Optional[torch.Tensor], scale_q: Optional[torch.Tensor],
              scale_k: Optional[torch.Tensor], scale_v: Optional[torch.Tensor], out: torch.Tensor) -> None:
    dense_launch(q, k_cache, v_cache, lens, starts, s_aux, scale_q, scale_k, scale_v, out)


@torch.library.custom_op(f"{_LIB}::paged_decode", mutates_args=("out",), device_types="cuda")
def _paged_op(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, bt: torch.Tensor, lens: torch.Tensor,
              s_aux: Optional[torch.Tensor], scale_q: Optional[torch.Tensor], scale_k: Optional[torch.Tensor],
              scale_v: Optional[torch.Tensor], out: torch.Tensor) -> None:
    paged_launch(q, k_pool, v_pool, bt, lens, s_aux, scale_q, scale_k, scale_v, out)


@torch.library.custom_op(f"{_LIB}::paged_kv_append", mutates_args=("k_pool", "v_pool", "positions", "status"),
                         device_types="cuda")
def _append_op(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
               bt: torch.Tensor, positions: torch.Tensor, increment: bool, scale_k: Optional[torch.Tensor],
               scale_v: Optional[torch.Tensor], status: Optional[torch.Tensor]) -> None:
    append_launch(k_new, v_new, k_pool, v_pool, bt, positions, increment, scale_k, scale_v, status)


@torch.library.custom_op(f"{_LIB}::qk_norm_rope", mutates_args=("q_out", "k_out", "k_pool", "v_pool", "status"),
                         device_types="cuda")
def _rope_op(q: torch.Tensor, k: torch.Tensor, v: Optional[torch.Tensor], cos: Optional[torch.Tensor],
             sin: Optional[torch.Tensor], positions: Optional[torch.Tensor], seq_ids: Optional[torch.Tensor],
             bt: Optional[torch.Tensor], q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
             eps: float, interleaved: bool, scale_k: Optional[torch.Tensor], scale_v: Optional[torch.Tensor],
             q_out: torch.Tensor, k_out: Optional[torch.Tensor], k_pool: Optional[torch.Tensor],
             v_pool: Optional[torch.Tensor], status: Optional[torch.Tensor]) -> None:
    rope_launch(q, k, v, cos, sin, positions, seq_ids, bt, q_weight, k_weight, eps, interleaved, scale_k, scale_v,
                q_out, k_out, k_pool, v_pool, status)


@torch.library.custom_op(f"{_LIB}::shared_prefix_decode", mutates_args=("out",), device_types="cuda")
def _shared_prefix_op(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, prefix_table: torch.Tensor,
                      prefix_len: Optional[torch.Tensor], prefix_len_host: int, bt: torch.Tensor, lens: torch.Tensor,
                      s_aux: Optional[torch.Tensor], scale_q: Optional[torch.Tensor], scale_k: Optional[torch.Tensor],
                      scale_v: Optional[torch.Tensor], out: torch.Tensor) -> None:
    shared_prefix_launch(q, k_pool, v_pool, prefix_table, prefix_len, prefix_len_host, bt, lens, s_aux, scale_q, scale_k,
                         scale_v, out)


# The outputs are preallocated by the callers, so the fake (meta)
# implementations have nothing to compute.
for _op in (_varlen_op, _dense_op, _paged_op, _append_op, _rope_op, _shared_prefix_op):
    _op.register_fake(lambda *args, **kwargs: None)


def _dispatch(op, launch):
    def call(*args):
        if torch.compiler.is_compiling():
            return op(*args)
        return launch(*args)
    return call


varlen = _dispatch(_varlen_op, varlen_launch)
dense = _dispatch(_dense_op, dense_launch)
paged = _dispatch(_paged_op, paged_launch)
append = _dispatch(_append_op, append_launch)
rope = _dispatch(_rope_op, rope_launch)
shared_prefix = _dispatch(_shared_prefix_op, shared_prefix_launch)
