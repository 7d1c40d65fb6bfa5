"""Per-head norms and position rotation of queries and keys in one kernel.

What a layer does to q and k between its projections and the decode call: an
RMS norm over each head's dims (optional) and the rotation of the first
``2 * cos.shape[-1]`` dims by the angles of the token's position.  The
reference leaves both to the model's separate torch ops.  Computed in 32 bits,
rounded once.  Forward only: inputs that require grad are refused.
"""
from __future__ import annotations

import torch

from . import _native as N  # noqa: F401  (loads the library on first use)
from . import _ops
from .gqa_decode import HEAD_DIMS, _check_idx

_HALF = (torch.float16, torch.bfloat16)
_TABLE = (torch.float16, torch.bfloat16, torch.float32)


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0, *, inv_freq=None, device="cuda"):
    """(cos, sin), float32 [max_positions, rotary_dim / 2]: row p holds the
    angles p * base ** (-2 i / rotary_dim) (or p * inv_freq[i]).  The angles are
    made in 64 bits: in 32 a far position's angle has no fraction left."""
    if rotary_dim <= 0 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a positive multiple of 16")
    if inv_freq is None:
        i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
        inv_freq = float(base) ** (-2.0 * i / rotary_dim)
    elif inv_freq.numel() != rotary_dim // 2:
        raise ValueError("inv_freq must have rotary_dim / 2 entries")
    ang = torch.arange(int(max_positions), dtype=torch.float64, device=device)[:, None] * \
        inv_freq.to(device=device, dtype=torch.float64)
    return ang.cos().float(), ang.sin().float()


def _check_heads(q, k, name):
    """(tokens, head dim, device) of q and k, checked."""
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be [T, Q_H, D] and [T, KV_H, D]")
    if not q.is_cuda:
        raise ValueError(f"{name} runs on CUDA tensors only")
    dev, dt = q.device, q.dtype
    if k.device != dev:
        raise ValueError("q and k must be on the same device")
    if dt not in _HALF or k.dtype != dt:
        raise TypeError("q and k must both be float16 or bfloat16")
    T, QH, D = q.shape
    Tk, KH, Dk = k.shape
    if Tk != T or Dk != D:
        raise ValueError("q and k must have the same tokens and head dim")
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
    if QH == 0 or KH == 0:
        raise ValueError("q and k must have heads")
    return T, D, dev


def _check_no_grad(name, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no backward pass; call it under torch.no_grad()")


def _check_table(cos, sin, D, dev):
    """The rotated dims (0: no rotation)."""
    if cos is None or sin is None:
        if cos is not None or sin is not None:
            raise ValueError("cos and sin go together")
        return 0
    dt, shape = cos.dtype, cos.shape
    if len(shape) != 2 or sin.shape != shape or sin.dtype != dt or dt not in _TABLE:
        raise ValueError("cos and sin must be [max_positions, rotary_dim / 2] of one type: float32, float16 or bfloat16")
    if cos.device != dev or sin.device != dev:
        raise ValueError("cos and sin must be on q's device")
    R = 2 * shape[1]
    if R == 0 or R > D or R % 16:
        raise ValueError("rotary_dim (2 * cos.shape[1]) must be a multiple of 16 up to the head dim")
    if shape[0] == 0:
        raise ValueError("the cos / sin tables must have rows")
    return R


def _check_weight(w, name, D, dev):
    """w as the kernel reads it, its D entries one after another."""
    if w is None:
        return None
    if w.device != dev or w.numel() != D or w.dtype not in _TABLE:
        raise ValueError(f"{name} must have head_dim entries (float32, float16 or bfloat16) on q's device")
    return w if w.is_contiguous() else w.contiguous()


def _check_out(out, like, name):
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)  # 1.4 us; new_empty 2.4, empty 3.4
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or out.stride(-1) != 1:
        raise ValueError(f"{name} must have the shape, dtype and device of its input, with unit inner stride")
    return out


def _check_status(status, dev):
    if status is not None and (status.dtype != torch.int32 or status.device != dev or status.numel() < 1):
        raise ValueError("status must be an int32 tensor on q's device")


def qk_norm_rope(q, k, cos, sin, positions=None, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                 interleaved: bool = False, q_out=None, k_out=None, status=None):
    """Norm and rotate each head of q [T, Q_H, D] and k [T, KV_H, D] (float16 or
    bfloat16, D = 128 or 64; slices of a packed projection are fine).

    cos / sin [max_positions, R / 2] (float32, float16 or bfloat16) rotate the
    first R dims (a multiple of 16) by row ``positions[t]``; pairs are dims
    (i, i + R / 2), or (2 i, 2 i + 1) when ``interleaved``.  ``cos = sin = None``
    norms only.  Without ``positions`` token t takes row t % max_positions (the
    tables hold the tokens' own rows).  ``q_weight`` / ``k_weight`` [D] apply
    ``x * rsqrt(mean(x^2) + eps) * weight`` first.  ``q_out`` / ``k_out`` may be
    q / k themselves.

    A position outside the tables zeroes the token's rows and sets
    FK_STATUS_BAD_POSITION in ``status`` (an int32 device tensor), if given.
    Returns (q_out, k_out)."""
    T, D, dev = _check_heads(q, k, "qk_norm_rope")
    _check_no_grad("qk_norm_rope", q, k, q_weight, k_weight)
    R = _check_table(cos, sin, D, dev)
    if positions is not None:
        positions = _check_idx(positions, "positions", dev)
        if positions.numel() != T:
            raise ValueError("positions must have one entry per token")
    elif R == 0:
        positions = torch.zeros(T, dtype=torch.int32, device=dev)
    q_weight = _check_weight(q_weight, "q_weight", D, dev)
    k_weight = _check_weight(k_weight, "k_weight", D, dev)
    q_out = _check_out(q_out, q, "q_out")
    k_out = _check_out(k_out, k, "k_out")
    _check_status(status, dev)
    _ops.rope(q, k, None, cos, sin, positions, None, None, q_weight, k_weight, float(eps), bool(interleaved), None, None,
              q_out, k_out, None, None, status)
    return q_out, k_out


def _angles_once(t, tables):
    """Each angle of an HF table [.., columns] once: [.., R / 2]."""
    return t[..., : t.shape[-1] // 2] if tables == "halves" else t[..., ::2].contiguous() if tables == "pairs" else t


def _hf_tables(cos, D, tables, interleaved):
    """How the tables of an HF model hold their angles, where ``tables`` and the
    number of columns say it; refused where they do not."""
    cols = cos.shape[-1]
    if tables not in (None, "halves", "pairs", "once"):
        raise ValueError("tables must be 'halves', 'pairs' or 'once'")
    if tables is None:
        if interleaved:
            raise ValueError("interleaved pairs come with tables='pairs' (each angle twice, side by side) or 'halves'")
        if 2 * cols == D:
            raise ValueError("cos / sin of head_dim / 2 columns are all angles once (tables='once') or a rotation of half "
                             "the dims (tables='halves'): pass tables")
        tables = "halves"
    R = 2 * cols if tables == "once" else cols
    if R == 0 or R > D or R % 16:
        raise ValueError(f"cos / sin of {cols} columns rotate {R} of {D} dims: must be a multiple of 16 up to the head dim")
    return tables


def custom_hf_apply_rotary_pos_emb(q, k, cos, sin, unsqueeze_dim: int = 1, *, tables=None, interleaved: bool = False,
                                   **kwargs):
    """Drop-in for the ``apply_rotary_pos_emb`` of transformers' model files, the
    way ``custom_hf_decode_attention_forward`` stands in for their attention:
    q [B, Q_H, S, D], k [B, KV_H, S, D] (``unsqueeze_dim=2``: heads after S),
    cos / sin [B or 1, S, columns].  Both are rotated by one kernel; returned in
    the layout they came in.

    As it is, it stands in for the function of Llama, Qwen, Mistral and most
    others: half-split pairs, the angles repeated in the second half of the
    columns, one column per rotated dim.  Model files that pair or hold them
    otherwise have the same signature, so these two say which, bound with
    ``functools.partial``: ``interleaved`` rotates dims (2 i, 2 i + 1);
    ``tables`` says how the columns hold the angles, "halves" (a, b, a, b), "pairs"
    (a, a, b, b) or "once" (a, b).  GPT-OSS: tables="once".  Cohere:
    interleaved=True, tables="pairs".  Ernie 4.5, GLM, Helium: interleaved=True,
    tables="halves".  GLM-4 MoE (half of the dims rotated): tables="halves".
    Tables of head_dim / 2 columns are refused without ``tables``."""
    if q.dim() != 4 or k.dim() != 4 or cos.dim() != 3 or unsqueeze_dim not in (1, 2):
        raise ValueError("q, k must be 4-D, cos / sin [B, S, R], unsqueeze_dim 1 or 2")
    if unsqueeze_dim == 1:
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    B, S = q.shape[:2]
    if cos.shape[1] != S or cos.shape[0] not in (1, B) or sin.shape != cos.shape:
        raise ValueError("cos / sin must have q's sequence length and its batch (or 1)")
    tables = _hf_tables(cos, q.shape[-1], tables, interleaved)
    cos, sin = (_angles_once(t.reshape(-1, t.shape[-1]), tables) for t in (cos, sin))
    if cos.dtype not in _TABLE:
        cos, sin = cos.float(), sin.float()
    qo, ko = qk_norm_rope(q.reshape(B * S, *q.shape[2:]), k.reshape(B * S, *k.shape[2:]), cos, sin,
                          interleaved=interleaved)
    qo, ko = qo.view(q.shape), ko.view(k.shape)
    return (qo.transpose(1, 2), ko.transpose(1, 2)) if unsqueeze_dim == 1 else (qo, ko)
