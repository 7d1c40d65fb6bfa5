"""Plain 64-bit references of the rotation, append and shared-prefix operators
(elementary torch ops, any device)."""
import math

import torch


def norm_rope_ref(x, cos, sin, pos, weight=None, eps=1e-6, interleaved=False):
    """(y, amp): the normed and rotated rows in 64 bits, and the size of the
    terms each output is a sum of (what 32-bit rounding errors scale with).
    x [T, H, D]; cos / sin [P, R/2] or None; pos [T]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    y, amp = x.clone(), x.abs()
    if cos is not None:
        c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
        half = c.shape[-1]
        ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
        ib = ia + (1 if interleaved else half)
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        amp = amp.clone()
        amp[..., ia] = amp[..., ib] = a.abs() + b.abs()
    return y, amp


def rounding_bound(ref, amp, dtype):
    """How far a value computed in 32 bits and rounded once may be from ref.
    The 32-bit part: a sum of 128 squares by 8 serial and 4 (3) tree additions
    (each at most 2^-24 of the sum, all terms positive; halved by the square
    root), rsqrt (2 ulp), two products, then two products and an addition: under
    32 roundings of 2^-24, each of at most amp."""
    d = 2.0 ** -19 * amp
    info = torch.finfo(dtype)
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float8_e4m3fn: 2.0 ** -10}[dtype]  # half a subnormal step
    return info.eps / 2 * (ref.abs() + d) + d + tiny


def shared_prefix_ref(q, kp, vp, prefix, kt, vt, lens, sink=None):
    """Decode attention over [prefix ; own tokens], 64 bits.  q [B, QH, D];
    kp / vp [KVH, P', D] (the first `prefix` rows count); kt / vt [B, KVH, T, D]
    (the first lens[b]).  A row with nothing to attend is zero."""
    B, QH, D = q.shape
    KVH = kp.shape[0]
    G = QH // KVH
    out = torch.zeros(B, QH, D, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lens[b])
        for h in range(KVH):
            k = torch.cat([kp[h, :prefix], kt[b, h, :n]]).double()
            v = torch.cat([vp[h, :prefix], vt[b, h, :n]]).double()
            if k.shape[0] == 0:
                continue
            x = q[b, h * G:(h + 1) * G].double() @ k.T / math.sqrt(D)
            if sink is not None:
                x = torch.cat([x, sink[h * G:(h + 1) * G, None].double()], 1)
            w = torch.softmax(x, -1)[:, :k.shape[0]]
            out[b, h * G:(h + 1) * G] = w @ v
    return out


def attention_bound(q, kp, vp, prefix, kt, vt, lens, sink, ref, p_dtype, out_dtype):
    """How far shared-prefix attention may be from ref, relative to sum w |v|.
    The softmax numerators are rounded to p_dtype (half a step each), the result
    to out_dtype.  In 32 bits: logits (2^-22 of sum |q k| / sqrt(D), which is
    under 64 in these tests: 2^-16), exponents (2^-24 of up to 64: 2^-18, times
    ln 2), ex2 (2^-22); the sum over P tokens 16 at a time (2^-24 a step), the
    numerators that vanish in f16 (under 2^-32 of the largest's for the prefix,
    2^-25 for own tokens)."""
    amp = shared_prefix_ref(q, kp, vp.abs(), prefix, kt, vt.abs(), lens, sink)
    u, uo = torch.finfo(p_dtype).eps / 2, torch.finfo(out_dtype).eps / 2
    tiny = 2.0 ** -25 if out_dtype == torch.float16 else 0.0
    own = kt.shape[2]
    f32 = 2.0 ** -15 + (prefix + own) / 16 * 2.0 ** -24 + prefix * 2.0 ** -32 + own * 2.0 ** -25
    return (u + f32) * amp * (1 + uo) + uo * ref.abs() + tiny
