"""qk_norm_rope and paged_kv_append_rope: against 64-bit references, their
refusals, graphs, streams and device-side conditions."""
import struct

import pytest
import torch

import fasterkernels_b200 as fk
from fasterkernels_b200 import _native as N
from fasterkernels_b200.paged_attn import paged_kv_append
from _operator_refs import norm_rope_ref, rounding_bound

gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------ CPU: host logic and refusals
def test_rope_table_angles_are_exact_at_far_positions():
    cos, sin = fk.rope_table(1_000_001, 16, base=1e6, device="cpu")
    assert cos.shape == sin.shape == (1_000_001, 8) and cos.dtype == torch.float32
    import math
    for i in range(8):
        a = 1_000_000 * 1e6 ** (-i / 8)
        assert abs(float(cos[1_000_000, i]) - math.cos(a)) < 2 ** -22
        assert abs(float(sin[1_000_000, i]) - math.sin(a)) < 2 ** -22
    c2, _ = fk.rope_table(5, 32, inv_freq=torch.ones(16), device="cpu")
    assert torch.allclose(c2[:, 3], torch.cos(torch.arange(5.0)))
    for bad in (0, 24, -16):
        with pytest.raises(ValueError, match="rotary_dim"):
            fk.rope_table(4, bad, device="cpu")
    with pytest.raises(ValueError, match="inv_freq"):
        fk.rope_table(4, 32, inv_freq=torch.ones(15), device="cpu")


def test_wrappers_refuse_cpu_tensors_and_wrong_ranks():
    q, k = torch.zeros(2, 4, 128, dtype=torch.float16), torch.zeros(2, 2, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        fk.qk_norm_rope(q, k, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        fk.paged_kv_append_rope(q, k, k, k, k, k, k, None, None)
    with pytest.raises(ValueError, match="T, Q_H, D"):
        fk.qk_norm_rope(q[0], k, None, None)
    with pytest.raises(ValueError, match="4-D"):
        fk.custom_hf_apply_rotary_pos_emb(q, k, q, q)


_FIELDS = ("q k v q_out k_out k_pool v_pool cos sin positions seq_ids block_table q_weight k_weight scale_k scale_v status "
           "q_t q_h k_t k_h v_t v_h qo_t qo_h ko_t ko_h kp_p kp_h kp_s vp_p vp_h vp_s cos_row sin_row bt_b "
           "tokens q_heads kv_heads head_dim rotary_dim interleaved max_pos table_rows max_blocks num_pages "
           "dtype pool_dtype table_dtype q_weight_dtype k_weight_dtype eps").split()


def _args(**kw):
    a = dict.fromkeys(_FIELDS, 0)
    a.update(q=16, k=16, q_out=16, k_out=16, cos=16, sin=16, positions=16, tokens=1, q_heads=2, kv_heads=1, head_dim=128,
             rotary_dim=128, max_pos=4, table_dtype=3, cos_row=64, sin_row=64, eps=0.0)
    a.update(kw)
    return struct.pack("17Q34qd", *(a[f] for f in _FIELDS))


@pytest.mark.parametrize("kw, rc, msg", [
    (dict(q=0), 1, "non-null"),
    (dict(head_dim=96), 2, "head_dim"),
    (dict(q_heads=0), 1, "bad sizes"),
    (dict(tokens=-1), 1, "bad sizes"),
    (dict(dtype=2), 2, "f16 or bf16"),
    (dict(rotary_dim=24), 2, "rotary_dim"),
    (dict(rotary_dim=144), 2, "rotary_dim"),
    (dict(cos=0), 1, "cos and sin"),
    (dict(max_pos=0), 1, "rows"),
    (dict(table_dtype=2), 2, "f32, f16 or bf16"),
    (dict(cos=20), 1, "aligned"),
    (dict(sin_row=66), 1, "aligned"),
    (dict(positions=0, rotary_dim=0), 1, "positions"),
    (dict(q_weight=16, q_weight_dtype=2), 2, "weights"),
    (dict(k_weight=8, k_weight_dtype=3), 1, "weights"),
    (dict(q_h=12), 1, "multiples of 16"),
    (dict(q=18), 1, "16-byte aligned"),
    (dict(k_out=0), 1, "k_out"),
    (dict(k_pool=16), 1, "v, v_pool"),
    (dict(k_pool=16, v_pool=16, v=16, block_table=16, positions=0), 1, "positions"),
    (dict(k_pool=16, v_pool=16, v=16, block_table=16, num_pages=0), 1, "pool sizes"),
    (dict(k_pool=16, v_pool=16, v=16, block_table=16, num_pages=1, pool_dtype=1), 1, "16-bit pool"),
    (dict(k_pool=16, v_pool=16, v=16, block_table=16, num_pages=1, pool_dtype=2, kp_s=8), 1, "multiples of 16"),
    (dict(k_pool=16, v_pool=24, v=16, block_table=16, num_pages=1), 1, "16-byte aligned"),
])
def test_c_entry_refuses_bad_arguments_without_a_device(kw, rc, msg):
    assert N.lib().fk_qk_norm_rope(_args(**kw), None) == rc
    assert msg in N.last_error()


def test_c_entry_takes_an_empty_call():
    assert N.lib().fk_qk_norm_rope(_args(tokens=0, q=0), None) == 0
    assert N.lib().fk_qk_norm_rope(None, None) == 1


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _heads(dev, T, QH, KVH, D, dtype, seed, packed=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (1.5 * torch.randn(T, QH + 2 * KVH, D, generator=g, device=dev)).to(dtype)
    q, k, v = x[:, :QH], x[:, QH:QH + KVH], x[:, QH + KVH:]
    return (q, k, v) if packed else (q.contiguous(), k.contiguous(), v.contiguous())


def _weights(dev, D, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(1000 + seed)
    return [(1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(dtype) for _ in range(2)]


def _inside(got, ref, amp):
    err = (got.double() - ref).abs()
    bound = rounding_bound(ref, amp, got.dtype)
    assert bool((err <= bound).all()), float((err / bound).max())


@gpu
@pytest.mark.parametrize("D,R,il", [(128, 128, False), (128, 128, True), (128, 96, False), (128, 16, False), (64, 64, False),
                                    (64, 32, True), (64, 48, False), (128, 0, False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,QH,KVH,norm", [(1, 1, 1, True), (7, 32, 8, True), (511, 5, 1, False), (513, 71, 3, True),
                                            (1023, 4, 2, True), (1024, 4, 2, True), (2777, 9, 3, True), (1500, 3, 1, False)])
def test_norm_rope_matches_reference(dev, D, R, il, dtype, T, QH, KVH, norm):
    q, k, _ = _heads(dev, T, QH, KVH, D, dtype, seed=T + D + R)
    qw, kw = _weights(dev, D, dtype, T) if norm else (None, None)
    cos, sin = fk.rope_table(5000, R, device=dev) if R else (None, None)
    pos = torch.randint(0, 5000, (T,), device=dev, dtype=torch.int32)
    pos[0] = 4999
    before = q.clone(), k.clone()
    qo, ko = fk.qk_norm_rope(q, k, cos, sin, pos, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=il)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
        _inside(got, *norm_rope_ref(x, cos, sin, pos, w, 1e-5, il))
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])


@gpu
def test_norm_rope_types_of_tables_and_weights_and_one_weight_only(dev):
    q, k, _ = _heads(dev, 33, 6, 2, 128, torch.float16, seed=3)
    w = _weights(dev, 128, torch.float32, 3)
    cos, sin = fk.rope_table(64, 64, device=dev)
    pos = torch.arange(33, device=dev)  # int64 positions are taken too
    for tt in (torch.float32, torch.float16, torch.bfloat16):
        c, s = cos.to(tt), sin.to(tt)
        qo, ko = fk.qk_norm_rope(q, k, c, s, pos, q_weight=None, k_weight=w[1])
        _inside(qo, *norm_rope_ref(q, c, s, pos))
        _inside(ko, *norm_rope_ref(k, c, s, pos, w[1]))
    # tables as columns of a wider one, without positions: token t takes row t % rows
    wide = torch.cat([cos, sin], 1)[:11]
    qo, ko = fk.qk_norm_rope(q, k, wide[:, :32], wide[:, 32:], q_weight=w[0])
    row = torch.arange(33, device=dev) % 11
    _inside(qo, *norm_rope_ref(q, cos, sin, row, w[0]))
    _inside(ko, *norm_rope_ref(k, cos, sin, row))


def _scattered_weights(D, dtype, device):
    """Norm weights whose entries do not lie one after another."""
    g = torch.Generator().manual_seed(23)
    layers = (1 + 0.2 * torch.randn(D, 8, generator=g)).to(dtype).to(device)
    return [layers[:, 3], layers.reshape(-1)[::8], layers[:, 2:3], layers[3:4, :1].expand(D, 1), layers[0, :1].expand(D),
            layers.t()[5:6]]


def test_weights_are_handed_on_contiguous():
    from fasterkernels_b200.qk_norm_rope import _check_weight
    for w in _scattered_weights(64, torch.float16, "cpu"):
        got = _check_weight(w, "q_weight", 64, w.device)
        assert got.is_contiguous() and torch.equal(got.reshape(-1), w.reshape(-1))
    w = torch.ones(64)
    assert _check_weight(w, "q_weight", 64, w.device) is w and _check_weight(None, "q_weight", 64, w.device) is None


@gpu
@pytest.mark.parametrize("T", [5, 4000])
def test_norm_weights_of_any_layout(dev, T):
    """A column of stacked parameters, every eighth entry, an expanded one."""
    D = 128
    q, k, v = _heads(dev, T, 4, 2, D, torch.float16, seed=7)
    cos, sin = fk.rope_table(64, D, device=dev)
    pos = torch.arange(T, device=dev, dtype=torch.int32) % 64
    kp, vp = (torch.zeros(T // 16 + 1, 2, 16, D, dtype=torch.float16, device=dev) for _ in range(2))
    bt = torch.arange(T // 16 + 1, dtype=torch.int32, device=dev)[None]
    zero = torch.zeros(T, dtype=torch.int32, device=dev)
    at = torch.arange(T, dtype=torch.int32, device=dev)
    for dtype in (torch.float32, torch.float16):
        for w in _scattered_weights(D, dtype, dev):
            qo, ko = fk.qk_norm_rope(q, k, cos, sin, pos, q_weight=w, k_weight=w)
            for got, x in ((qo, q), (ko, k)):
                _inside(got, *norm_rope_ref(x, cos, sin, pos, w.reshape(-1)))
            qa = fk.paged_kv_append_rope(q, k, v, kp, vp, bt, at, None, None, seq_ids=zero, q_weight=w, k_weight=w)
            _inside(qa, *norm_rope_ref(q, None, None, at, w.reshape(-1)))
            kept = kp.transpose(1, 2).reshape(-1, 2, D)[:T]
            _inside(kept, *norm_rope_ref(k, None, None, at, w.reshape(-1)))


@gpu
def test_norm_rope_small_and_large_rows(dev):
    # rows of zeros stay zero (eps keeps the norm finite); rows near the type's ends stay inside the bound
    q, k, _ = _heads(dev, 4, 8, 2, 128, torch.bfloat16, seed=9, packed=False)
    q[0] = 0
    q[1] *= 1e15
    q[2] *= 1e-30
    w = _weights(dev, 128, torch.float32, 9)
    cos, sin = fk.rope_table(8, 128, device=dev)
    pos = torch.arange(4, device=dev, dtype=torch.int32)
    qo, _ = fk.qk_norm_rope(q, k, cos, sin, pos, q_weight=w[0], k_weight=w[1])
    ref, amp = norm_rope_ref(q, cos, sin, pos, w[0])
    _inside(qo, ref, amp)
    assert bool((qo[0] == 0).all())


@gpu
def test_norm_rope_in_place_unaligned_and_strided(dev):
    cos, sin = fk.rope_table(100, 128, device=dev)
    pos = torch.randint(0, 100, (19,), device=dev, dtype=torch.int32)
    q, k, _ = _heads(dev, 19, 4, 2, 128, torch.float16, seed=5)
    qo, ko = fk.qk_norm_rope(q, k, cos, sin, pos)
    q2, k2 = q.clone(), k.clone()
    r = fk.qk_norm_rope(q2, k2, cos, sin, pos, q_out=q2, k_out=k2)
    assert r[0] is q2 and torch.equal(q2, qo) and torch.equal(k2, ko)
    # a view that starts between 16-byte boundaries, and one whose dims are not adjacent
    flat = torch.empty(19 * 4 * 128 + 3, dtype=torch.float16, device=dev)
    qu = flat[3:].view(19, 4, 128)
    qu.copy_(q)
    ks = torch.empty(19, 2, 256, dtype=torch.float16, device=dev)[..., ::2]
    ks.copy_(k)
    a, b = fk.qk_norm_rope(qu, ks, cos, sin, pos)
    assert torch.equal(a, qo) and torch.equal(b, ko)
    # outputs inside larger buffers leave the rest alone
    big = torch.full((21, 8, 128), 7.0, dtype=torch.float16, device=dev)
    fk.qk_norm_rope(q, k, cos, sin, pos, q_out=big[1:20, 2:6], k_out=k2)
    assert torch.equal(big[1:20, 2:6], qo)
    big[1:20, 2:6] = 7.0
    assert bool((big == 7.0).all())


@gpu
def test_norm_rope_empty_and_bad_positions(dev):
    cos, sin = fk.rope_table(10, 128, device=dev)
    e = torch.empty(0, 4, 128, dtype=torch.float16, device=dev)
    qo, ko = fk.qk_norm_rope(e, e, cos, sin, torch.empty(0, dtype=torch.int32, device=dev))
    assert qo.shape == ko.shape == e.shape
    q, k, _ = _heads(dev, 5, 4, 4, 128, torch.float16, seed=1)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    pos = torch.tensor([0, 10, 9, -1, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    qo, ko = fk.qk_norm_rope(q, k, cos, sin, pos, status=st)
    ok = pos.clamp(0, 9)
    ref, amp = norm_rope_ref(q, cos, sin, ok)
    for t in (0, 2):
        _inside(qo[t], ref[t], amp[t])
    assert bool((qo[[1, 3, 4]] == 0).all()) and bool((ko[[1, 3, 4]] == 0).all())
    assert int(st) == N.FK_STATUS_BAD_POSITION


@gpu
@pytest.mark.parametrize("T", [7, 3000])
@pytest.mark.parametrize("layout", ["heads first", "in place", "wide"])
def test_norm_rope_layouts_and_bad_positions_among_many(dev, T, layout):
    """Few and many tokens take different kernels: rows that do not lie one
    after another, outputs over inputs, a token too wide to stream."""
    QH, KVH = (300, 150) if layout == "wide" else (8, 2)
    q, k, _ = _heads(dev, T, QH, KVH, 128, torch.float16, seed=13)
    cos, sin = fk.rope_table(500, 128, device=dev)
    pos = torch.randint(0, 500, (T,), device=dev, dtype=torch.int32)
    pos[::5] = -1
    pos[3] = 500
    w = _weights(dev, 128, torch.float16, 1)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    ok = (pos >= 0) & (pos < 500)
    refs = [norm_rope_ref(x, cos, sin, pos.clamp(0, 499), w[i]) for i, x in enumerate((q, k))]
    if layout == "heads first":
        q, k = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k))
    out = (q, k) if layout == "in place" else (None, None)
    qo, ko = fk.qk_norm_rope(q, k, cos, sin, pos, q_weight=w[0], k_weight=w[1], q_out=out[0], k_out=out[1], status=st)
    for got, (ref, amp) in zip((qo, ko), refs):
        _inside(got[ok], ref[ok], amp[ok])
        assert bool((got[~ok] == 0).all())
    assert int(st) == N.FK_STATUS_BAD_POSITION


@gpu
def test_wrapper_refusals(dev):
    q, k, v = _heads(dev, 4, 4, 2, 128, torch.float16, seed=1)
    cos, sin = fk.rope_table(10, 128, device=dev)
    pos = torch.zeros(4, dtype=torch.int32, device=dev)
    kp = torch.zeros(3, 2, 16, 128, dtype=torch.float16, device=dev)
    bt = torch.zeros(4, 1, dtype=torch.int32, device=dev)
    z = torch.ones((), device=dev)
    bad = [
        lambda: fk.qk_norm_rope(q, k.bfloat16(), cos, sin, pos),
        lambda: fk.qk_norm_rope(q.float(), k.float(), cos, sin, pos),
        lambda: fk.qk_norm_rope(q, k[:3], cos, sin, pos),
        lambda: fk.qk_norm_rope(q, k.cpu(), cos, sin, pos),
        lambda: fk.qk_norm_rope(q[..., :96], k[..., :96], cos, sin, pos),
        lambda: fk.qk_norm_rope(q, k[:, :0], cos, sin, pos),
        lambda: fk.qk_norm_rope(q, k, cos, None, pos),
        lambda: fk.qk_norm_rope(q, k, cos, sin[:, :32], pos),
        lambda: fk.qk_norm_rope(q, k, cos[:, :12], sin[:, :12], pos),
        lambda: fk.qk_norm_rope(q, k, cos[:0], sin[:0], pos),
        lambda: fk.qk_norm_rope(q, k, cos.cpu(), sin.cpu(), pos),
        lambda: fk.qk_norm_rope(q, k, cos.double(), sin.double(), pos),
        lambda: fk.qk_norm_rope(q, k, cos, sin, pos[:3]),
        lambda: fk.qk_norm_rope(q, k, cos, sin, pos.cpu()),
        lambda: fk.qk_norm_rope(q, k, cos, sin, pos, q_weight=cos[0]),
        lambda: fk.qk_norm_rope(q, k, cos, sin, pos, k_weight=torch.ones(128)),
        lambda: fk.qk_norm_rope(q, k, cos, sin, pos, q_out=k),
        lambda: fk.qk_norm_rope(q, k, cos, sin, pos, status=pos.long()),
        lambda: fk.qk_norm_rope(q.detach().requires_grad_(), k, cos, sin, pos),
        lambda: fk.qk_norm_rope(q, k, cos, sin, pos, q_weight=torch.ones(128, device=dev, requires_grad=True)),
        lambda: fk.paged_kv_append_rope(q, k, v[:, :1], kp, kp, bt, pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp[:, :1], kp[:, :1], bt, pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp, kp.bfloat16(), bt, pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp.bfloat16(), kp.bfloat16(), bt, pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp.float(), kp.float(), bt, pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp.to(E4M3), kp.to(E4M3), bt, pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp, kp, bt[:3], pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp, kp, bt.cpu(), pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp, kp, bt, pos[:2], cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v, kp, kp, bt, pos, cos, sin, seq_ids=pos[:2]),
        lambda: fk.paged_kv_append_rope(q, k, v, kp[..., ::2], kp[..., ::2], bt, pos, cos, sin),
        lambda: fk.paged_kv_append_rope(q, k, v.detach().requires_grad_(), kp, kp, bt, pos, cos, sin),
    ]
    del z
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():  # inference on leaves that require grad is what serving does
        fk.qk_norm_rope(q.detach().requires_grad_(), k, cos, sin, pos)


def _pages(dev, counts, starts, extra=3, seed=0):
    """A block table over random pages for sequences of start + count tokens."""
    need = [(s + c + 15) // 16 for s, c in zip(starts, counts)]
    P = sum(need) + extra
    perm = torch.randperm(P, generator=torch.Generator().manual_seed(seed))
    bt = torch.full((len(need), max(need) + 1), -1, dtype=torch.int32)
    i = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[i:i + n].to(torch.int32)
        i += n
    return bt.to(dev), P


def _check_pools(kp, vp, k0, v0, bt, seq, pos, kref, kamp, v, sk, sv):
    """Appended slots against the references, every other slot unchanged."""
    page, slot = bt[seq.long(), pos.long() // 16].long(), pos.long() % 16
    e4 = kp.dtype == E4M3
    got = kp[page, :, slot]
    if e4:
        _inside_e4m3(got, kref / sk, kamp / sk)
        want_v = (v.float() / sv).clamp(-448, 448).to(E4M3)
        assert torch.equal(vp[page, :, slot].view(torch.uint8), want_v.view(torch.uint8))
    else:
        _inside(got, kref, kamp)
        assert torch.equal(vp[page, :, slot], v)
    as_bits = (lambda t: t.view(torch.uint8)) if e4 else (lambda t: t.view(torch.int16))
    a, b = as_bits(kp.clone()), as_bits(k0.clone())
    c, d = as_bits(vp.clone()), as_bits(v0.clone())
    for t in (a, b, c, d):
        t[page, :, slot] = 0
    assert torch.equal(a, b) and torch.equal(c, d)


def _inside_e4m3(got, ref, amp):
    ref = ref.clamp(-448, 448)
    err = (got.to(torch.float64) - ref).abs()
    bound = rounding_bound(ref, amp, E4M3) + 2.0 ** -22 * amp  # the division rounds once more
    assert bool((err <= bound).all()), float((err / bound).max())


@gpu
@pytest.mark.parametrize("pool", ["same", "e4m3"])
@pytest.mark.parametrize("D,R,il,dtype", [(128, 128, False, torch.bfloat16), (128, 64, True, torch.float16),
                                          (64, 64, False, torch.float16), (64, 16, False, torch.bfloat16)])
@pytest.mark.parametrize("counts,starts", [([1] * 5, [0, 15, 16, 333, 31]), ([1], [0]), ([3, 40, 1, 700], [14, 0, 47, 5]),
                                           ([1, 900, 2, 333, 600], [15, 7, 0, 1000, 1])])
def test_append_rope_matches_reference(dev, pool, D, R, il, dtype, counts, starts):
    QH, KVH = 6, 3
    T = sum(counts)
    q, k, v = _heads(dev, T, QH, KVH, D, dtype, seed=T + D)
    qw, kw = _weights(dev, D, dtype, T)
    cos, sin = fk.rope_table(2000, R, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).to(dev)
    pos = torch.cat([torch.arange(s, s + c) for s, c in zip(starts, counts)]).to(device=dev, dtype=torch.int32)
    bt, P = _pages(dev, counts, starts)
    pdt = dtype if pool == "same" else E4M3
    kp = torch.randn(P, KVH, 16, D, device=dev).to(pdt)
    vp = torch.randn(P, KVH, 16, D, device=dev).to(pdt)
    k0, v0 = kp.clone(), vp.clone()
    sk, sv = (torch.tensor(0.013, device=dev), torch.tensor(0.002, device=dev)) if pool == "e4m3" else (None, None)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    qo = fk.paged_kv_append_rope(q, k, v, kp, vp, bt, pos, cos, sin, seq_ids=None if T == len(counts) else seq,
                                 q_weight=qw, k_weight=kw, interleaved=il, scale_k=sk, scale_v=sv, k_out=ko, status=st)
    qref = norm_rope_ref(q, cos, sin, pos, qw, 1e-6, il)
    kref, kamp = norm_rope_ref(k, cos, sin, pos, kw, 1e-6, il)
    _inside(qo, *qref)
    _inside(ko, kref, kamp)
    _check_pools(kp, vp, k0, v0, bt, seq, pos, kref, kamp, v, sk, sv)
    assert int(st) == 0
    # the outputs are those of qk_norm_rope, bit for bit
    q2, k2 = fk.qk_norm_rope(q, k, cos, sin, pos, q_weight=qw, k_weight=kw, interleaved=il)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


@gpu
@pytest.mark.parametrize("pool", [torch.float16, E4M3])
def test_append_rope_without_rotation_equals_paged_kv_append(dev, pool):
    B, KVH, D = 9, 8, 128
    q, k, v = _heads(dev, B, 8, KVH, D, torch.float16, seed=2)
    starts = [0, 1, 15, 16, 17, 100, 31, 32, 63]
    bt, P = _pages(dev, [1] * B, starts)
    pos = torch.tensor(starts, dtype=torch.int32, device=dev)
    pools = [torch.zeros(P, KVH, 16, D, device=dev).to(pool) for _ in range(4)]
    s = torch.tensor(0.02, device=dev)
    kw = dict(scale_k=s, scale_v=s) if pool == E4M3 else {}
    paged_kv_append(k.contiguous(), v.contiguous(), pools[0], pools[1], bt, pos, **kw)
    qo = fk.paged_kv_append_rope(q, k, v, pools[2], pools[3], bt, pos, None, None, **kw)
    assert torch.equal(qo, q)
    for a, b in ((0, 2), (1, 3)):
        assert torch.equal(pools[a].view(torch.uint8), pools[b].view(torch.uint8))


@gpu
@pytest.mark.parametrize("T", [64, 4096])
@pytest.mark.parametrize("scale", [1.0, 0.25, 1.5, 3.0, 0.0125, 0.7071, -0.3, 1e-33, 3e-39, 1e33, 0.0, float("inf")])
def test_append_rope_quantises_every_value_as_a_division_does(dev, T, scale):
    KVH, D = 8, 128
    every = torch.arange(65536, dtype=torch.int32, device=dev).to(torch.int16).view(torch.bfloat16).view(64, KVH, D)
    v = every.repeat(T // 64, 1, 1)
    k = torch.zeros_like(v)
    P = T // 16
    bt = torch.arange(P, dtype=torch.int32, device=dev)[None]
    pos, seq = torch.arange(T, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int32, device=dev)
    pools = [torch.zeros(P, KVH, 16, D, device=dev).to(E4M3) for _ in range(4)]
    s = torch.tensor(scale, device=dev)
    fk.paged_kv_append_rope(k[:, :1], k, v, pools[0], pools[1], bt, pos, None, None, seq_ids=seq, scale_k=s, scale_v=s)
    paged_kv_append(k, v, pools[2], pools[3], bt[0][:, None].repeat_interleave(16, 0), pos % 16, scale_k=s, scale_v=s)
    assert torch.equal(pools[0].view(torch.uint8), pools[2].view(torch.uint8))
    assert torch.equal(pools[1].view(torch.uint8), pools[3].view(torch.uint8))
    # each quotient, rounded to f32 and to e4m3
    want = (v.float() / s).clamp(-448, 448).to(E4M3).float()
    got = pools[1].transpose(1, 2).reshape(T, KVH, D).float()
    assert torch.equal(torch.nan_to_num(got, nan=1e4), torch.nan_to_num(want, nan=1e4))


@gpu
def test_append_rope_device_side_conditions(dev):
    q, k, v = _heads(dev, 7, 4, 2, 128, torch.float16, seed=8)
    cos, sin = fk.rope_table(50, 128, device=dev)
    #        fine  past max_blocks  unallocated  page >= pool  bad position  bad seq  fine
    pos = torch.tensor([3, 40, 20, 5, 50, 0, 17], dtype=torch.int32, device=dev)
    seq = torch.tensor([0, 0, 1, 2, 0, 9, 0], dtype=torch.int32, device=dev)
    bt = torch.tensor([[0, 1], [2, -1], [4, 3]], dtype=torch.int32, device=dev)
    kp, vp = torch.zeros(4, 2, 16, 128, dtype=torch.float16, device=dev), torch.zeros(4, 2, 16, 128, dtype=torch.float16, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    qo = fk.paged_kv_append_rope(q, k, v, kp, vp, bt, pos, cos, sin, seq_ids=seq, status=st)
    assert int(st) == N.FK_STATUS_BAD_POSITION | N.FK_STATUS_BAD_PAGE
    ref, amp = norm_rope_ref(q, cos, sin, pos.clamp(max=49))
    for t in (0, 1, 2, 3, 5, 6):  # a bad page still returns the rotated q
        _inside(qo[t], ref[t], amp[t])
    assert bool((qo[4] == 0).all())
    want = torch.zeros_like(vp)
    want[0, :, 3], want[1, :, 1] = v[0], v[6]
    assert torch.equal(vp, want)
    kz = kp.clone()
    kz[0, :, 3] = 0
    kz[1, :, 1] = 0
    assert bool((kz == 0).all())


@gpu
def test_append_rope_offsets_past_32_bits(dev):
    # 140,000 pages of 16 KB: the last pages start past 2^31 elements
    KVH, D, P = 8, 128, 140_000
    kp = torch.zeros(P, KVH, 16, D, dtype=E4M3, device=dev)
    vp = torch.zeros(P, KVH, 16, D, dtype=E4M3, device=dev)
    q, k, v = _heads(dev, 2, 8, KVH, D, torch.float16, seed=4)
    bt = torch.tensor([[P - 1], [131_072]], dtype=torch.int32, device=dev)
    pos = torch.tensor([15, 0], dtype=torch.int32, device=dev)
    one = torch.ones((), device=dev)
    fk.paged_kv_append_rope(q, k, v, kp, vp, bt, pos, None, None, scale_k=one, scale_v=one)
    for pool, x in ((kp, k), (vp, v)):
        assert torch.equal(pool[P - 1, :, 15].view(torch.uint8), x[0].float().to(E4M3).view(torch.uint8))
        assert torch.equal(pool[131_072, :, 0].view(torch.uint8), x[1].float().to(E4M3).view(torch.uint8))
        assert int((pool.view(torch.uint8) != 0).sum()) == int((x.float().to(E4M3).view(torch.uint8) != 0).sum())


@gpu
def test_append_rope_strided_pools_and_tables(dev):
    # one layer of a [L, P, ...] cache with K and V interleaved, a block table with spare columns
    D, KVH = 128, 2
    kv = torch.zeros(3, 6, 2, KVH, 16, D, dtype=torch.bfloat16, device=dev)
    kp, vp = kv[1, :, 0], kv[1, :, 1]
    q, k, v = _heads(dev, 2, 4, KVH, D, torch.bfloat16, seed=4)
    wide = torch.full((4, 9), 77, dtype=torch.int32, device=dev)
    wide[1, 2], wide[3, 2] = 5, 0
    bt = wide[1::2, 2:4]
    pos = torch.tensor([7, 8], dtype=torch.int32, device=dev)
    cos, sin = fk.rope_table(50, 128, device=dev)
    fk.paged_kv_append_rope(q, k, v, kp, vp, bt, pos, cos, sin)
    ref, amp = norm_rope_ref(k, cos, sin, pos)
    _inside(kp[[5, 0], :, [7, 8]], ref, amp)
    assert torch.equal(vp[[5, 0], :, [7, 8]], v)
    kv[1, [5, 0], :, :, [7, 8]] = 0
    assert bool((kv == 0).all())


@gpu
def test_append_rope_captured_and_replayed_with_new_positions(dev):
    B, D = 3, 128
    q, k, v = (t.clone() for t in _heads(dev, B, 4, 2, D, torch.float16, seed=6))
    cos, sin = fk.rope_table(64, 128, device=dev)
    bt = torch.arange(B * 4, dtype=torch.int32, device=dev).view(B, 4)
    kp, vp = torch.zeros(12, 2, 16, D, dtype=torch.float16, device=dev), torch.zeros(12, 2, 16, D, dtype=torch.float16, device=dev)
    pos = torch.zeros(B, dtype=torch.int32, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):  # nothing to warm up: the operator keeps no workspace
        qo = fk.paged_kv_append_rope(q, k, v, kp, vp, bt, pos, cos, sin)
        pos.add_(1)
    pos.copy_(torch.tensor([0, 15, 30], dtype=torch.int32))
    for step in range(4):
        p = pos.clone()
        q.normal_()
        k.normal_()
        v.normal_()
        g.replay()
        ref, amp = norm_rope_ref(q, cos, sin, p)
        _inside(qo, ref, amp)
        page, slot = bt[torch.arange(B, device=dev), p.long() // 16].long(), p.long() % 16
        _inside(kp[page, :, slot], *norm_rope_ref(k, cos, sin, p))
        assert torch.equal(vp[page, :, slot], v)


@gpu
def test_norm_rope_on_another_stream_and_two_at_once(dev):
    cos, sin = fk.rope_table(4096, 128, device=dev)
    jobs = []
    for i in range(2):
        q, k, _ = _heads(dev, 3000, 16, 4, 128, torch.bfloat16, seed=20 + i)
        jobs.append((q, k, torch.randint(0, 4096, (3000,), device=dev, dtype=torch.int32)))
    want = [fk.qk_norm_rope(q, k, cos, sin, p) for q, k, p in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for s, (q, k, p) in zip(streams, jobs):
        with torch.cuda.stream(s):
            got.append(fk.qk_norm_rope(q, k, cos, sin, p))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu
def test_compile_fullgraph(dev):
    torch._dynamo.reset()
    q, k, v = (t.contiguous() for t in _heads(dev, 4, 4, 2, 128, torch.float16, seed=6))
    cos, sin = fk.rope_table(64, 128, device=dev)
    bt = torch.arange(4, dtype=torch.int32, device=dev).view(4, 1)
    pos = torch.tensor([3, 4, 5, 6], dtype=torch.int32, device=dev)

    def step(q, k, v, kp, vp):
        a, b = fk.qk_norm_rope(q * 2, k, cos, sin, pos)
        c = fk.paged_kv_append_rope(a, b, v, kp, vp, bt, pos, cos, sin)
        return c + 1

    pools = [torch.zeros(4, 2, 16, 128, dtype=torch.float16, device=dev) for _ in range(4)]
    eager = step(q, k, v, *pools[:2])
    got = torch.compile(step, fullgraph=True)(q, k, v, *pools[2:])
    assert torch.equal(eager, got) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


@gpu
@pytest.mark.parametrize("unsqueeze_dim", [1, 2])
@pytest.mark.parametrize("cos_batch", [1, 3])
def test_hf_rotary_drop_in(dev, unsqueeze_dim, cos_batch):
    B, S, D = 3, 21, 128
    q, k, _ = _heads(dev, B * S, 8, 2, D, torch.bfloat16, seed=11)
    q, k = q.reshape(B, S, 8, D), k.reshape(B, S, 2, D)
    ang = torch.rand(cos_batch, S, D // 2, device=dev) * 6
    cos = torch.cat([ang, ang], -1).cos().bfloat16()
    sin = torch.cat([ang, ang], -1).sin().bfloat16()
    args = (q.transpose(1, 2), k.transpose(1, 2)) if unsqueeze_dim == 1 else (q, k)
    qo, ko = fk.custom_hf_apply_rotary_pos_emb(*args, cos, sin, unsqueeze_dim=unsqueeze_dim)
    assert qo.shape == args[0].shape and ko.shape == args[1].shape
    if unsqueeze_dim == 1:
        qo, ko = qo.transpose(1, 2), ko.transpose(1, 2)
    c, s = (t.expand(B, S, D).reshape(B * S, D)[:, :D // 2] for t in (cos, sin))
    row = torch.arange(B * S, device=dev)
    for got, x in ((qo, q), (ko, k)):
        ref, amp = norm_rope_ref(x.reshape(B * S, -1, D), c, s, row)
        _inside(got.reshape(B * S, -1, D), ref, amp)
    with pytest.raises(ValueError, match="sequence length"):
        fk.custom_hf_apply_rotary_pos_emb(*args, cos[:, :3], sin[:, :3], unsqueeze_dim=unsqueeze_dim)


@gpu
def test_hf_rotary_drop_in_inside_a_random_weight_model(dev, monkeypatch):
    """A small random-init Qwen3 whose layers rotate with the drop-in: same
    logits as with transformers' own function (which rounds the two products
    and their sum to f16 where the drop-in rounds once), prompt and steps."""
    from transformers import DynamicCache, Qwen3Config, Qwen3ForCausalLM
    from transformers.models.qwen3 import modeling_qwen3
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=512)
    torch.manual_seed(0)
    model = Qwen3ForCausalLM(cfg).to(device=dev, dtype=torch.float16).eval()
    prompt = torch.randint(0, 512, (2, 33), device=dev)
    feed = torch.randint(0, 512, (3, 2, 1), device=dev)

    def run():
        cache, logits = DynamicCache(config=cfg), []
        with torch.no_grad():
            logits.append(model(input_ids=prompt, past_key_values=cache, use_cache=True).logits[:, -1].float())
            for t in feed:
                logits.append(model(input_ids=t, past_key_values=cache, use_cache=True).logits[:, -1].float())
        return torch.stack(logits)

    want, calls = run(), []
    monkeypatch.setattr(modeling_qwen3, "apply_rotary_pos_emb",
                        lambda *a, **k: calls.append(1) or fk.custom_hf_apply_rotary_pos_emb(*a, **k))
    got = run()
    assert len(calls) == 2 * 4
    torch.testing.assert_close(got, want, atol=3e-2, rtol=3e-2)


# model file -> what the drop-in takes for it, rotated dims of 128, columns
_HF_LAYOUTS = {
    "llama": (dict(), 128, 128),
    "phi3": (dict(), 96, 96),
    "glm4_moe": (dict(tables="halves"), 64, 64),
    "gpt_oss": (dict(tables="once"), 128, 64),
    "cohere": (dict(tables="pairs", interleaved=True), 128, 128),
    "ernie4_5": (dict(tables="halves", interleaved=True), 128, 128),
    "glm": (dict(tables="halves", interleaved=True), 64, 64),
}


def _hf_case(model, device, dtype):
    import importlib
    kw, R, cols = _HF_LAYOUTS[model]
    own = importlib.import_module(f"transformers.models.{model}.modeling_{model}").apply_rotary_pos_emb
    g = torch.Generator().manual_seed(31)
    B, S, D = 2, 9, 128
    q, k = (torch.randn(B, h, S, D, generator=g).to(dtype).to(device) for h in (4, 2))
    ang = 6 * torch.rand(B, S, R // 2, generator=g)
    c, s = ang.cos().to(device), ang.sin().to(device)
    wide = [t if cols == R // 2 else t.repeat_interleave(2, -1) if kw.get("tables") == "pairs" else torch.cat([t, t], -1)
            for t in (c, s)]
    assert wide[0].shape[-1] == cols
    return kw, own, q, k, *wide, c.reshape(B * S, -1), s.reshape(B * S, -1)


@pytest.mark.parametrize("model", _HF_LAYOUTS)
def test_hf_table_layouts_are_those_of_the_model_files(model):
    from fasterkernels_b200.qk_norm_rope import _angles_once, _hf_tables
    kw, own, q, k, cos, sin, *once = _hf_case(model, "cpu", torch.float32)
    tables = _hf_tables(cos, 128, kw.get("tables"), kw.get("interleaved", False))
    c, s = (_angles_once(t.reshape(-1, t.shape[-1]), tables) for t in (cos, sin))
    assert torch.equal(c, once[0]) and torch.equal(s, once[1])
    row = torch.arange(18)
    for want, x in zip(own(q, k, cos, sin), (q, k)):
        ref, amp = norm_rope_ref(x.transpose(1, 2).reshape(18, -1, 128), c, s, row, interleaved=kw.get("interleaved", False))
        # f32 there: two products and a sum, half a step each
        assert bool(((want.transpose(1, 2).reshape(ref.shape).double() - ref).abs() <= 3 * 2.0 ** -24 * amp).all())


def test_hf_tables_that_do_not_say_what_they_are_are_refused():
    q, k = torch.zeros(1, 4, 3, 128), torch.zeros(1, 2, 3, 128)
    t = lambda cols: torch.zeros(1, 3, cols)  # noqa: E731
    f = fk.custom_hf_apply_rotary_pos_emb
    for cols, kw, match in ((64, {}, "tables"), (128, dict(interleaved=True), "tables"), (128, dict(tables="twice"), "tables must"),
                            (128, dict(tables="once"), "256 of 128"), (33, {}, "33 columns"), (256, {}, "256 columns"),
                            (0, {}, "0 columns"), (8, dict(tables="pairs"), "multiple of 16")):
        with pytest.raises(ValueError, match=match):
            f(q, k, t(cols), t(cols), **kw)
    with pytest.raises(ValueError, match="sequence length"):
        f(q, k, t(128), t(64))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("model", _HF_LAYOUTS)
def test_hf_rotary_drop_in_for_each_table_layout(dev, model, dtype):
    kw, own, q, k, cos, sin, c, s = _hf_case(model, dev, dtype)
    got = fk.custom_hf_apply_rotary_pos_emb(q, k, cos, sin, **kw)
    row = torch.arange(18, device=dev)
    for g, want, x in zip(got, own(q.float(), k.float(), cos, sin), (q, k)):
        ref, amp = norm_rope_ref(x.transpose(1, 2).reshape(18, -1, 128), c, s, row, interleaved=kw.get("interleaved", False))
        _inside(g.transpose(1, 2).reshape(ref.shape), ref, amp)
        assert bool(((want.transpose(1, 2).reshape(ref.shape).double() - ref).abs() <= 2.0 ** -20 * amp).all())


def test_custom_ops_declare_what_they_write():
    ns = torch.ops.fasterkernels_b200
    for name, mutated in (("qk_norm_rope", {"q_out", "k_out", "k_pool", "v_pool", "status"}),
                          ("shared_prefix_decode", {"out"})):
        schema = getattr(ns, name).default._schema
        written = {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
        assert written == mutated, (name, written)
