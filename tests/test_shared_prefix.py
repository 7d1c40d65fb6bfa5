"""paged_flash_decode_shared_prefix against 64-bit references: row and token
counts around the tile sizes, types, sinks, bad pages, graphs, streams."""
import struct

import pytest
import torch

import fasterkernels_b200 as fk
from fasterkernels_b200 import _native as N
from _operator_refs import attention_bound, shared_prefix_ref

gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def make(dev, P, lens, QH, KVH, D=128, dtype=torch.float16, pool=None, sinks=False, seed=0, q_scale=1.0):
    """Random pages for the prefix and every own tail; slots past the ends hold NaN."""
    pool = pool or dtype
    B = len(lens)
    g = torch.Generator(device=dev).manual_seed(seed)
    npre = (P + 15) // 16
    need = [(n + 15) // 16 for n in lens]
    pages = npre + sum(need) + 2
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    c = dict(P=P, lens=list(lens), QH=QH, KVH=KVH, D=D)
    c["q"] = (q_scale * torch.randn(B, QH, D, generator=g, device=dev)).to(dtype)
    c["table"] = perm[:npre].clone()
    c["bt"] = torch.full((B, max(need) if need else 0), -1, dtype=torch.int32, device=dev)
    i = npre
    for b, n in enumerate(need):
        c["bt"][b, :n] = perm[i:i + n]
        i += n
    c["seq"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    c["plen"] = torch.tensor([P], dtype=torch.int32, device=dev)
    c["sk"] = c["sv"] = None
    for name in ("k", "v"):
        x = torch.randn(pages, KVH, 16, D, generator=g, device=dev)
        if pool == E4M3:
            x = (80 * x).clamp(-448, 448)
            c["s" + name] = torch.tensor(1 / 80, device=dev)
        x = x.to(pool)
        nan = x.view(torch.uint8) if pool == E4M3 else x
        fill = 0x7f if pool == E4M3 else float("nan")
        nan[perm[i:].long()] = fill  # pages of nobody
        if P % 16:
            nan[int(c["table"][-1]), :, P % 16:] = fill
        for b, n in enumerate(lens):
            if n % 16:
                nan[int(c["bt"][b, n // 16]), :, n % 16:] = fill
        c[name] = x
    c["sink"] = torch.randn(QH, generator=g, device=dev) if sinks else None
    return c


def flat(c):
    """The logical K / V in 64 bits: prefix [KVH, P', D], own [B, KVH, T, D]."""
    out = []
    for name in ("k", "v"):
        s = 1.0 if c["s" + name] is None else c["s" + name].double()
        x = c[name].to(torch.float32).double() * s
        p = x[c["table"].long()].transpose(0, 1).reshape(c["KVH"], -1, c["D"])
        t = x[c["bt"].long().clamp(min=0)].transpose(1, 2).reshape(len(c["lens"]), c["KVH"], -1, c["D"])
        out.append((p, t))
    (kp, kt), (vp, vt) = out
    return kp, vp, kt, vt


def call(c, plen=None, **kw):
    return fk.paged_flash_decode_shared_prefix(c["q"], c["k"], c["v"], c["table"], c["plen"] if plen is None else plen,
                                               c["bt"], c["seq"], 16, s_aux=c["sink"], scale_k=c["sk"], scale_v=c["sv"], **kw)


def check(c, got, q=None, prefix=None, lens=None):
    kp, vp, kt, vt = flat(c)
    q = c["q"].double() if q is None else q
    prefix = c["P"] if prefix is None else prefix
    lens = c["lens"] if lens is None else lens
    ref = shared_prefix_ref(q, kp, vp, prefix, kt, vt, lens, c["sink"])
    p_dtype = torch.bfloat16 if c["k"].dtype == torch.bfloat16 else torch.float16
    bound = attention_bound(q, kp, vp, prefix, kt, vt, lens, c["sink"], ref, p_dtype, got.dtype)
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())


@gpu
@pytest.mark.parametrize("P", [128, 1, 15, 17, 127, 129, 256, 257, 1000, 4096])
def test_prefix_lengths(dev, P):
    c = make(dev, P, [0, 1, 16, 40], 8, 2, seed=P)
    check(c, call(c))


@gpu
@pytest.mark.parametrize("B,G", [(1, 1), (127, 1), (128, 1), (43, 3), (32, 4), (64, 4), (257, 1), (24, 16), (100, 5), (7, 40)])
def test_row_counts(dev, B, G):
    c = make(dev, 600, [(37 * b) % 90 for b in range(B)], 2 * G, 2, seed=B + G, sinks=True)
    check(c, call(c))


@gpu
@pytest.mark.parametrize("D,dtype,pool", [(128, torch.float16, None), (128, torch.bfloat16, None), (64, torch.float16, None),
                                          (64, torch.bfloat16, None), (128, torch.float16, E4M3), (128, torch.bfloat16, E4M3)])
@pytest.mark.parametrize("B,G,KVH,P", [(3, 4, 8, 700), (80, 4, 3, 1333)])
@pytest.mark.parametrize("sinks", [False, True])
def test_types(dev, D, dtype, pool, B, G, KVH, P, sinks):
    c = make(dev, P, [(61 * b) % 300 for b in range(B)], G * KVH, KVH, D, dtype, pool, sinks, seed=P)
    check(c, call(c))


@gpu
def test_long_prefix_crosses_many_segments(dev):
    c = make(dev, 40_001, [5, 0], 4, 2, seed=3)
    check(c, call(c))


@gpu
@pytest.mark.parametrize("B,tail,P", [(16, 0, 4096), (16, 20, 4096), (16, 80, 8192), (16, 300, 4096), (37, 77, 5003), (64, 200, 2048)])
def test_prefix_beside_own_parts_of_any_size(dev, B, tail, P):
    """None, some and all SMs busy with the own part: the prefix is cut differently."""
    c = make(dev, P, [max(tail - b % 7, 0) for b in range(B)], 16, 4, seed=B + tail)
    out = call(c)
    check(c, out)
    assert torch.equal(out, call(c)) and fk.read_status() == 0


@gpu
@pytest.mark.parametrize("dtype,pool", [(torch.float16, None), (torch.bfloat16, None), (torch.float16, E4M3)])
def test_sharp_softmax_and_rising_maxima(dev, dtype, pool):
    c = make(dev, 900, [50, 3], 8, 2, dtype=dtype, pool=pool, sinks=True, seed=5, q_scale=6.0)
    check(c, call(c))
    # logits that rise along the prefix move the running maximum in every tile
    u = torch.sign(torch.randn(128, device=dev))
    c["q"][:] = u.to(dtype)
    n = c["table"].numel() * 16
    ramp = (torch.arange(n, device=dev) / n * 3.5).view(-1, 1, 16, 1) * u
    if pool == E4M3:
        ramp = ramp * 80
    c["k"][c["table"].long()] = ramp.expand(-1, 2, -1, -1).to(c["k"].dtype)
    check(c, call(c))


@gpu
def test_same_as_paged_flash_decode_over_whole_tables(dev):
    c = make(dev, 512, [0, 1, 15, 100, 33], 32, 8, sinks=True, seed=8)
    whole = torch.cat([c["table"].expand(5, -1), c["bt"]], 1)
    lens = c["seq"] + 512
    want = fk.paged_flash_decode(c["q"], c["k"], c["v"], whole, lens, 16, s_aux=c["sink"])
    got = fk.paged_flash_decode_shared_prefix(c["q"], c["k"], c["v"], whole[0, :32], 512, whole[:, 32:], lens - 512, 16,
                                              s_aux=c["sink"])
    check(c, got)
    check(c, want)
    assert torch.equal(got, call(c))  # twice the same bits, and a column slice is a block table


@gpu
def test_nothing_to_attend_and_empty_parts(dev):
    c = make(dev, 100, [0, 30, 0], 8, 2, sinks=True, seed=4)
    check(c, call(c))
    out = call(c, plen=0)
    check(c, out, prefix=0)
    assert bool((out[[0, 2]] == 0).all()) and bool((out[1] != 0).any())
    c0 = make(dev, 100, [0, 0], 8, 2, seed=4)
    assert c0["bt"].shape == (2, 0)
    check(c0, call(c0))
    assert bool((call(c0, plen=0) == 0).all())
    e = c0["table"][:0]
    out = fk.paged_flash_decode_shared_prefix(c0["q"], c0["k"], c0["v"], e, 0, c0["bt"], c0["seq"], 16)
    assert bool((out == 0).all())
    z = fk.paged_flash_decode_shared_prefix(c0["q"][:0], c0["k"], c0["v"], c0["table"], 100, c0["bt"], c0["seq"], 16)
    assert z.shape == (0, 8, 128)
    assert fk.read_status() == 0


@gpu
@pytest.mark.parametrize("dtype,pool", [(torch.float16, None), (torch.bfloat16, None), (torch.float16, E4M3)])
@pytest.mark.parametrize("P,lens", [(200, [40, 0, 70]), (0, [40, 33, 70]), (200, [0, 0, 0])])
def test_a_nan_reaches_the_rows_that_attend_it_and_no_others(dev, dtype, pool, P, lens):
    c = make(dev, P, lens, 8, 2, dtype=dtype, pool=pool, seed=6)
    clean = call(c)
    assert not bool(clean.isnan().any())
    c["q"][0, 1, 5] = float("nan")
    c["q"][1, 7, 0] = float("nan")
    out = call(c)
    hit = torch.zeros(3, 8, dtype=torch.bool, device=dev)
    hit[0, 1] = hit[1, 7] = True
    assert bool(out[hit].isnan().all()) and torch.equal(out[~hit], clean[~hit])
    c = make(dev, P, lens, 8, 2, dtype=dtype, pool=pool, seed=6)
    hit[:] = False
    for row, page in ((slice(None), c["table"]), (2, c["bt"][2])):  # a K row of head 1: in the prefix, in sequence 2
        if page.numel():
            page = int(page[0])
            if pool == E4M3:
                c["k"].view(torch.uint8)[page, 1, 3] = 0x7f
            else:
                c["k"][page, 1, 3, 9] = float("nan")
            hit[row, 4:] = True
            out = call(c)
            assert bool(out[hit].isnan().all()) and torch.equal(out[~hit], clean[~hit])


@gpu
def test_scales_of_zero_and_nan(dev):
    c = make(dev, 200, [0, 0], 8, 2, pool=E4M3, seed=7)
    for k, v in ((0.0, 0.02), (0.02, 0.0)):
        c["sk"], c["sv"] = torch.tensor(k, device=dev), torch.tensor(v, device=dev)
        check(c, call(c))
    for k, v in ((float("nan"), 0.02), (0.02, float("nan"))):
        c["sk"], c["sv"] = torch.tensor(k, device=dev), torch.tensor(v, device=dev)
        assert bool(call(c).isnan().all())


@gpu
def test_prefix_length_on_the_host_and_on_the_device(dev):
    c = make(dev, 700, [20, 5], 8, 2, seed=6)
    want = call(c)
    assert torch.equal(want, call(c, plen=700))
    assert torch.equal(want, call(c, plen=torch.tensor(700, device=dev)))  # 0-dim, int64
    for n in (1, 129, 650):  # shorter than the table
        check(c, call(c, plen=n), prefix=n)
    # longer than the table: the missing tokens are masked and reported
    fk.read_status()
    got = call(c, plen=torch.tensor([5000], dtype=torch.int32, device=dev))
    c["k"][int(c["table"][-1])] = 0.5  # the table's last page was NaN past token 700
    c["v"][int(c["table"][-1])] = 0.25
    assert fk.read_status() == N.FK_STATUS_BAD_PAGE
    got = call(c, plen=torch.tensor([5000], dtype=torch.int32, device=dev))
    check(c, got, prefix=704)
    fk.read_status()
    assert bool((call(c, plen=torch.tensor([-3], dtype=torch.int32, device=dev)) == call(c, plen=0)).all())


@gpu
@pytest.mark.parametrize("pool", [torch.float16, E4M3])
def test_bad_pages_are_masked_and_reported(dev, pool):
    c = make(dev, 1024, [40, 0, 20], 64, 1, pool=pool, seed=2)
    fk.read_status()
    kp, vp, kt, vt = flat(c)
    for pg, bad in ((0, -1), (9, 10 ** 6), (63, -7)):
        c["table"][pg] = bad
    c["bt"][0, 1] = -1
    got = call(c)
    assert fk.read_status() == N.FK_STATUS_BAD_PAGE
    keep = torch.ones(64, 16, dtype=torch.bool, device=dev)
    keep[[0, 9, 63]] = False
    keep = keep.view(-1)
    kp, vp = kp[:, keep], vp[:, keep]
    own = torch.ones(kt.shape[2], dtype=torch.bool, device=dev)
    kt0, vt0 = kt.clone(), vt.clone()
    own[16:32] = False
    kt0[0, :, :24], vt0[0, :, :24] = kt[0, :, :40][:, own[:40]], vt[0, :, :40][:, own[:40]]
    args = (c["q"].double(), kp, vp, kp.shape[1], kt0, vt0, [24, 0, 20])
    ref = shared_prefix_ref(*args)
    bound = attention_bound(*args, None, ref, torch.float16, got.dtype)
    assert bool(((got.double() - ref).abs() <= bound).all())
    # a prefix of bad pages alone leaves the own tokens, and zeros where there are none
    c["table"][:] = -1
    got = call(c)
    args = (c["q"].double(), kp, vp, 0, kt0, vt0, [24, 0, 20])
    ref = shared_prefix_ref(*args)
    assert bool(((got.double() - ref).abs() <= attention_bound(*args, None, ref, torch.float16, got.dtype)).all())
    assert bool((got[1] == 0).all())
    fk.read_status()


@gpu
def test_strides_alignment_and_given_output(dev):
    c = make(dev, 333, [20, 7, 0], 12, 3, dtype=torch.bfloat16, seed=9)
    want = call(c)
    base = torch.full((3, 20, 130), 3.0, dtype=torch.bfloat16, device=dev)
    q = base[:, 4:16, 2:]  # rows on 4-byte boundaries only
    q.copy_(c["q"])
    outb = torch.full((3, 14, 136), 7.0, dtype=torch.bfloat16, device=dev)
    out = outb[:, 1:13, 4:132]
    c2 = dict(c, q=q)
    assert call(c2, out=out) is out and torch.equal(out, want)
    out.fill_(7.0)
    assert bool((outb == 7.0).all())
    # one layer of a cache that interleaves K and V pages
    P = c["k"].shape[0]
    kv = torch.randn(2, P, 2, 3, 16, 128, device=dev).bfloat16()
    kv[1, :, 0], kv[1, :, 1] = c["k"], c["v"]
    assert torch.equal(call(dict(c, k=kv[1, :, 0], v=kv[1, :, 1])), want)
    # the same page at several places of the prefix
    c["table"][3] = c["table"][1]
    check(c, call(c))


@gpu
def test_query_types_scales_and_output_types_over_e4m3(dev):
    c = make(dev, 300, [20, 33], 16, 2, pool=E4M3, sinks=True, seed=10)
    for sk in (-1 / 80, 0.0, 1 / 40):
        c["sk"] = torch.tensor(sk, device=dev)
        check(c, call(c))
    c["sk"] = 1 / 80  # a number is taken too
    got = call(c, out_dtype=torch.bfloat16)
    c["sk"] = torch.tensor(1 / 80, device=dev)
    assert got.dtype == torch.bfloat16
    check(c, got)
    q8 = (c["q"] * 100).clamp(-448, 448).to(E4M3)
    sq = torch.tensor(0.01, device=dev)
    got = fk.paged_flash_decode_shared_prefix(q8, c["k"], c["v"], c["table"], c["plen"], c["bt"], c["seq"], 16,
                                              s_aux=c["sink"], scale_q=sq, scale_k=c["sk"], scale_v=c["sv"])
    # q8 * scale rounded to f16 is what the kernel multiplies
    check(c, got, q=(q8.float() * sq).half().double())


@gpu
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("G,KVH", [(5, 4), (6, 8), (7, 4), (8, 4), (8, 8)])
@pytest.mark.parametrize("qtype", [torch.float16, torch.bfloat16, E4M3])
def test_own_tokens_of_four_heads_an_item(dev, G, KVH, qtype, aligned):
    """e4m3 pools, KV heads a multiple of four, groups of 5 to 8: the own part
    takes four KV heads at a time, with 32 slots a record, where the rows of q are
    16-byte aligned, and two where they are not."""
    c = make(dev, 500, [700, 0, 1, 33, 4000], G * KVH, KVH, dtype=torch.bfloat16 if qtype == torch.bfloat16 else torch.float16,
             pool=E4M3, sinks=True, seed=G + KVH)
    q, sq = c["q"], None
    if qtype == E4M3:
        q, sq = (100 * q).clamp(-448, 448).to(E4M3), torch.tensor(0.01, device=dev)
    if not aligned:
        wide = torch.zeros(5, G * KVH, 130 if qtype != E4M3 else 136, dtype=q.dtype, device=dev)
        wide[..., 2:130].copy_(q)
        q = wide[..., 2:130]
    got = fk.paged_flash_decode_shared_prefix(q, c["k"], c["v"], c["table"], c["plen"], c["bt"], c["seq"], 16, s_aux=c["sink"],
                                              scale_q=sq, scale_k=c["sk"], scale_v=c["sv"])
    # what the kernel multiplies: q (times its scale) rounded to f16
    check(c, got, q=(q.float() * sq).half().double() if sq is not None else q.half().double())


@gpu
def test_offsets_past_32_bits(dev):
    P = 140_000  # pages of 16 KB: the last ones start past 2^31 elements
    pages = [P - 1, 131_073, 5, P - 2, 139_000, 131_072]
    k = torch.zeros(P, 8, 16, 128, dtype=E4M3, device=dev)
    v = torch.zeros(P, 8, 16, 128, dtype=E4M3, device=dev)
    small = [torch.randn(6, 8, 16, 128, device=dev).to(E4M3) for _ in range(2)]
    k[pages], v[pages] = small[0], small[1]
    q = torch.randn(2, 16, 128, device=dev).half()
    one = torch.ones((), device=dev)
    bt = torch.tensor([[pages[4]], [pages[5]]], dtype=torch.int32, device=dev)
    seq = torch.tensor([16, 9], dtype=torch.int32, device=dev)
    a = fk.paged_flash_decode_shared_prefix(q, k, v, torch.tensor(pages[:4], dtype=torch.int32, device=dev), 60, bt, seq, 16,
                                            scale_k=one, scale_v=one)
    b = fk.paged_flash_decode_shared_prefix(q, small[0], small[1], torch.arange(4, dtype=torch.int32, device=dev), 60,
                                            torch.tensor([[4], [5]], dtype=torch.int32, device=dev), seq, 16,
                                            scale_k=one, scale_v=one)
    assert torch.equal(a, b)


@gpu
def test_two_graphs_replayed_at_once_with_new_lengths(dev):
    cases = [make(dev, 2000, [100] * 20, 16, 4, seed=20), make(dev, 900, [64] * 70, 16, 4, seed=21, sinks=True)]
    for c in cases:
        call(c)  # makes the status word
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    for step, (plen, own) in enumerate([(2000, 100), (1, 0), (777, 17), (128, 64)]):
        want = []
        for c in cases:
            c["plen"].fill_(min(plen, c["P"]))
            c["seq"].copy_(torch.arange(len(c["lens"]), device=dev).remainder(own + 1).clamp(max=min(c["lens"])))
            want.append(call(c))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert torch.equal(w, o), step
    assert fk.read_status() == 0


@gpu
def test_eager_calls_on_two_streams(dev):
    cases = [make(dev, 5000, [30] * 40, 32, 8, seed=30), make(dev, 3000, [200] * 10, 32, 8, seed=31)]
    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(call(cases[i]))
    torch.cuda.synchronize()
    for w, got in zip(want, outs):
        assert all(torch.equal(w, o) for o in got)


@gpu
def test_compile_fullgraph(dev):
    torch._dynamo.reset()
    c = make(dev, 300, [20, 33], 16, 2, seed=10)
    eager = call(c) + 1

    def step(q):
        return call(dict(c, q=q)) + 1

    assert torch.equal(torch.compile(step, fullgraph=True)(c["q"]), eager)


@gpu
def test_bounded_wait_runs_out_and_the_next_call_is_right(dev):
    c = make(dev, 1500, [20, 33], 16, 2, seed=10)
    want = call(c)
    fk.read_status()
    lib = N.lib()
    assert lib.fk_debug_configure(200_000_000, 1) == 0
    try:
        call(c)
        torch.cuda.synchronize()
    finally:
        assert lib.fk_debug_configure(4_000_000_000, 0) == 0
    assert fk.read_status() & N.FK_STATUS_TIMEOUT
    assert torch.equal(call(c), want) and fk.read_status() == 0


def entry_args(c, out, status):
    """fk_prefix_args of a 16-bit case."""
    kv = N.dtype_code(c["k"].dtype)
    B, QH, D = c["q"].shape
    a = dict(q=c["q"].data_ptr(), k_pool=c["k"].data_ptr(), v_pool=c["v"].data_ptr(), prefix_table=c["table"].data_ptr(),
             prefix_len_dev=c["plen"].data_ptr(), block_table=c["bt"].data_ptr(), seq_lens=c["seq"].data_ptr(), s_aux=0,
             out=out.data_ptr(), status=status.data_ptr(), prefix_len=0, prefix_blocks=c["table"].numel(), batch=B, q_heads=QH,
             kv_heads=c["KVH"], head_dim=D, num_pages=c["k"].shape[0], max_blocks=c["bt"].shape[1], q_dtype=kv, kv_dtype=kv,
             out_dtype=kv, bt_b=c["bt"].stride(0))
    for t, names in ((c["q"], "q_b q_h"), (c["k"], "kp_p kp_h kp_s"), (c["v"], "vp_p vp_h vp_s"), (out, "o_b o_h")):
        a.update(zip(names.split(), t.stride()))
    return _args(**a)


@gpu
@pytest.mark.parametrize("word", [0x3f800000, 0x7fffffff, -1, 1])
@pytest.mark.parametrize("lens", [[20, 33], [4000, 0, 7]])
def test_a_wait_that_ran_out_over_any_scratch_is_a_status(dev, word, lens):
    """The own part gives up before it says where its records are: what the
    scratch held there must not be taken for them."""
    c = make(dev, 1500, lens, 16, 2, seed=10)
    want = call(c)
    lib = N.lib()
    need = lib.fk_shared_prefix_workspace_bytes(0, len(lens), 16, 2, 128, N.FK_DTYPE_F16)
    ws = torch.full((need // 4,), word, dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.empty_like(want)
    stream = N.stream_of(dev)
    assert lib.fk_debug_configure(100_000_000, 1) == 0
    try:
        assert lib.fk_paged_shared_prefix_decode(entry_args(c, out, status), ws.data_ptr(), need, stream) == 0
        torch.cuda.synchronize()
    finally:
        assert lib.fk_debug_configure(4_000_000_000, 0) == 0
    assert int(status) == N.FK_STATUS_TIMEOUT
    status.zero_()
    assert lib.fk_paged_shared_prefix_decode(entry_args(c, out, status), ws.data_ptr(), need, stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want) and int(status) == 0


@gpu
def test_wrapper_refusals(dev):
    c = make(dev, 100, [20, 7], 8, 2, seed=1)
    q, k, v, table, bt, seq = c["q"], c["k"], c["v"], c["table"], c["bt"], c["seq"]
    f = fk.paged_flash_decode_shared_prefix
    bad = [
        lambda: f(q[0], k, v, table, 100, bt, seq, 16),
        lambda: f(q, k[0], v, table, 100, bt, seq, 16),
        lambda: f(q, k, v[:1], table, 100, bt, seq, 16),
        lambda: f(q, k, v.bfloat16(), table, 100, bt, seq, 16),
        lambda: f(q.bfloat16(), k, v, table, 100, bt, seq, 16),
        lambda: f(q.float(), k, v, table, 100, bt, seq, 16),
        lambda: f(q, k, v, table, 100, bt, seq, 32),
        lambda: f(q[:, :7], k, v, table, 100, bt, seq, 16),
        lambda: f(q[..., :64], k, v, table, 100, bt, seq, 16),
        lambda: f(q[..., :64], k[..., :64].to(E4M3), v[..., :64].to(E4M3), table, 100, bt, seq, 16),
        lambda: f(q, k, v, table[None], 100, bt, seq, 16),
        lambda: f(q, k, v, table.cpu(), 100, bt, seq, 16),
        lambda: f(q, k, v, table, 113, bt, seq, 16),
        lambda: f(q, k, v, table, -1, bt, seq, 16),
        lambda: f(q, k, v, table, seq, bt, seq, 16),
        lambda: f(q, k, v, table, 100, bt[:1], seq, 16),
        lambda: f(q, k, v, table, 100, bt.cpu(), seq, 16),
        lambda: f(q, k, v, table, 100, bt, seq[:1], 16),
        lambda: f(q, k, v, table, 100, bt, seq.cpu(), 16),
        lambda: f(q, k, v, table, 100, bt, seq, 16, s_aux=torch.zeros(7, device=dev)),
        lambda: f(q, k, v, table, 100, bt, seq, 16, out=torch.empty(2, 8, 64, dtype=q.dtype, device=dev)),
        lambda: f(q, k, v, table, 100, bt, seq, 16, out_dtype=torch.float32),
        lambda: f(q.detach().requires_grad_(), k, v, table, 100, bt, seq, 16),
    ]
    for i, one in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            one()
            pytest.fail(f"call {i} was not refused")


# ------------------------------------------------------------------ CPU: refusals of the C entry
_FIELDS = ("q k_pool v_pool prefix_table prefix_len_dev block_table seq_lens s_aux out scale_q scale_k scale_v status "
           "prefix_len prefix_blocks batch q_heads kv_heads head_dim num_pages max_blocks q_dtype kv_dtype out_dtype "
           "q_b q_h kp_p kp_h kp_s vp_p vp_h vp_s bt_b o_b o_h").split()


def _args(**kw):
    a = dict.fromkeys(_FIELDS, 0)
    a.update(q=16, k_pool=16, v_pool=16, prefix_table=16, block_table=16, seq_lens=16, out=16, prefix_len=16,
             prefix_blocks=1, batch=1, q_heads=2, kv_heads=1, head_dim=128, num_pages=4, max_blocks=1)
    a.update(kw)
    return struct.pack("13Q22q", *(a[f] for f in _FIELDS))


@pytest.mark.parametrize("kw, rc, msg", [
    (dict(batch=-1), 1, "bad sizes"),
    (dict(q_heads=0), 1, "bad sizes"),
    (dict(batch=2 ** 31), 1, "bad sizes"),
    (dict(num_pages=0), 1, "page counts"),
    (dict(prefix_blocks=-1), 1, "page counts"),
    (dict(prefix_len=-1), 1, "page counts"),
    (dict(max_blocks=-1), 1, "page counts"),
    (dict(prefix_table=0), 1, "prefix_table"),
    (dict(q=0), 1, "non-null"),
    (dict(head_dim=96), 2, "head_dim"),
    (dict(head_dim=64, kv_dtype=2), 2, "head_dim"),
    (dict(q_heads=3, kv_heads=2), 1, "multiple"),
    (dict(kv_dtype=3), 2, "kv dtype"),
    (dict(q_dtype=1), 1, "q dtype"),
    (dict(out_dtype=2), 2, "out dtype"),
    (dict(k_pool=8), 1, "16-byte aligned"),
])
def test_c_entry_refuses_bad_arguments_without_a_device(kw, rc, msg):
    assert N.lib().fk_paged_shared_prefix_decode(_args(**kw), 256, 1 << 30, None) == rc
    assert msg in N.last_error()


def test_c_entry_without_workspace_and_for_an_empty_batch():
    assert N.lib().fk_paged_shared_prefix_decode(_args(), None, 0, None) == 3
    assert N.lib().fk_paged_shared_prefix_decode(_args(batch=0, q=0), None, 0, None) == 0
    assert N.lib().fk_paged_shared_prefix_decode(None, None, 0, None) == 1
    assert N.lib().fk_shared_prefix_workspace_bytes(0, 4, 36, 8, 128, 0) == 0 and "bad sizes" in N.last_error()


def test_wrapper_refuses_cpu_tensors():
    q, k = torch.zeros(1, 4, 128, dtype=torch.float16), torch.zeros(2, 2, 16, 128, dtype=torch.float16)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fk.paged_flash_decode_shared_prefix(q, k, k, i[0], 1, i, i[0], 16)
