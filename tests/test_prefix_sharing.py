"""Sequences that share pages: PagedKVCache's bookkeeping (CPU), and the step of
a layer as a server runs it (GPU): norm, rotate and append into forked
sequences, decode behind the shared prefix, through the cache and through the
paged adapter."""
import pytest
import torch

import fasterkernels_b200 as fk
from fasterkernels_b200.paged_attn import PAGE_SIZE, PagedKVCache, paged_kv_append
from fasterkernels_b200.paged_attn.shared_prefix import shared_prefix_pays
from _operator_refs import attention_bound, norm_rope_ref, shared_prefix_ref

gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def make(pages=12, seqs=4, blocks=6, device="cpu", dtype=torch.float16, layers=2, heads=2, head_dim=128):
    return PagedKVCache(num_layers=layers, num_pages=pages, max_seqs=seqs, max_blocks_per_seq=blocks, num_kv_heads=heads,
                        head_dim=head_dim, dtype=dtype, device=device)


def prefill(c, sid, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(c.num_kv_heads, n, c.head_dim, generator=g).to(c.dtype)
    for layer in range(c.num_layers):
        c.write_prefill(sid, layer, k, k)
    return k


# ------------------------------------------------------------------ CPU
def test_fork_shares_full_pages_and_frees_them_with_the_last_holder():
    c = make()
    a = c.allocate_sequence()
    prefill(c, a, 40)
    assert c.pages_used == 3
    b = c.fork_sequence(a, 32)
    d = c.fork_sequence(b, 16)
    assert c.pages_used == 3 and (c.seq_len(b), c.seq_len(d)) == (32, 16)
    assert c.block_table[b].tolist()[:3] == c.block_table[a].tolist()[:2] + [-1]
    assert (c.shared_prefix_pages([a, b]), c.shared_prefix_pages([a, b, d]), c.shared_prefix_pages([d, a])) == (2, 1, 1)
    # new tokens go to pages of their own
    bt, pos, lens = c.begin_step([a, b, d])
    assert pos.tolist() == [40, 32, 16] and lens.tolist() == [41, 33, 17]
    c.end_step()
    assert c.pages_used == 5 and len(set(c._pages[b]) & set(c._pages[a])) == 2
    assert c.shared_prefix_pages([a, b]) == 2
    free = c.pages_free
    c.free_sequence(a)  # b and d still hold its first pages
    assert c.pages_free == free + 1
    assert c.shared_prefix_pages([b, d]) == 1
    c.free_sequence(d)
    assert c.pages_free == free + 2
    c.free_sequence(b)
    assert c.pages_free == c.num_pages and sorted(c._free_pages) == list(range(c.num_pages)) and not c._page_refs


def test_fork_refusals():
    c = make()
    a = c.allocate_sequence()
    prefill(c, a, 40)
    for n in (0, -16, 17, 48):
        with pytest.raises(ValueError, match="multiple"):
            c.fork_sequence(a, n)
    with pytest.raises(ValueError, match="active"):
        c.fork_sequence(3, 16)
    with pytest.raises(ValueError, match="active"):
        c.fork_sequence(99, 16)
    for _ in range(3):
        c.fork_sequence(a, 16)
    with pytest.raises(RuntimeError, match="occupied"):
        c.fork_sequence(a, 16)
    assert all(n == 4 for n in c._page_refs.values())  # a refused fork takes no reference
    with pytest.raises(RuntimeError, match="shared"):
        prefill(c, a, 40)
    with pytest.raises(RuntimeError, match="shared"):
        prefill(c, 1, 5)


def test_an_empty_prefill_of_a_sequence_with_shared_pages_is_refused():
    c = make(layers=1)
    a = c.allocate_sequence()
    prefill(c, a, 40)
    b = c.fork_sequence(a, 32)
    before = c.k_pool.clone()
    for sid in (a, b):
        with pytest.raises(RuntimeError, match="shared"):
            c.write_prefill(sid, 0, c.k_pool.new_zeros(2, 0, 128), c.k_pool.new_zeros(2, 0, 128))
    assert (c.seq_len(a), c.seq_len(b), c.shared_prefix_pages([a, b])) == (40, 32, 2)
    c.append_kv(b, 0, torch.ones(1, 2, 1, 128), torch.ones(1, 2, 1, 128))
    pages = c.block_table[a, :3].long()
    assert torch.equal(c.k_pool[0, pages], before[0, pages])
    c.free_sequence(b)  # a holds its pages alone again
    c.write_prefill(a, 0, c.k_pool.new_zeros(2, 0, 128), c.k_pool.new_zeros(2, 0, 128))
    assert c.seq_len(a) == 0


def test_shared_prefix_of_unrelated_single_and_repeated_sequences():
    c = make()
    a, b = c.allocate_sequence(), c.allocate_sequence()
    assert c.shared_prefix_pages([]) == 0 and c.shared_prefix_pages([a]) == 0 and c.shared_prefix_pages([a, b]) == 0
    prefill(c, a, 40)
    prefill(c, b, 40)
    assert c.shared_prefix_pages([a, b]) == 0 and c.shared_prefix_pages([a]) == 2 and c.shared_prefix_pages([a, a]) == 2
    assert not shared_prefix_pays(1, 10 ** 6) and not shared_prefix_pays(2, 0) and shared_prefix_pays(64, 32768)


@pytest.mark.parametrize("batch,prefix,own,kw,pays", [
    (2, 2048, 64, dict(), True), (16, 2048, 64, dict(), True), (64, 16384, 64, dict(), True), (2, 256, 64, dict(), False),
    (2, 16384, 64, dict(kv_dtype=E4M3), False), (2, 4096, 64, dict(head_dim=64), False), (16, 4096, 64, dict(head_dim=64), True),
    (4, 16384, 64, dict(q_heads=8, kv_heads=1), False), (64, 16384, 64, dict(q_heads=8, kv_heads=1), True),
    (4, 4096, 1000, dict(), False), (16, 4096, 1000, dict(), True), (2, 16384, 1000, dict(), False),
    (2, 2048, 64, dict(q_heads=64, kv_dtype=E4M3), True), (2, 2048, 64, dict(q_heads=128), True)])
def test_the_shared_path_is_taken_where_it_measured_faster(batch, prefix, own, kw, pays):
    """Sizes at which the two ways are 3 % or more apart, in times measured."""
    assert shared_prefix_pays(batch, prefix, own, **kw) == pays


def test_begin_chunk_places_ragged_tokens_and_commits_their_counts():
    c = make()
    a, b, d = (c.allocate_sequence() for _ in range(3))
    prefill(c, a, 14)
    bt, pos, seq = c.begin_chunk([a, b, d], [5, 0, 17])
    assert pos.tolist() == [14, 15, 16, 17, 18] + list(range(17)) and seq.tolist() == [0] * 5 + [2] * 17
    assert (bt[0, :2] >= 0).all() and (bt[1] == -1).all() and (bt[2, :2] >= 0).all() and (bt[2, 2:] == -1).all()
    with pytest.raises(RuntimeError, match="begin_step"):
        c.append_kv_batch(0, torch.zeros(22, 2, 128), torch.zeros(22, 2, 128))
    assert c.end_step().tolist() == [19, 0, 17]
    used = c.pages_used
    with pytest.raises(RuntimeError, match="Out of KV pages"):
        c.begin_chunk([a, b], [60, 96])
    with pytest.raises(RuntimeError, match="max_blocks"):
        c.begin_chunk([b], [97])
    with pytest.raises(ValueError, match="once"):
        c.begin_chunk([a, a], [1, 1])
    with pytest.raises(ValueError, match="counts"):
        c.begin_chunk([a, b], [1])
    assert c.pages_used == used  # a refused chunk takes no page
    with pytest.raises(RuntimeError, match="begin_chunk"):
        c.append_qkv_batch(0, None, None, None, None, None)


@pytest.mark.parametrize("chunk", [False, True])
def test_a_step_past_the_cos_sin_rows_is_refused_before_anything_is_appended(chunk):
    c = make(layers=1)
    a, b = c.allocate_sequence(), c.allocate_sequence()
    prefill(c, a, 40)
    prefill(c, b, 7)
    before = c.k_pool.clone()
    T = 6 if chunk else 2
    x = torch.zeros(T, 2, 128, dtype=c.dtype)
    if chunk:
        c.begin_chunk([b, a], [4, 2])  # positions 7 .. 10 and 40, 41
    else:
        c.begin_step([b, a])           # 7 and 40
    table = torch.zeros(41 if chunk else 40, 64)
    with pytest.raises(ValueError, match=f"position {41 if chunk else 40}"):
        c.append_qkv_batch(0, x, x, x, table, table)
    assert torch.equal(c.k_pool, before) and (c.seq_len(a), c.seq_len(b)) == (40, 7)
    with pytest.raises(ValueError, match="CUDA"):  # one more row, or no rotation: on to the kernel's own checks
        c.append_qkv_batch(0, x, x, x, *(torch.zeros(42, 64) for _ in range(2)))
    with pytest.raises(ValueError, match="CUDA"):
        c.append_qkv_batch(0, x, x, x, None, None)
    c.end_step()


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _check_attention(got, q, k, v, prefix, lens, p_dtype):
    """got against attention of q over per-sequence k / v [B, KVH, T, D] (the
    first `prefix` tokens are sequence 0's for all)."""
    kp, vp = k[0, :, :prefix], v[0, :, :prefix]
    args = (q.double(), kp, vp, prefix, k[:, :, prefix:], v[:, :, prefix:], [n - prefix for n in lens])
    ref = shared_prefix_ref(*args)
    bound = attention_bound(*args, None, ref, p_dtype, got.dtype)
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())


def _gathered(c, layer, ids, width):
    bt = c.get_block_table_tensor(ids).long().clamp(min=0)[:, : (width + 15) // 16]
    out = []
    for pool, s in ((c.k_pool, c.k_scale), (c.v_pool, c.v_scale)):
        x = pool[layer][bt].float().double() * (s.double() if c.dtype == E4M3 else 1.0)
        out.append(x.transpose(1, 2).reshape(len(ids), c.num_kv_heads, -1, c.head_dim))
    return out


@gpu
@pytest.mark.parametrize("dtype,pool", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, E4M3)])
def test_prompt_then_forked_steps_together(dev, dtype, pool):
    """A prompt appended in chunks with norms and rotation, forked four times,
    then three steps: rotate + append + shared-prefix decode, each against 64
    bits on what the cache holds."""
    L, KVH, QH, D, P = 2, 4, 16, 128, 150
    c = make(pages=64, seqs=6, blocks=16, device=str(dev), dtype=pool, layers=L, heads=KVH)
    if pool == E4M3:
        c.set_fp8_scales(0.02, 0.02)
    g = torch.Generator(device=dev).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    cos, sin = fk.rope_table(512, D, device=dev)
    qw, kw = (1 + 0.2 * rnd(D)).to(dtype), (1 + 0.2 * rnd(D)).to(dtype)
    a = c.allocate_sequence()
    prompt = [(1.5 * rnd(P, QH + 2 * KVH, D)).to(dtype) for _ in range(L)]
    cut = lambda x: (x[:, :QH], x[:, QH:QH + KVH], x[:, QH + KVH:])  # noqa: E731
    for lo, hi in ((0, 70), (70, P)):
        c.begin_chunk([a], [hi - lo])
        for layer in range(L):
            q, k, v = cut(prompt[layer][lo:hi])
            k_out = torch.empty(hi - lo, KVH, D, dtype=dtype, device=dev)
            q_out = c.append_qkv_batch(layer, q, k, v, cos, sin, q_weight=qw, k_weight=kw, k_out=k_out)
            both = fk.qk_norm_rope(q, k, cos, sin, torch.arange(lo, hi, device=dev), q_weight=qw, k_weight=kw)
            assert torch.equal(q_out, both[0]) and torch.equal(k_out, both[1])
        c.end_step()
    assert c.seq_len(a) == P
    n = P // PAGE_SIZE * PAGE_SIZE
    ids = [c.fork_sequence(a, n) for _ in range(4)]
    ref_rows = norm_rope_ref(cut(prompt[1])[1], cos, sin, torch.arange(P, device=dev), kw)[0]
    kk, _ = _gathered(c, 1, [ids[2]], n)
    step = {torch.float16: 2 ** -10, torch.bfloat16: 2 ** -7, E4M3: 2 ** -3}[pool]
    assert float((kk[0].transpose(0, 1) - ref_rows[:n]).abs().max()) <= step * float(ref_rows.abs().max())
    for s in range(3):
        bt, pos, lens = c.begin_step(ids)
        shared = c.shared_prefix_pages(ids)
        assert shared == n // PAGE_SIZE
        for layer in range(L):
            q, k, v = cut((1.5 * rnd(4, QH + 2 * KVH, D)).to(dtype))
            qr = c.append_qkv_batch(layer, q, k, v, cos, sin, q_weight=qw, k_weight=kw)
            kw8 = dict(scale_k=c.k_scale, scale_v=c.v_scale) if pool == E4M3 else {}
            out = fk.paged_flash_decode_shared_prefix(qr, c.k_pool[layer], c.v_pool[layer], bt[0, :shared], n, bt[:, shared:],
                                                      lens - n, PAGE_SIZE, **kw8)
            ks, vs = _gathered(c, layer, ids, n + s + 1)
            _check_attention(out, qr, ks, vs, n, lens.tolist(), torch.bfloat16 if pool == torch.bfloat16 else torch.float16)
        c.end_step()
    assert fk.read_status() == 0


@gpu
@pytest.mark.parametrize("graphed", [False, True])
def test_inputs_written_right_before_the_call(dev, graphed):
    """What precedes the call in the stream writes what it reads, its prefix
    too: a torch op writes q and a prefix page, the append kernel the step's
    token; 200 steps, each against the same decode after a synchronisation."""
    B, QH, KVH, D, P = 6, 16, 4, 128, 1600
    g = torch.Generator(device=dev).manual_seed(9)
    n = P // 16
    pages = n + 4 * B
    kp = torch.randn(pages, KVH, 16, D, generator=g, device=dev).half()
    vp = torch.randn(pages, KVH, 16, D, generator=g, device=dev).half()
    table = torch.arange(n, dtype=torch.int32, device=dev)
    bt = (n + torch.arange(4 * B, dtype=torch.int32, device=dev)).view(B, 4)
    q = torch.zeros(B, QH, D, dtype=torch.float16, device=dev)
    pos = torch.zeros(B, dtype=torch.int32, device=dev)
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    src = torch.randn(3, B, max(QH, KVH), D, generator=g, device=dev).half()
    page = torch.zeros(1, dtype=torch.int64, device=dev)
    fresh = torch.randn(2, 1, KVH, 16, D, generator=g, device=dev).half()
    plen = torch.tensor([P - 3], dtype=torch.int32, device=dev)

    def decode():
        return fk.paged_flash_decode_shared_prefix(q, kp, vp, table, plen, bt, lens, 16)

    def step():
        kp.index_copy_(0, page, fresh[0])
        vp.index_copy_(0, page, fresh[1])
        q.copy_(src[0])
        paged_kv_append(src[1][:, :KVH], src[2][:, :KVH], kp, vp, bt, pos)
        torch.add(pos, 1, out=lens)
        return decode()

    step()
    out = None
    if graphed:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    for i in range(200):
        src.normal_(generator=g)
        fresh.normal_(generator=g)
        pos.fill_(i % 64)
        page.fill_((7 * i) % n)
        if graphed:
            graph.replay()
        else:
            out = step()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, decode()), i
    assert fk.read_status() == 0


@gpu
def test_the_cache_reports_what_a_step_could_not_append(dev):
    """A step whose positions or pages change behind the cache's back (here by
    hand, as a replayed graph could) leaves its bit in read_status()."""
    from fasterkernels_b200 import _native as N
    c = make(pages=8, device=str(dev), layers=1)
    a = c.allocate_sequence()
    x = torch.randn(1, 2, 128, device=dev).half()
    cos, sin = fk.rope_table(64, 128, device=dev)
    fk.read_status()
    for what, bit in ((None, 0), ("pos", N.FK_STATUS_BAD_POSITION), ("bt", N.FK_STATUS_BAD_PAGE)):
        c.begin_step([a])
        if what == "pos":
            c._step_pos.fill_(64)
        elif what == "bt":
            c._step_bt.fill_(-1)
        c.append_qkv_batch(0, x, x, x, cos, sin)
        c.end_step()
        assert fk.read_status() == bit
    mine = torch.zeros(1, dtype=torch.int32, device=dev)
    c.begin_step([a])
    c._step_pos.fill_(-1)
    c.append_qkv_batch(0, x, x, x, cos, sin, status=mine)
    assert int(mine) == N.FK_STATUS_BAD_POSITION and fk.read_status() == 0


def test_kept_words_can_be_written_in_any_mode():
    from fasterkernels_b200 import _native as N
    with torch.inference_mode():
        w = N._kept_zeros(3, torch.int32, "cpu")
        w[:1].fill_(1)
    w[1:2].fill_(2)
    with torch.inference_mode():
        w[2:].fill_(3)
    assert w.tolist() == [1, 2, 3] and not w.is_inference()


@gpu
def test_read_status_after_first_calls_under_inference_mode(dev):
    """The status word and the decode workspace are made by whoever calls first."""
    from fasterkernels_b200 import _native as N
    kept = dict(N._status), dict(N._ws)
    N._status.clear()
    N._ws.clear()
    try:
        with torch.inference_mode():
            q, kp = torch.randn(2, 4, 128, device=dev).half(), torch.randn(4, 2, 16, 128, device=dev).half()
            bt = torch.tensor([[1], [-1]], dtype=torch.int32, device=dev)
            lens = torch.tensor([5, 5], dtype=torch.int32, device=dev)
            fk.paged_flash_decode(q, kp, kp, bt, lens, 16)
            fk.paged_flash_decode_shared_prefix(q, kp, kp, bt[0], 16, bt, lens, 16)
        assert fk.read_status() == N.FK_STATUS_BAD_PAGE and fk.read_status() == 0
        with torch.inference_mode():
            fk.paged_flash_decode_shared_prefix(q, kp, kp, bt[0], 16, bt, lens, 16)
            assert fk.read_status() == N.FK_STATUS_BAD_PAGE and fk.read_status() == 0
    finally:
        for d, k in zip((N._status, N._ws), kept):
            d.update(k)


@gpu
def test_the_first_append_of_a_cache_can_be_a_captured_one(dev):
    from fasterkernels_b200 import _native as N
    words = dict(N._status)
    N._status.clear()
    try:
        c = make(pages=8, device=str(dev), layers=1)
        a = c.allocate_sequence()
        x = torch.randn(1, 2, 128, device=dev).half()
        cos, sin = fk.rope_table(64, 128, device=dev)
        c.begin_step([a])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q = c.append_qkv_batch(0, x, x, x, cos, sin)
        graph.replay()
        assert torch.equal(q, x) and torch.equal(c.k_pool[0, c._pages[a][0], :, 0], x[0]) and fk.read_status() == 0
    finally:
        N._status.update(words)


@gpu
@pytest.mark.parametrize("inject", [0, 4])
@pytest.mark.parametrize("graphed", [False, True])
def test_inputs_written_right_before_the_call_against_64_bits(dev, graphed, inject):
    """Every input of a step is written by the kernels right before it: q, a page
    of the prefix, the own tokens, both tables, both lengths.  Against attention
    over what was written, with the prefix kernel taking the own part's word for
    it (inject 0) and waiting for it (4)."""
    from fasterkernels_b200 import _native as N
    B, QH, KVH, D, blocks = 3, 4, 2, 128, 20
    g = torch.Generator(device=dev).manual_seed(19)
    pages = blocks + 2 * B
    kp, vp = (torch.randn(pages, KVH, 16, D, generator=g, device=dev).half() for _ in range(2))
    src_k, src_v = kp.clone(), vp.clone()
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table, bt = perm[:blocks].clone(), perm[blocks:].view(B, 2).clone()
    src_table, src_bt = table.clone(), bt.clone()
    q, src_q = (torch.randn(B, QH, D, generator=g, device=dev).half() for _ in range(2))
    lens, src_lens = (torch.zeros(B, dtype=torch.int32, device=dev) for _ in range(2))
    plen, src_plen = (torch.full((1,), 16 * blocks, dtype=torch.int32, device=dev) for _ in range(2))

    def step():
        for dst, src in ((kp, src_k), (vp, src_v), (table, src_table), (bt, src_bt), (lens, src_lens), (plen, src_plen), (q, src_q)):
            dst.copy_(src)
        return fk.paged_flash_decode_shared_prefix(q, kp, vp, table, plen, bt, lens, 16)

    lib = N.lib()
    assert lib.fk_debug_configure(4_000_000_000, inject) == 0
    try:
        out = step()
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        for i in range(40):
            src_q.normal_(generator=g)
            src_k.normal_(generator=g)
            src_v.normal_(generator=g)
            perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
            src_table.copy_(perm[:blocks])
            src_bt.copy_(perm[blocks:].view(B, 2))
            own, prefix = [(5 * i + 11 * b) % 33 for b in range(B)], 1 + (37 * i) % (16 * blocks)
            src_lens.copy_(torch.tensor(own))
            src_plen.fill_(prefix)
            torch.cuda.synchronize()
            if graphed:
                graph.replay()
            else:
                out = step()
            pk, pv = (x[src_table.long()].transpose(0, 1).reshape(KVH, -1, D) for x in (src_k, src_v))
            tk, tv = (x[src_bt.long()].transpose(1, 2).reshape(B, KVH, -1, D) for x in (src_k, src_v))
            args = (src_q.double(), pk, pv, prefix, tk, tv, own)
            ref = shared_prefix_ref(*args)
            bound = attention_bound(*args, None, ref, torch.float16, out.dtype)
            assert bool(((out.double() - ref).abs() <= bound).all()), i
    finally:
        assert lib.fk_debug_configure(4_000_000_000, 0) == 0
    assert fk.read_status() == 0


class _Module:
    is_causal = True

    def __init__(self, layer_idx):
        self.layer_idx = layer_idx
        self.num_key_value_groups = 4


@gpu
@pytest.mark.parametrize("forked", [False, True])
def test_paged_adapter_with_queries_that_require_grad(dev, forked):
    """A model run without no_grad: the same step as under it, forks or not."""
    outs = []
    for grad in (False, True):
        c = make(pages=2 * 290, seqs=3, blocks=290, device=str(dev), layers=2)
        g = torch.Generator(device=dev).manual_seed(15)
        k = torch.randn(2, 2, 2, 4416, 128, generator=g, device=dev).half()
        a = c.allocate_sequence()
        for layer in range(2):
            c.write_prefill(a, layer, k[layer, 0], k[layer, 1])
        ids = [a, c.fork_sequence(a, 4416)] if forked else [a]
        q = torch.randn(len(ids), 8, 1, 128, generator=g, device=dev).half().requires_grad_(grad)
        kv = torch.randn(2, len(ids), 2, 1, 128, generator=g, device=dev).half().requires_grad_(grad)
        fk.set_paged_attention_cache(c, ids)
        try:
            outs.append([fk.custom_paged_attention_forward(_Module(i), q, kv[0], kv[1], None, 128 ** -0.5)[0] for i in range(2)])
        finally:
            fk.set_paged_attention_cache(None, [])
        assert [c.seq_len(s) for s in ids] == [4417] * len(ids)
    for x, y in zip(*outs):
        assert torch.equal(x, y) and not y.requires_grad


@gpu
def test_paged_adapter_leaves_the_shared_path_where_tails_are_long(dev, monkeypatch):
    """The same forks with short and long own parts: the rule is asked with what is bound."""
    from fasterkernels_b200.paged_attn import paged_adapter
    asked = []
    monkeypatch.setattr(paged_adapter, "shared_prefix_pays", lambda *a, **k: asked.append((a, k)) or shared_prefix_pays(*a, **k))
    taken = []
    real = paged_adapter.paged_flash_decode_shared_prefix
    monkeypatch.setattr(paged_adapter, "paged_flash_decode_shared_prefix", lambda *a, **k: taken.append(a[4]) or real(*a, **k))
    c = make(pages=4 * 120, seqs=5, blocks=140, device=str(dev), layers=1, heads=8)
    a = c.allocate_sequence()
    k = torch.randn(8, 1024, 128, device=dev).half()
    c.write_prefill(a, 0, k, k)
    ids = [c.fork_sequence(a, 1024) for _ in range(4)]
    for tail in (20, 980):
        c.begin_chunk(ids, [tail] * 4)
        x = torch.randn(4 * tail, 8, 128, device=dev).half()
        c.append_qkv_batch(0, x, x, x, None, None)
        c.end_step()
        fk.set_paged_attention_cache(c, ids)
        try:
            q = torch.randn(4, 32, 1, 128, device=dev).half()
            x = torch.randn(4, 8, 1, 128, device=dev).half()
            fk.custom_paged_attention_forward(_Module(0), q, x, x, None, 128 ** -0.5)
        finally:
            fk.set_paged_attention_cache(None, [])
    heads = dict(q_heads=32, kv_heads=8, head_dim=128, kv_dtype=torch.float16)
    assert asked == [((4, 1024, 21), heads), ((4, 1024, 1002), heads)] and taken == [1024]


@gpu
@pytest.mark.parametrize("pool", [torch.float16, E4M3])
def test_paged_adapter_decodes_forked_sequences_behind_their_prefix(dev, pool, monkeypatch):
    """Forked sequences through the adapter give what unforked copies of them
    give, and only the forked ones take the shared path."""
    from fasterkernels_b200.paged_attn import paged_adapter
    B, L, P = 5, 2, 4400
    calls = []
    real = paged_adapter.paged_flash_decode_shared_prefix
    monkeypatch.setattr(paged_adapter, "paged_flash_decode_shared_prefix", lambda *a, **k: calls.append(a[4]) or real(*a, **k))
    outs, caches = [], []
    for forked in (True, False):
        c = make(pages=6 * 300, seqs=6, blocks=290, device=str(dev), dtype=pool, layers=L, heads=2)
        if pool == E4M3:
            c.set_fp8_scales(0.02, 0.02)
        g = torch.Generator(device=dev).manual_seed(5)
        k = torch.randn(L, 2, 2, P, 128, generator=g, device=dev).half()
        n = P // 16 * 16
        if forked:
            a = c.allocate_sequence()
            for layer in range(L):
                c.write_prefill(a, layer, k[layer, 0], k[layer, 1])
            ids = [c.fork_sequence(a, n) for _ in range(B)]
        else:
            ids = [c.allocate_sequence() for _ in range(B)]
            for sid in ids:
                for layer in range(L):
                    c.write_prefill(sid, layer, k[layer, 0, :, :n], k[layer, 1, :, :n])
        fk.set_paged_attention_cache(c, ids)
        got = []
        try:
            for step in range(3):
                for layer in range(L):
                    q = torch.randn(B, 8, 1, 128, generator=g, device=dev).half()
                    kv = torch.randn(2, B, 2, 1, 128, generator=g, device=dev).half()
                    o, _ = fk.custom_paged_attention_forward(_Module(layer), q, kv[0], kv[1], None, 128 ** -0.5)
                    assert o.shape == (B, 8, 1, 128)
                    got.append((q.squeeze(2), layer, o.squeeze(2), [c.seq_len(s) + (layer < L - 1) for s in ids]))
        finally:
            fk.set_paged_attention_cache(None, [])
        outs.append(got)
        caches.append((c, ids, n))
    assert calls == [n] * (3 * L)
    for (q, layer, a, lens), (_, _, b, _) in zip(*outs):
        c, ids, n = caches[0]
        ks, vs = _gathered(c, layer, ids, n + 3)
        for got in (a, b):
            _check_attention(got, q, ks, vs, n, lens, torch.float16)
