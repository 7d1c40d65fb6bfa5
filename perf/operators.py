"""What the serving operators around a decode step cost: the position rotation
(with the per-head norms) of queries and keys, the same on the way into a paged
KV cache, and decode attention of a batch that shares a prefix.

``own = False`` computes each operator in plain torch in 32 bits; ``own =
True`` calls the framework's kernels.  Both take the same prepared state.
"""
import math

import torch

own = False

PAGE = 16
EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------- the cases
def listed():
    rot = {"op": "rope", "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "interleaved": False,
           "norm": True, "packed": True, "max_pos": 32768, "dtype": "bf16"}
    app = {"op": "append", "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "interleaved": False,
           "norm": True, "packed": True, "max_pos": 32768, "dtype": "bf16", "pool": "bf16"}
    pre = {"op": "prefix", "q_heads": 32, "kv_heads": 8, "head_dim": 128, "dtype": "f16", "pool": "f16", "sinks": False}
    return [
        # one decode step of 32 sequences on a contiguous cache: a few tokens, all latency
        dict(rot, name="rope_step", tokens=32),
        # the prompts of a batch in one pass: bound by memory
        dict(rot, name="rope_prompt", tokens=16384),
        # heads of 64, a rotation of the first 32 dims in adjacent pairs, no norms, odd counts
        dict(rot, name="rope_odd", tokens=4099, q_heads=12, kv_heads=3, head_dim=64, rotary=32, interleaved=True,
             norm=False, packed=False, dtype="f16"),
        # one decode step of 64 sequences into 16-bit pages
        dict(app, name="append_step", seqs=64, tokens=64, context=2000, dtype="f16", pool="f16"),
        # one decode step of 128 sequences of 64 query heads into e4m3 pages
        dict(app, name="append_step_e4m3", seqs=128, tokens=128, context=1000, q_heads=64, dtype="f16", pool="e4m3"),
        # prompt chunks of 8 sequences, each continuing at its own position
        dict(app, name="append_prompt", seqs=8, tokens=16384, context=1000),
        # the same into e4m3 pages, with ragged odd counts, a partial rotation and no norms
        dict(app, name="append_odd_e4m3", seqs=5, tokens=6007, context=333, q_heads=24, kv_heads=4, rotary=64,
             norm=False, packed=False, pool="e4m3"),
        # a handful of samples of one short prompt: latency
        dict(pre, name="prefix_few", batch=4, prefix=1000, tail=40),
        # 64 requests behind one long system prompt, 16-bit pages
        dict(pre, name="prefix_batch", batch=64, prefix=32768, tail=512),
        # 128 requests of 64 query heads behind a very long document, e4m3 pages with sinks
        dict(pre, name="prefix_long_e4m3", batch=128, q_heads=64, prefix=65536, tail=1000, pool="e4m3", sinks=True),
        # two samples of a very long document: bound by reading it once
        dict(pre, name="prefix_two", batch=2, prefix=131072, tail=100, dtype="bf16", pool="bf16"),
        # heads of 64, an odd group, a prefix that ends inside a page
        dict(pre, name="prefix_odd", batch=37, q_heads=15, kv_heads=3, head_dim=64, prefix=5003, tail=77, dtype="bf16",
             pool="bf16", sinks=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "prefix"])
    head_dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8])
    c = {"op": op, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": rng.choice(["f16", "bf16"])}
    if op == "prefix":
        c["q_heads"] = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
        c["batch"] = _log(rng, 1, 160)
        most = 128 * 64 * 65536 // (c["batch"] * c["q_heads"])
        c["prefix"] = _log(rng, 1, min(131072, most))
        c["tail"] = _log(rng, 1, 1024)
        c["pool"] = rng.choice(["e4m3", c["dtype"]]) if head_dim == 128 else c["dtype"]
        c["sinks"] = rng.random() < 0.5
        return c
    c["q_heads"] = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    c["rotary"] = rng.choice([r for r in (16, 32, 48, 64, 96, 128) if r <= head_dim] + [head_dim])
    c["interleaved"] = rng.random() < 0.3
    c["norm"] = rng.random() < 0.6
    c["packed"] = rng.random() < 0.5
    most = 16384 * 48 * 128 // ((c["q_heads"] + 2 * kv_heads) * head_dim)
    c["tokens"] = _log(rng, 1, min(16384, most))
    c["max_pos"] = 32768
    if op == "append":
        c["seqs"] = c["tokens"] if c["tokens"] <= 256 and rng.random() < 0.7 else min(c["tokens"], _log(rng, 1, 32))
        c["context"] = _log(rng, 1, 2000) if c["seqs"] <= 64 else _log(rng, 1, 500)
        c["pool"] = rng.choice(["e4m3", c["dtype"]])
    return c


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _table(case):
    # angles of far positions lose their fraction in 32 bits: made in 64, kept in 32
    half = case["rotary"] // 2
    freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    ang = torch.arange(case["max_pos"], dtype=torch.float64, device="cuda")[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def _heads(case, g, with_v):
    T, D, H, K = case["tokens"], case["head_dim"], case["q_heads"], case["kv_heads"]
    dt = DTYPES[case["dtype"]]
    if case["packed"]:  # one projection's output, cut into q, k (and v)
        qkv = (1.5 * _randn(g, T, (H + 2 * K) * D)).to(dt).view(T, H + 2 * K, D)
        q, k, v = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
    else:
        q, k, v = ((1.5 * _randn(g, T, n, D)).to(dt) for n in (H, K, K))
    return (q, k, v) if with_v else (q, k)


def _pages(g, pages, most):
    pool = most + most // 4 + 1  # a quarter more than any seed's lengths need, in random order
    return pool, torch.randperm(pool, generator=g, device="cuda")[:pages].to(torch.int32)


def _pool(g, pool, case):
    shape = (pool, case["kv_heads"], PAGE, case["head_dim"])
    return _randn(g, *shape).to(DTYPES[case["pool"]])


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "prefix":
        return _prepare_prefix(case, g)
    s = {"case": case}
    s["cos"], s["sin"] = _table(case)
    dt = DTYPES[case["dtype"]]
    s["qw"] = s["kw"] = None
    if case["norm"]:
        s["qw"], s["kw"] = ((1 + 0.2 * _randn(g, case["head_dim"])).to(dt) for _ in range(2))
    T = case["tokens"]
    if case["op"] == "rope":
        s["q"], s["k"] = _heads(case, g, False)
        s["pos"] = torch.randint(0, case["max_pos"], (T,), generator=g, device="cuda", dtype=torch.int32)
        return s
    B = case["seqs"]
    s["q"], s["k"], s["v"] = _heads(case, g, True)
    # ragged counts that add up to T, each at least one token
    cuts = torch.randperm(T - 1, generator=g, device="cuda")[:B - 1].sort().values + 1 if T > 1 else torch.zeros(0, device="cuda")
    edge = torch.cat([torch.zeros(1, device="cuda"), cuts.float(), torch.full((1,), float(T), device="cuda")]).long()
    count = edge[1:] - edge[:-1]
    start = torch.randint(0, case["context"] + 1, (B,), generator=g, device="cuda")
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), count)
    s["pos"] = (start[seq] + torch.arange(T, device="cuda") - edge[seq]).to(torch.int32)
    s["seq"] = None if B == T else seq.to(torch.int32)
    need = (start + count + PAGE - 1) // PAGE
    blocks, total = int(need.max()), int(need.sum())
    pool, perm = _pages(g, total, (B * (case["context"] + PAGE - 1) + T) // PAGE)
    bt = torch.full((B, blocks), -1, dtype=torch.int32, device="cuda")
    bt[torch.arange(blocks, device="cuda")[None] < need[:, None]] = perm
    s["bt"] = bt
    s["k_pool"], s["v_pool"] = _pool(g, pool, case), _pool(g, pool, case)
    s["sk"] = s["sv"] = None
    if case["pool"] == "e4m3":
        s["sk"], s["sv"] = torch.tensor(0.021, device="cuda"), torch.tensor(0.017, device="cuda")
    return s


def _prepare_prefix(case, g):
    B, H, K, D = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"]
    s = {"case": case}
    s["q"] = _randn(g, B, H, D).to(DTYPES[case["dtype"]])
    lens = torch.randint(0, case["tail"] + 1, (B,), generator=g, device="cuda")
    need = (lens + PAGE - 1) // PAGE
    shared = -(-case["prefix"] // PAGE)
    blocks, total = max(1, int(need.max())), int(need.sum())
    pool, perm = _pages(g, shared + total, shared + B * -(-case["tail"] // PAGE))
    s["table"] = perm[:shared].contiguous()
    bt = torch.full((B, blocks), -1, dtype=torch.int32, device="cuda")
    bt[torch.arange(blocks, device="cuda")[None] < need[:, None]] = perm[shared:]
    s["bt"], s["lens"] = bt, lens.to(torch.int32)
    s["plen"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
    s["sink"] = _randn(g, H) if case["sinks"] else None
    s["sk"] = s["sv"] = None
    if case["pool"] == "e4m3":  # values spread over the format's range, as amax / 448 scales leave them
        s["k_pool"], s["v_pool"] = ((80 * _randn(g, pool, K, PAGE, D)).clamp(-448, 448).to(DTYPES["e4m3"]) for _ in range(2))
        s["sk"], s["sv"] = torch.tensor(1 / 80, device="cuda"), torch.tensor(1 / 80, device="cuda")
    else:
        s["k_pool"], s["v_pool"] = _pool(g, pool, case), _pool(g, pool, case)
    return s


# ------------------------------------------------------------------- the passes
def run(s):
    op = s["case"]["op"]
    if own:
        return {"rope": _own_rope, "append": _own_append, "prefix": _own_prefix}[op](s)
    return {"rope": _plain_rope, "append": _plain_append, "prefix": _plain_prefix}[op](s)


def _own_rope(s):
    import fasterkernels_b200 as fk
    c = s["case"]
    return fk.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["pos"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                           interleaved=c["interleaved"])


def _own_append(s):
    import fasterkernels_b200 as fk
    c = s["case"]
    q = fk.paged_kv_append_rope(s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], s["bt"], s["pos"], s["cos"], s["sin"],
                                seq_ids=s["seq"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                                interleaved=c["interleaved"], scale_k=s["sk"], scale_v=s["sv"])
    return q, s["k_pool"], s["v_pool"]


def _own_prefix(s):
    import fasterkernels_b200 as fk
    return fk.paged_flash_decode_shared_prefix(s["q"], s["k_pool"], s["v_pool"], s["table"], s["plen"], s["bt"], s["lens"],
                                               PAGE, s_aux=s["sink"], scale_k=s["sk"], scale_v=s["sv"])


def _norm_rope(x, weight, cos, sin, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :half], head[..., half:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([head, rest], -1)


def _plain_rope(s):
    pos = s["pos"].long()
    cos, sin, il = s["cos"][pos], s["sin"][pos], s["case"]["interleaved"]
    return (_norm_rope(s["q"], s["qw"], cos, sin, il).to(s["q"].dtype),
            _norm_rope(s["k"], s["kw"], cos, sin, il).to(s["k"].dtype))


def _to_pool(x, scale, dtype):
    return (x / scale).clamp(-448, 448).to(dtype) if scale is not None else x.to(dtype)


def _plain_append(s):
    pos = s["pos"].long()
    cos, sin, il = s["cos"][pos], s["sin"][pos], s["case"]["interleaved"]
    q = _norm_rope(s["q"], s["qw"], cos, sin, il).to(s["q"].dtype)
    k = _norm_rope(s["k"], s["kw"], cos, sin, il)
    seq = torch.arange(pos.numel(), device=pos.device) if s["seq"] is None else s["seq"].long()
    page, slot = s["bt"][seq, pos // PAGE].long(), pos % PAGE
    s["k_pool"][page, :, slot] = _to_pool(k, s["sk"], s["k_pool"].dtype)
    s["v_pool"][page, :, slot] = _to_pool(s["v"].float(), s["sv"], s["v_pool"].dtype)
    return q, s["k_pool"], s["v_pool"]


def _plain_prefix(s):
    q, lens = s["q"].float(), s["lens"].long()
    B, H, D = q.shape
    K = s["k_pool"].shape[1]
    G, P = H // K, s["case"]["prefix"]
    sk, sv = (1.0, 1.0) if s["sk"] is None else (s["sk"], s["sv"])
    q = q.view(B, K, G, D) * D ** -0.5
    # the prefix once for all: [K, P, D]
    kp = s["k_pool"][s["table"].long()].float().transpose(0, 1).reshape(K, -1, D)[:, :P] * sk
    vp = s["v_pool"][s["table"].long()].float().transpose(0, 1).reshape(K, -1, D)[:, :P] * sv
    # each sequence's own tokens: [B, K, T, D]
    bt = s["bt"].long().clamp(min=0)
    kt = s["k_pool"][bt].float().transpose(1, 2).reshape(B, K, -1, D) * sk
    vt = s["v_pool"][bt].float().transpose(1, 2).reshape(B, K, -1, D) * sv
    live = torch.arange(kt.shape[2], device=q.device)[None] < lens[:, None]
    qk = q.transpose(0, 1).reshape(K, B * G, D)
    xp = torch.bmm(qk, kp.transpose(1, 2)).view(K, B, G, P)
    xt = torch.matmul(q, kt.transpose(2, 3)).masked_fill(~live[:, None, None], -math.inf)
    top = torch.maximum(xp.amax(-1).transpose(0, 1), xt.amax(-1))
    if s["sink"] is not None:
        sink = s["sink"].view(1, K, G)
        top = torch.maximum(top, sink)
    wp = torch.exp(xp - top.transpose(0, 1)[..., None])
    wt = torch.exp(xt - top[..., None])
    total = wp.sum(-1).transpose(0, 1) + wt.sum(-1)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.bmm(wp.view(K, B * G, P), vp).view(K, B, G, D).transpose(0, 1)
    out = out + torch.matmul(wt, vt.masked_fill(~live[:, None, :, None], 0.0))
    return (out / total[..., None]).reshape(B, H, D).to(s["q"].dtype)


# ------------------------------------------------------ what a pass cannot do without
def work(case):
    D, H, K = case["head_dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "prefix":
        own_tokens = case["batch"] * case["tail"] / 2
        es = 1 if case["pool"] == "e4m3" else 2
        tokens = case["prefix"] + own_tokens
        io = 2 * 2 * case["batch"] * H * D
        return {"bytes": 2 * tokens * K * D * es + io,
                "flops": 4 * D * H * (case["batch"] * case["prefix"] + own_tokens)}
    T = case["tokens"]
    io = T * (H + K) * D * 2
    table = min(T, case["max_pos"]) * case["rotary"] * 4
    flops = T * (H + K) * (3 * case["rotary"] + (4 * D if case["norm"] else 0))
    if case["op"] == "rope":
        return {"bytes": 2 * io + table + 4 * T, "flops": flops}
    es = 1 if case["pool"] == "e4m3" else 2
    return {"bytes": T * (H + 2 * K) * D * 2 + T * H * D * 2 + T * 2 * K * D * es + table + 8 * T, "flops": flops}


# --------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "prefix": _exact_prefix}[case["op"]](s)


def _turned(x, weight, s):
    # each pair as a complex number, times e^(i angle) of its position
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    pos = s["pos"].long()
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]
    r = 2 * turn.shape[-1]
    pairs = x[..., :r].unflatten(-1, (-1, 2) if s["case"]["interleaved"] else (2, -1))
    pairs = pairs if s["case"]["interleaved"] else pairs.transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z if s["case"]["interleaved"] else z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), x[..., r:]], -1)


def _exact_rope(s):
    return _turned(s["q"], s["qw"], s), _turned(s["k"], s["kw"], s)


def _exact_append(s):
    at = s["pos"].long()
    seq = torch.arange(at.numel(), device=at.device) if s["seq"] is None else s["seq"].long()
    row = s["bt"].long()[seq, at // PAGE] * PAGE + at % PAGE
    got = []
    for pool, x, scale in ((s["k_pool"], _turned(s["k"], s["kw"], s), s["sk"]), (s["v_pool"], s["v"].double(), s["sv"])):
        p, k, _, d = pool.shape
        if scale is not None:
            x = (x / scale.double()).clamp(-448, 448)
        flat = pool.double().transpose(1, 2).reshape(p * PAGE, k, d)
        got.append(flat.index_copy(0, row, x).view(p, PAGE, k, d).transpose(1, 2).contiguous())
    return (_turned(s["q"], s["qw"], s), *got)


def _exact_prefix(s):
    q = s["q"].double()
    B, H, D = q.shape
    K, P = s["k_pool"].shape[1], s["case"]["prefix"]
    G = H // K
    sk, sv = (1.0, 1.0) if s["sk"] is None else (s["sk"].double(), s["sv"].double())
    live = torch.arange(s["bt"].shape[1] * PAGE, device=q.device)[None] < s["lens"][:, None]
    out = torch.empty(B, H, D, dtype=torch.float64, device=q.device)
    for h in range(K):  # one KV head at a time: memory
        qh = q[:, h * G:(h + 1) * G]
        kp = s["k_pool"][s["table"].long(), h].double().reshape(-1, D)[:P] * sk
        vp = s["v_pool"][s["table"].long(), h].double().reshape(-1, D)[:P] * sv
        rows = s["bt"].long().clamp(min=0)
        kt = s["k_pool"][rows, h].double().reshape(B, -1, D) * sk
        vt = s["v_pool"][rows, h].double().reshape(B, -1, D) * sv
        x = torch.cat([qh @ kp.T, (qh @ kt.transpose(1, 2)).masked_fill(~live[:, None], -math.inf)], -1) / math.sqrt(D)
        if s["sink"] is not None:
            x = torch.cat([x, s["sink"].double()[None, h * G:(h + 1) * G, None].expand(B, G, 1)], -1)
        w = torch.softmax(x, -1)
        out[:, h * G:(h + 1) * G] = w[..., :P] @ vp + w[..., P:P + kt.shape[1]] @ (vt * live[..., None])
    return out
