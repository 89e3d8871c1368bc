"""Workloads of the token-generation operators: page bookkeeping, the 8-bit KV cache and the attention
that reads it, and sampling.

``run`` is one pass through one operator, either in its plain form (elementary torch operations) or,
with ``own`` set, through the entry points of ``munet_b200.Context``. ``exact`` restates each operator
in 64 bits. The sizes are those of the decoder configs of ``bench.py`` (16 heads of 128, 8 heads of 64,
vocabularies of 32000 and 8192, contexts of 1024) and generic ones around them.
"""
import math

import torch

own = False

F32, BF16 = 0, 2  # dtype codes of the C ABI
E4M3_MAX = 448.0
MIN_EXP = -64  # smallest exponent of a page's scale
DEV = "cuda"


def _code(dtype):
    return BF16 if dtype == "bf16" else F32


def _torch_dtype(dtype):
    return torch.bfloat16 if dtype == "bf16" else torch.float32


def _cdiv(a, b):
    return -(-a // b)


# ---- the cases ----------------------------------------------------------------------------------


def listed():
    return [
        # one decode step of a full batch: every request gains one token, few need a new page
        dict(name="pages decode 64", op="pages", requests=64, page=64, max_context=1024, max_new=1, pad=0),
        # a scheduler step that admits many prompts beside running requests
        dict(name="pages prompts 512", op="pages", requests=512, page=16, max_context=4096, max_new=511, pad=1000),
        # one token for each of 64 running requests
        dict(name="append decode 64", op="append", requests=64, page=64, heads=16, dim=128, max_context=1024,
             max_new=1, dtype="bf16", slab=True),
        # the prompts of a whole batch (64 sequences of up to 1024 tokens)
        dict(name="append prompts 64x1024", op="append", requests=64, page=64, heads=16, dim=128, max_context=1,
             max_new=1024, dtype="bf16", slab=True),
        # float32 model with an odd head size, prompt chunks that start inside a page
        dict(name="append f32 d80", op="append", requests=9, page=16, heads=5, dim=80, max_context=300,
             max_new=177, dtype="f32", slab=False),
        # one interactive request of the small decoder in float32
        dict(name="attn f32 one request", op="attn", requests=1, page=16, q_heads=8, kv_heads=8, dim=64,
             min_context=777, max_context=777, max_new=1, dtype="f32", causal=True),
        # a full decode batch of the large decoder
        dict(name="attn decode 64x16x128", op="attn", requests=64, page=64, q_heads=16, kv_heads=16, dim=128,
             min_context=129, max_context=2048, max_new=1, dtype="bf16", causal=True),
        # few requests with long contexts and shared key/value heads
        dict(name="attn decode long grouped", op="attn", requests=3, page=32, q_heads=16, kv_heads=2, dim=128,
             min_context=30000, max_context=131072, max_new=1, dtype="bf16", causal=True),
        # prompt chunks beside decoding requests in one call
        dict(name="attn chunks mixed", op="attn", requests=8, page=64, q_heads=16, kv_heads=4, dim=128,
             min_context=1024, max_context=8192, max_new=2048, dtype="bf16", causal=True),
        # the next token of one request
        dict(name="sample 1x32000", op="sample", rows=1, cols=32000, dtype="bf16", top_k=50, top_p=0.95, min_p=0.0),
        # the next tokens of a batch whose requests ask for different things
        dict(name="sample 64x32000", op="sample", rows=64, cols=32000, dtype="bf16", top_k=-1, top_p=0.9,
             min_p=0.02),
        # a large batch with a large vocabulary, float32 logits
        dict(name="sample 256x100003 f32", op="sample", rows=256, cols=100003, dtype="f32", top_k=0, top_p=0.97,
             min_p=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("pages", "append", "attn", "attn", "sample"))
    if op == "pages":
        requests = _log(rng, 1, 1024)
        return dict(op=op, requests=requests, page=rng.choice((16, 32, 48, 64, 128)), max_context=_log(rng, 1, 8192),
                    max_new=_log(rng, 1, max(1, min(2048, 200000 // requests))), pad=rng.choice((0, 0, rng.randint(1, 500))))
    if op == "append":
        requests, heads, dim = _log(rng, 1, 300), rng.randint(1, 16), rng.choice((16, 40, 64, 80, 96, 100, 128, 256))
        most = max(1, min(1024, 100_000_000 // (requests * heads * dim)))
        return dict(op=op, requests=requests, page=rng.choice((16, 32, 48, 64, 128)), heads=heads, dim=dim,
                    max_context=_log(rng, 1, 500), max_new=_log(rng, 1, most), dtype=rng.choice(("bf16", "bf16", "f32")),
                    slab=rng.random() < 0.5)
    if op == "attn":
        kv = rng.choice((1, 2, 3, 4, 8, 16))
        group = rng.choice((1, 1, 2, 3, 4, 7, 8))
        dim = rng.choice((64, 64, 128, 128, 128, 32, 80, 96, 256))
        dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
        requests = _log(rng, 1, 128)
        top = max(64, min(65536, 400_000_000 // (requests * kv * dim)))
        context = _log(rng, 40, top)
        new = 1
        if rng.random() < 0.4:
            new = min(context, max(1, 150_000_000 // (requests * kv * group * context)))
            if dim not in (64, 128) or dtype == "f32":
                new = min(new, max(1, 8_000_000_000 // (requests * kv * group * context * dim)))
            new = _log(rng, 1, min(700, new))
        return dict(op=op, requests=requests, page=rng.choice((16, 32, 48, 64, 128)), q_heads=kv * group, kv_heads=kv,
                    dim=dim, min_context=rng.randint(1, context), max_context=context, max_new=new, dtype=dtype,
                    causal=rng.random() < 0.85)
    rows = _log(rng, 1, 512)
    cols = _log(rng, 50, min(131072, 25_000_000 // rows))
    return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(("bf16", "f32")),
                top_k=rng.choice((0, 0, -1, rng.randint(1, 200), max(1, cols // 3))),
                top_p=rng.choice((1.0, round(rng.uniform(0.05, 0.999), 3))),
                min_p=rng.choice((0.0, round(rng.uniform(0.001, 0.2), 3))))


# ---- inputs -------------------------------------------------------------------------------------


def _lengths(case, seed):
    """Tokens in the cache before the call and new ones, per request (host lists). The seed decides which
    request has which lengths; the lengths themselves go with the case, so that sizes do not vary."""
    g = torch.Generator().manual_seed(11)
    n = case["requests"]
    lo, hi, new = case.get("min_context", 0), case["max_context"], case["max_new"]
    total = torch.randint(lo, hi + 1, (n,), generator=g) if hi > lo else torch.full((n,), hi)
    add = torch.randint(1, new + 1, (n,), generator=g) if new > 1 else torch.ones(n, dtype=torch.int64)
    if new > 1 and n > 2:  # decoding requests between the prompts, one of each kind at least
        add[torch.rand(n, generator=g) < 0.3] = 1
        add[0], add[1] = 1, new
    if case["op"] == "attn":  # context counts the new tokens
        total = total.clamp(min=1)
        if hi > lo:
            total[-1] = hi
        add = torch.minimum(add, total)
        total = total - add
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed))
    return total[order].tolist(), add[order].tolist()


def _tables(case, ctx, new, g, extra):
    """A block table whose pages are scattered over the pool, and the pool's size."""
    page = case["page"]
    pages = [_cdiv(c + m, page) for c, m in zip(ctx, new)]
    width = max(pages) + 1
    num_pages = sum(pages) + extra
    perm = torch.randperm(num_pages, generator=g, device=DEV).to(torch.int32)
    have = torch.tensor(pages, device=DEV)
    first = torch.cumsum(have, 0) - have
    col = torch.arange(width, device=DEV)
    table = perm[(first[:, None] + col).clamp(max=num_pages - 1)]
    return torch.where(col < have[:, None], table, torch.full_like(table, -1)), perm, num_pages


def _cache(shape, g):
    """An e4m3 cache as quantised normal values fill it, with a power-of-two scale per page and head."""
    flat = torch.empty(math.prod(shape), dtype=torch.uint8, device=DEV)
    some = torch.randn(min(flat.numel(), 1 << 24), generator=g, device=DEV) * 90
    some = some.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    for at in range(0, flat.numel(), some.numel()):
        part = flat[at:at + some.numel()]
        part.copy_(some[:part.numel()])
    scale = torch.exp2(torch.randint(-8, -5, shape[:2], generator=g, device=DEV).float())
    return flat.view(shape), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case), "op": op}
    if op == "sample":
        rows, cols = case["rows"], case["cols"]
        # logits of a language model: a broad bell and a few tokens that stand out
        x = torch.randn(rows, cols, generator=g, device=DEV) * 2.0
        peaks = torch.randint(0, cols, (rows, 12), generator=g, device=DEV)
        x.scatter_add_(1, peaks, torch.rand(rows, 12, generator=g, device=DEV) * 9.0)
        s["logits"] = x.to(_torch_dtype(case["dtype"]))
        s["u"] = torch.rand(rows, generator=g, device=DEV)
        s["temperature"] = 0.3 + torch.rand(rows, generator=g, device=DEV)
        if rows > 8:
            s["temperature"][rows // 2] = 0.0  # a greedy request in the batch
        k = case["top_k"]
        if k:
            s["top_k"] = (torch.full((rows,), k, device=DEV) if k > 0 else
                          torch.randint(0, min(cols, 100) + 1, (rows,), generator=g, device=DEV)).to(torch.int32)
        else:
            s["top_k"] = None
        s["top_p"] = torch.full((rows,), case["top_p"], device=DEV) if case["top_p"] < 1 else None
        s["min_p"] = torch.full((rows,), case["min_p"], device=DEV) if case["min_p"] > 0 else None
        s["idx"] = torch.empty(rows, dtype=torch.int32, device=DEV)
        s["prob"] = torch.empty(rows, device=DEV)
        return s
    ctx, new = _lengths(case, seed)
    page, B = case["page"], case["requests"]
    s["n_new"] = sum(new)
    s["new"] = torch.tensor(new, dtype=torch.int32, device=DEV)
    s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    table, perm, num_pages = _tables(case, ctx, new, g, 7)
    s["num_pages"] = num_pages
    if op == "pages":
        have = (s["ctx"] + (page - 1)) // page
        col = torch.arange(table.shape[1], device=DEV)
        s["table"] = torch.where(col < have[:, None], table, torch.full_like(table, -1)).contiguous()
        s["free"] = perm.flip(0).contiguous()
        s["n_slots"] = s["n_new"] + case["pad"]
        s["query_start"] = torch.empty(B + 1, dtype=torch.int32, device=DEV)
        s["seq"] = torch.empty(B, dtype=torch.int32, device=DEV)
        s["slots"] = torch.empty(s["n_slots"], dtype=torch.int32, device=DEV)
        s["positions"] = torch.empty(s["n_slots"], dtype=torch.int32, device=DEV)
        s["taken"] = torch.empty(1, dtype=torch.int32, device=DEV)
        return s
    s["table"] = table.contiguous()
    start = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    start[1:] = torch.cumsum(s["new"], 0)
    s["query_start"], s["seq"] = start, s["ctx"] + s["new"]
    if op == "append":
        H, D, N = case["heads"], case["dim"], s["n_new"]
        dt = _torch_dtype(case["dtype"])
        amp = torch.exp(torch.randn(H, 1, generator=g, device=DEV) * 0.7)  # heads differ in magnitude
        if case["slab"]:  # columns of the fused projection's output
            x = torch.randn(N, 3, H, D, generator=g, device=DEV)
            x[:, 1:] *= amp
            x = x.to(dt)
            s["k"], s["v"], s["ld"] = x[:, 1], x[:, 2], 3 * H * D
        else:
            s["k"] = (torch.randn(N, H, D, generator=g, device=DEV) * amp).to(dt)
            s["v"] = (torch.randn(N, H, D, generator=g, device=DEV) * amp).to(dt)
            s["ld"] = H * D
        t = torch.arange(N, device=DEV, dtype=torch.int32)
        r = torch.searchsorted(start[1:], t, right=True)
        pos = s["ctx"][r] + t - start[r]
        s["slots"] = (table[r, (pos // page).long()] * page + pos % page).to(torch.int32)
        s["runs"] = sum(_cdiv(c + m, page) - c // page for c, m in zip(ctx, new))
        s["k_cache"], s["k_scale"] = _cache((num_pages, H, page, D), g)
        s["v_cache"], s["v_scale"] = _cache((num_pages, H, page, D), g)
        return s
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["dim"]
    N = s["n_new"]
    s["k_cache"], s["k_scale"] = _cache((num_pages, Hkv, page, D), g)
    s["v_cache"], s["v_scale"] = _cache((num_pages, Hkv, page, D), g)
    s["q"] = (torch.randn(N, Hq, D, generator=g, device=DEV) * 1.5).to(_torch_dtype(case["dtype"]))
    s["out"] = torch.zeros_like(s["q"])
    s["max_new"], s["max_seq"] = max(new), max(c + m for c, m in zip(ctx, new))
    return s


# ---- the plain forms ----------------------------------------------------------------------------


def _plain_pages(s):
    page, B = s["case"]["page"], s["case"]["requests"]
    ctx, new, table, free = s["ctx"].long(), s["new"].long(), s["table"], s["free"]
    ends = torch.cumsum(new, 0)
    start = ends - new
    old = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page - old
    upto = torch.cumsum(need, 0)
    col = torch.arange(table.shape[1], device=DEV)
    at = (upto - need)[:, None] + col - old[:, None]
    fresh = (col >= old[:, None]) & (col < (old + need)[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    s["query_start"][0] = 0
    s["query_start"][1:] = ends
    s["seq"].copy_(ctx + new)
    t = torch.arange(s["n_slots"], device=DEV)
    r = torch.searchsorted(ends, t, right=True).clamp(max=B - 1)
    pos = ctx[r] + t - start[r]
    live = t < ends[-1]
    slot = table[r, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    s["slots"].copy_(torch.where(live, slot, -1))
    s["positions"].copy_(torch.where(live, pos, 0))
    s["taken"].copy_(upto[-1:])


def _scale_of(amax):
    """Smallest power of two s >= 2^MIN_EXP with amax <= 448 s."""
    m, e = torch.frexp(amax)
    x = torch.where(m <= 0.875, e - 9, e - 8)
    x = torch.where(amax > 0, x, MIN_EXP).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), x)


def _e4m3(v):
    return v.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append_one(s, x, cache, scale):
    page = s["case"]["page"]
    slots = s["slots"].long()
    p, off = slots // page, slots % page
    lead = torch.ones_like(p, dtype=torch.bool)
    lead[1:] = p[1:] != p[:-1]
    at = torch.argsort((~lead).to(torch.uint8), stable=True)[:s["runs"]]  # first token of each page's run
    run = torch.cumsum(lead, 0) - 1
    pages, first = p[at], off[at]
    x = x.float()
    H = x.shape[1]
    amax = torch.zeros(s["runs"], H, device=DEV).scatter_reduce_(0, run[:, None].expand(-1, H), x.abs().amax(-1), "amax")
    old = torch.where((first > 0)[:, None], scale[pages], torch.zeros_like(amax))
    now = torch.maximum(old, _scale_of(amax))
    kept = cache[pages]  # what the touched pages hold
    again = _e4m3(kept.view(torch.float8_e4m3fn).float() * (old / now)[:, :, None, None])
    earlier = torch.arange(page, device=DEV) < first[:, None]
    cache[pages] = torch.where(earlier[:, None, :, None], again, kept)
    scale[pages] = now
    cache[p, :, off] = _e4m3(x / now[run][:, :, None])


def _plain_attn(s):
    c = s["case"]
    page, Hq, Hkv, D, B = c["page"], c["q_heads"], c["kv_heads"], c["dim"], c["requests"]
    G, M, S = Hq // Hkv, s["max_new"], s["max_seq"]
    use = s["table"][:, :_cdiv(S, page)].long().clamp(min=0)
    start, n, seq = s["query_start"][:-1].long(), s["new"].long(), s["seq"].long()

    def whole(cache, scale):  # [B, Hkv, tokens, D]
        x = cache[use].view(torch.float8_e4m3fn).float() * scale[use][..., None, None]
        return x.transpose(1, 2).reshape(B, Hkv, -1, D)

    i = torch.arange(M, device=DEV)
    rows = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(B, M, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * M, D)
    w = torch.matmul(q, whole(s["k_cache"], s["k_scale"]).transpose(2, 3)).mul_(1.0 / math.sqrt(D))
    last = (seq - n)[:, None] + i if c["causal"] else (seq - 1)[:, None].expand(B, M)
    last = torch.minimum(last, (seq - 1)[:, None])
    j = torch.arange(w.shape[-1], device=DEV)
    w = w.view(B, Hkv, G, M, -1).masked_fill_((j > last[..., None])[:, None, None], -math.inf)
    w = torch.exp(w.sub_(w.amax(-1, keepdim=True)))
    w = w.div_(w.sum(-1, keepdim=True)).view(B, Hkv, G * M, -1)
    o = torch.matmul(w, whole(s["v_cache"], s["v_scale"])).view(B, Hkv, G, M, D).permute(0, 3, 1, 2, 4)
    t = torch.arange(s["n_new"], device=DEV)
    r = torch.searchsorted(s["query_start"][1:], t.int(), right=True)
    s["out"].copy_(o[r, t - start[r]].reshape(-1, Hq, D))


def _plain_sample(s):
    x = s["logits"].double()
    rows, cols = x.shape
    T = s["temperature"].double()[:, None]
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(cols, device=DEV)
    greedy = T <= 0
    w = torch.exp((xs - xs[:, :1]) / torch.where(greedy, 1.0, T))
    keep = torch.where(greedy, rank < 1, True)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep &= (rank < k) | (k <= 0)
    w = torch.where(keep, w, 0.0)
    if s["top_p"] is not None:
        before = torch.cumsum(w, 1) - w
        keep &= (before < s["top_p"].double()[:, None] * w.sum(1, keepdim=True)) | (rank < 1)
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    cdf = torch.cumsum(w, 1)
    total = cdf[:, -1:]
    idx = (cdf <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=cols - 1)
    s["idx"].copy_(idx[:, 0])
    s["prob"].copy_((torch.gather(w, 1, idx) / total)[:, 0])


# ---- one pass -----------------------------------------------------------------------------------

_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import munet_b200
        _ctx = munet_b200.Context(0)
    return _ctx


def _f8(cache):
    return cache.view(torch.float8_e4m3fn)


def run(s):
    c, op = s["case"], s["op"]
    if op == "pages":
        if own:
            _context().page_map(s["ctx"], s["new"], s["free"], s["free"].numel(), s["table"], s["table"].shape[1],
                                c["requests"], c["page"], s["num_pages"], s["query_start"], s["seq"], s["slots"],
                                s["positions"], s["n_slots"], s["taken"])
        else:
            _plain_pages(s)
        return {k: s[k] for k in ("table", "query_start", "seq", "slots", "positions", "taken")}
    if op == "append":
        if own:
            _context().kv_cache_append(s["k"], s["v"], s["ld"], s["slots"], s["n_new"], s["k_cache"], s["v_cache"],
                                       s["k_scale"], s["v_scale"], s["num_pages"], c["page"], c["heads"], c["dim"],
                                       _code(c["dtype"]))
        else:
            _plain_append_one(s, s["k"], s["k_cache"], s["k_scale"])
            _plain_append_one(s, s["v"], s["v_cache"], s["v_scale"])
        return {"k": _f8(s["k_cache"]), "v": _f8(s["v_cache"]), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "attn":
        if own:
            Hq, Hkv, D, dt = c["q_heads"], c["kv_heads"], c["dim"], _code(c["dtype"])
            if "ws" not in s:  # kept by the program, like the cache
                s["ws_bytes"] = _context().attention_paged_workspace_bytes(s["n_new"], c["requests"], Hq, Hkv, D, dt)
                s["ws"] = torch.empty(max(s["ws_bytes"], 16), dtype=torch.uint8, device=DEV)
            _context().attention_paged(s["q"], Hq * D, s["out"], Hq * D, s["k_cache"], s["v_cache"], s["k_scale"],
                                       s["v_scale"], s["table"], s["table"].shape[1], s["query_start"], s["seq"],
                                       c["requests"], s["n_new"], Hq, Hkv, D, s["num_pages"], c["page"], c["causal"],
                                       dt, s["ws"], s["ws_bytes"])
        else:
            _plain_attn(s)
        return s["out"]
    if own:
        _context().sample(s["logits"], c["cols"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                          s["idx"], s["prob"], c["rows"], c["cols"], _code(c["dtype"]))
    else:
        _plain_sample(s)
    return {"token": s["idx"], "prob": s["prob"]}


# ---- work and exact results ---------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 28 * case["rows"], "flops": 4.0 * n}
    ctx, new = _lengths(case, 1)
    page, N, B = case["page"], sum(new), case["requests"]
    total = [c + m for c, m in zip(ctx, new)]
    if op == "pages":
        fresh = sum(_cdiv(t, page) - _cdiv(c, page) for t, c in zip(total, ctx))
        # the table is read where tokens join a page that is there already
        return {"bytes": 8 * B + 8 * fresh + 4 * B + 8 * B + 8 * (N + case["pad"]), "flops": 0.0}
    es = 2 if case["dtype"] == "bf16" else 4
    if op == "append":
        runs = sum(_cdiv(t, page) - c // page for t, c in zip(total, ctx))
        n = 2 * N * case["heads"] * case["dim"]
        return {"bytes": n * (es + 1) + 4 * N + 8 * runs * case["heads"], "flops": 3.0 * n}
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["dim"]
    pages = sum(_cdiv(t, page) for t in total)
    seen = sum(m * c + m * (m + 1) // 2 if case["causal"] else m * t for c, m, t in zip(ctx, new, total))
    return {"bytes": 2 * sum(total) * Hkv * D + 8 * pages * Hkv + 4 * pages + 2 * N * Hq * D * es,
            "flops": 4.0 * D * Hq * seen}


def _round_e4m3_64(v):
    """Nearest e4m3 value (ties to even) of 64-bit numbers, saturating."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(s, x, cache, scale):
    page = s["case"]["page"]
    values, scale = _f8(cache).double(), scale.double().clone()
    x = x.double()
    runs, at = [], 0
    slots = s["slots"].tolist()
    for t in range(1, len(slots) + 1):
        if t == len(slots) or slots[t] // page != slots[at] // page:
            runs.append((at, t))
            at = t
    for a, b in runs:
        p, off = slots[a] // page, slots[a] % page
        amax = x[a:b].abs().amax((0, 2))
        need = torch.exp2(torch.ceil(torch.log2(amax / E4M3_MAX)))
        need = torch.where(amax <= E4M3_MAX * need / 2, need / 2, torch.where(amax > E4M3_MAX * need, need * 2, need))
        need = need.clamp(min=2.0 ** MIN_EXP)
        if off:
            now = torch.maximum(scale[p], need)
            values[p, :, :off] = _round_e4m3_64(values[p, :, :off] * (scale[p] / now)[:, None, None])
        else:
            now = need
        scale[p] = now
        values[p, :, off:off + b - a] = _round_e4m3_64(x[a:b].transpose(0, 1) / now[:, None, None])
    return values, scale


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        k, ks = _exact_append(s, s["k"], s["k_cache"], s["k_scale"])
        v, vs = _exact_append(s, s["v"], s["v_cache"], s["v_scale"])
        return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}
    if case["op"] == "attn":
        Hq, Hkv, D, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        start, seq = s["query_start"].tolist(), s["seq"].tolist()
        for b in range(case["requests"]):
            n, L = start[b + 1] - start[b], seq[b]
            ids = s["table"][b, :_cdiv(L, page)].long()
            for h in range(Hkv):
                k = (_f8(s["k_cache"][ids, h]).double() * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, D)[:L]
                v = (_f8(s["v_cache"][ids, h]).double() * s["v_scale"][ids, h].double()[:, None, None]).reshape(-1, D)[:L]
                heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                a = torch.einsum("igd,jd->gij", s["q"][start[b]:start[b + 1], heads].double(), k) / math.sqrt(D)
                if case["causal"]:
                    seen = torch.ones(n, L, device=DEV, dtype=torch.bool).tril(L - n)
                    a = a.masked_fill(~seen, -math.inf)
                out[start[b]:start[b + 1], heads] = torch.einsum("gij,jd->igd", torch.softmax(a, -1), v)
        return out
    x = s["logits"].double()
    prob = torch.zeros(case["rows"], dtype=torch.float64, device=DEV)
    token = torch.zeros(case["rows"], dtype=torch.int64, device=DEV)
    for r in range(case["rows"]):
        T = float(s["temperature"][r])
        if T <= 0:
            token[r], prob[r] = torch.nonzero(x[r] == x[r].max())[0, 0], 1.0
            continue
        p = torch.softmax(x[r] / T, 0)
        best = torch.argsort(p, descending=True, stable=True)
        if s["top_k"] is not None and int(s["top_k"][r]) > 0:
            best = best[:int(s["top_k"][r])]
        mass = torch.cumsum(p[best], 0)
        if s["top_p"] is not None:
            cut = int((mass < float(s["top_p"][r]) * mass[-1]).sum()) + 1
            best = best[:cut]
        if s["min_p"] is not None:
            best = best[p[best] >= float(s["min_p"][r]) * p.max()]
        left = torch.sort(best).values
        mass = torch.cumsum(p[left], 0)
        i = min(int((mass <= float(s["u"][r]) * mass[-1]).sum()), left.numel() - 1)
        token[r], prob[r] = left[i], p[left[i]] / mass[-1]
    return {"token": token.to(torch.int32), "prob": prob}
