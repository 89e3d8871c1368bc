"""Page maps, the 8-bit KV cache and the attention that reads it, against 64-bit restatements."""
import numpy as np
import pytest

import oracle
from oracle import BF16, F32
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import munet_b200 as mb
    c = mb.Context(0)
    yield c
    c.close()


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def ints(a):
    return dev(np.asarray(a, np.int32))


def float_dev(x, dtype):
    """float64 values -> device tensor of the dtype, and the float64 values it holds."""
    import torch
    t = dev(x.astype(np.float32), torch.bfloat16 if dtype == BF16 else torch.float32)
    return t, t.double().cpu().numpy()


# ---- page map -------------------------------------------------------------------------------------


def run_page_map(ctx, c, n, free, table, page, num_pages, n_slots, n_free=None, stream=None):
    import torch
    B = len(c)
    t = ints(table)
    o = {k: torch.full((m,), -7, dtype=torch.int32, device="cuda")
         for k, m in (("qs", B + 1), ("seq", B), ("slots", n_slots), ("pos", n_slots), ("taken", 1))}
    f = ints(free)
    ctx.page_map(ints(c), ints(n), f, len(free) if n_free is None else n_free, t, table.shape[1], B, page, num_pages,
                 o["qs"], o["seq"], o["slots"], o["pos"], n_slots, o["taken"], stream=stream)
    return t.cpu().numpy(), {k: v.cpu().numpy() for k, v in o.items()}


@pytest.mark.parametrize("B,page,max_ctx,max_new,pad", [
    (1, 16, 1, 1, 0), (1, 64, 5000, 2000, 3), (3, 16, 40, 1, 0), (64, 64, 1024, 1, 0), (65, 48, 300, 70, 11),
    (1000, 16, 100, 40, 500), (5000, 16, 30, 3, 0), (16384, 32, 40, 1, 1),
])
def test_page_map(ctx, B, page, max_ctx, max_new, pad):
    rng = np.random.default_rng(B + page)
    c = rng.integers(0, max_ctx + 1, B)
    n = rng.integers(0, max_new + 1, B)  # requests that gain nothing among them
    have = -(-c // page)
    need = -(-(c + n) // page)
    num_pages = int(need.sum()) + 5
    perm = rng.permutation(num_pages).astype(np.int32)
    table = np.full((B, int(need.max(initial=0)) + 2), -1, np.int32)
    at = 0
    for r in range(B):
        table[r, :have[r]] = perm[at:at + have[r]]
        at += have[r]
    free = perm[at:]
    n_slots = int(n.sum()) + pad
    want = ref.page_map(c.tolist(), n.tolist(), free.tolist(), table, page, n_slots)
    t, o = run_page_map(ctx, c, n, free, table, page, num_pages, n_slots)
    ctx.check()
    assert np.array_equal(t, want[0])
    for key, w in zip(("qs", "seq", "slots", "pos"), want[1:5]):
        assert np.array_equal(o[key], np.asarray(w, np.int32)), key
    assert o["taken"][0] == want[5]


def test_page_map_without_requests(ctx):
    t, o = run_page_map(ctx, [], [], [1, 2], np.zeros((0, 4), np.int32), 16, 8, 5)
    ctx.check()
    assert o["qs"][0] == 0 and o["taken"][0] == 0 and (o["slots"] == -1).all() and (o["pos"] == 0).all()


@pytest.mark.parametrize("what,code", [("free", 6), ("table", 6), ("slots", 6), ("page", 5), ("length", 5)])
def test_page_map_reports_what_does_not_fit(ctx, what, code):
    import munet_b200 as mb
    c, n, page = [16, 5, 0], [20, 1, 40], 16
    table = np.array([[7, -1, -1], [3, -1, -1], [-1, -1, -1]], np.int32)
    free, pages, n_slots = [9, 8, 1, 2, 0], 10, 61
    if what == "free":
        free = free[:3]
    if what == "table":
        table = table[:, :2]
    if what == "slots":
        n_slots = 30
    if what == "page":
        free[1] = 10
    if what == "length":
        n[1] = -1
    t, o = run_page_map(ctx, c, n, free, table, page, pages, n_slots)
    with pytest.raises(mb.MuNetError) as e:
        ctx.check()
    assert e.value.code == code
    ctx.check()  # cleared
    slots = o["slots"]
    assert ((slots >= -1) & (slots < pages * page)).all()
    good = slots[:16]
    if what == "page":
        assert t[0, 2] == -1 and (slots[16:20] == -1).all() and (good >= 0).all()
    if what == "free":
        assert t[2].tolist() == [1, -1, -1] and (slots[21 + 16:] == -1).all() and o["taken"][0] == 3
    if what == "table":
        assert (slots[16:20] == -1).all() and (good == 9 * 16 + np.arange(16)).all()
    if what == "slots":
        assert (slots >= 0).all() and o["qs"][-1] == 61
    if what == "length":
        assert o["qs"].tolist() == [0, 20, 20, 60] and o["seq"].tolist() == [36, 0, 40]


def test_page_map_sums_beyond_32_bits(ctx):
    """Lengths whose sums pass 2^31: what fits the slots is right, the rest is reported."""
    import munet_b200 as mb
    big = 2 ** 30
    table = np.full((4, 2), -1, np.int32)
    table[0, 0] = 5
    t, o = run_page_map(ctx, [16, 0, 0, 2 ** 31 - 1], [8, big, big, 5], [7, 6, 4, 3, 2], table, 16, 8, 40)
    with pytest.raises(mb.MuNetError) as e:
        ctx.check()
    assert e.value.code in (5, 6)
    assert t.tolist() == [[5, 7], [6, 4], [3, 2], [-1, -1]]
    assert o["slots"].tolist() == [7 * 16 + i for i in range(8)] + [6 * 16 + i for i in range(16)] + [4 * 16 + i for i in range(16)]
    assert o["pos"].tolist() == [16 + i for i in range(8)] + list(range(32))
    assert o["qs"].tolist() == [0, 8, 8 + big, 2 ** 31 - 1, 2 ** 31 - 1] and o["taken"][0] == 5
    assert o["seq"].tolist() == [24, big, big, 0]  # the last request's sum does not fit: it counts as empty


# ---- append ---------------------------------------------------------------------------------------


def new_cache(rng, pages, H, page, D):
    code = rng.integers(0, 256, (pages, H, page, D)).astype(np.uint8)
    code[(code & 127) == 127] = 0
    return code, np.exp2(rng.integers(-9, -5, (pages, H))).astype(np.float32)


def run_append(ctx, k, v, ld, slots, n, kc, vc, ks, vs, dtype, stream=None):
    d = [dev(a) for a in (kc, vc, ks, vs)]
    ctx.kv_cache_append(k, v, ld, ints(slots), n, *d, kc.shape[0], kc.shape[2], kc.shape[1], kc.shape[3], dtype,
                        stream=stream)
    return [t.cpu().numpy() for t in d]


def check_append(ctx, kx, vx, k, v, ld, slots, caches, dtype):
    kc, vc, ks, vs = caches
    page = kc.shape[2]
    got = run_append(ctx, k, v, ld, slots, len(slots), kc, vc, ks, vs, dtype)
    for x, cache, scale, gc, gs in ((kx, kc, ks, got[0], got[2]), (vx, vc, vs, got[1], got[3])):
        wc, ws = ref.append(x, list(slots), cache, scale, page)
        assert np.array_equal(gs.astype(np.float64), ws)
        nan = np.isnan(ref.TABLE[wc])
        assert np.array_equal(np.where(nan, 127, wc), np.where(nan, gc & 127, gc))
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,D,page,starts,counts,slab", [
    (1, 128, 16, [0], [1], False), (2, 64, 16, [15], [1], True), (3, 128, 64, [0, 5, 63, 64], [1, 1, 1, 1], True),
    (2, 128, 64, [0, 10, 60], [200, 54, 5], True), (5, 80, 16, [3], [50], False), (2, 100, 32, [31, 0], [2, 64], False),
    (1, 1, 16, [4], [20], False), (2, 256, 48, [40], [120], True), (1, 8, 1024, [1000], [1100], False),
    (4, 7, 16, [0, 1, 2], [33, 1, 15], False), (16, 128, 16, [0] * 40, [1] * 40, False),
])
def test_append(ctx, dtype, H, D, page, starts, counts, slab):
    rng = np.random.default_rng(D + page + len(starts))
    slots, pages = [], 0
    order = rng.permutation(sum(-(-(s + c) // page) for s, c in zip(starts, counts)) + 3)
    for s, c in zip(starts, counts):
        slots += [int(order[pages + p // page]) * page + p % page for p in range(s, s + c)]
        pages += -(-(s + c) // page)
    n = len(slots)
    caches = new_cache(rng, len(order), H, page, D) + new_cache(rng, len(order), H, page, D)
    caches = (caches[0], caches[2], caches[1], caches[3])
    amp = np.exp(rng.standard_normal((H, 1)) * 2)
    if slab:
        t, x = float_dev(rng.standard_normal((n, 3, H, D)) * amp, dtype)
        check_append(ctx, x[:, 1], x[:, 2], t[:, 1], t[:, 2], 3 * H * D, slots, caches, dtype)
    else:
        k, kx = float_dev(rng.standard_normal((n, H, D)) * amp, dtype)
        v, vx = float_dev(rng.standard_normal((n, H, D)), dtype)
        check_append(ctx, kx, vx, k, v, H * D, slots, caches, dtype)
    ctx.check()


def test_append_many_tokens_per_cta(ctx):
    """Enough tokens that a CTA looks at several of them: runs that begin in one CTA's range and end in the next."""
    rng = np.random.default_rng(3)
    H, D, page, n = 16, 16, 16, 3000
    order = rng.permutation(400)
    slots, at, p = [], 0, 0
    while at < n:  # requests of 1 to 90 tokens, some starting inside a page, some padding between them
        c, s = int(rng.integers(1, 90)), int(rng.integers(0, page))
        slots += [int(order[(p + (s + i) // page)]) * page + (s + i) % page for i in range(c)]
        slots += [-1] * int(rng.integers(0, 3))
        p += (s + c - 1) // page + 1
        at = len(slots)
    k, kx = float_dev(rng.standard_normal((at, H, D)), BF16)
    v, vx = float_dev(rng.standard_normal((at, H, D)) * 5, BF16)
    a, b = new_cache(rng, 400, H, page, D), new_cache(rng, 400, H, page, D)
    check_append(ctx, kx, vx, k, v, H * D, slots, (a[0], b[0], a[1], b[1]), BF16)
    ctx.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_extremes(ctx, dtype):
    """Scales grow over a sequence of single tokens; zeros, tiny, huge, infinite and NaN rows; scales that are
    no power of two; a padded token."""
    rng = np.random.default_rng(1)
    H, D, page = 2, 32, 16
    a, b = new_cache(rng, 3, H, page, D), new_cache(rng, 3, H, page, D)
    caches = [a[0], b[0], a[1], b[1]]
    caches[2][1] = 0.3  # a page that someone else quantised
    for i, f in enumerate([0.0, 1e-30, 1e-3, 1.0, 7.0, 448.0, 449.0, 1e30, 1.0]):
        for slot in (i, page + 3 + i, -1):
            x = rng.standard_normal((1, H, D)) * f
            if i == 4:
                x[0, 0, 3], x[0, 0, 4], x[0, 1, 5] = np.inf, -np.inf, np.nan
            k, kx = float_dev(x, dtype)
            v, vx = float_dev(-x, dtype)
            caches = check_append(ctx, kx, vx, k, v, H * D, [slot], caches, dtype)
    ctx.check()


def test_append_repeated_slots_and_bad_slots(ctx):
    import munet_b200 as mb
    rng = np.random.default_rng(2)
    H, D, page = 2, 64, 16
    a, b = new_cache(rng, 4, H, page, D), new_cache(rng, 4, H, page, D)
    caches = (a[0], b[0], a[1], b[1])
    for slots in ([5, 5, 5], [9, 8, 7, 9], [20, 20, 21, 3], [17, 18, 17, 18] * 20):
        k, kx = float_dev(rng.standard_normal((len(slots), H, D)) * 3, BF16)
        check_append(ctx, kx, kx, k, k, H * D, slots, caches, BF16)
    ctx.check()
    slots = [4, 64, 21, 2 ** 31 - 1, -5, 38]  # a page in one place only, as the call asks for
    k, kx = float_dev(rng.standard_normal((6, H, D)), BF16)
    got = run_append(ctx, k, k, H * D, slots, 6, *caches, BF16)
    with pytest.raises(mb.MuNetError) as e:
        ctx.check()
    assert e.value.code == 5
    want = ref.append(kx, [4, -1, 21, -1, -1, 38], caches[0], caches[2], page)[0]
    assert np.array_equal(got[0], want)


# ---- attention ------------------------------------------------------------------------------------


def make_problem(rng, dtype, B, Hq, Hkv, D, page, lens, news, extra=3, pad_rows=2):
    pages = [-(-L // page) for L in lens]
    num = sum(pages) + extra
    perm = rng.permutation(num).astype(np.int32)
    table = np.full((B, max(pages) + 1), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, :pages[b]] = perm[at:at + pages[b]]
        at += pages[b]
    kc, ks = new_cache(rng, num, Hkv, page, D)
    vc, vs = new_cache(rng, num, Hkv, page, D)
    ks *= 4  # scores with some spread
    qs = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    n = int(qs[-1]) + pad_rows
    q, qx = float_dev(rng.standard_normal((n, Hq, D)), dtype)
    return dict(q=q, qx=qx, kc=kc, vc=vc, ks=ks, vs=vs, table=table, qs=qs, seq=np.asarray(lens, np.int32), n=n)


def run_attention(ctx, pr, dtype, causal, Hkv, page, stream=None, ws=None, out=None):
    import torch
    n, Hq, D = pr["q"].shape
    B = len(pr["seq"])
    nbytes = ctx.attention_paged_workspace_bytes(n, B, Hq, Hkv, D, dtype)
    if ws is None:
        ws = torch.full((nbytes,), 0xEE, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((n, Hq, D), 7.0, dtype=pr["q"].dtype, device="cuda")
    d = pr.get("dev") or [dev(pr[k]) for k in ("kc", "vc", "ks", "vs", "table", "qs", "seq")]
    pr["dev"] = d
    ctx.attention_paged(pr["q"], pr["q"].stride(0), out, out.stride(0), *d[:5], pr["table"].shape[1], d[5], d[6], B, n,
                        Hq, Hkv, D, pr["kc"].shape[0], page, causal, dtype, ws, nbytes, stream=stream)
    return out


def check_attention(pr, out, dtype, causal, page):
    """The tolerance is the sum of the roundings: scores are fp32 sums of D products (each step at most half a
    unit, the tensor cores up to a whole one: 2^-23 of sum |q k|, for the row and its largest entry), which
    changes a probability by that much of itself; probabilities carry fp16's 2^-11 in the bfloat16 kernel; the
    sums over keys are pieces of at most 2^-23 a step; the output is rounded once to its type. fp16's
    smallest step is 2^-24: the tensor-core kernel (head sizes that are multiples of 16) holds p_j vs_j with the
    row's largest at 2^15, for float32 as a sum of two, so each is off by up to half of 2^-24 * 2^-15 of the
    largest, and multiplies a code of at most 448. The prompt-chunk kernel (bfloat16, head size 64 or 128, more
    rows than requests) holds the largest between 2^7 and 2^15."""
    n_live = int(pr["qs"][-1])
    D = out.shape[2]
    want, weight, spread, top = ref.attention(pr["qx"], pr["kc"], pr["vc"], pr["ks"].astype(np.float64),
                                         pr["vs"].astype(np.float64), pr["table"], pr["qs"], pr["seq"], page, causal)
    got = out.double().cpu().numpy()
    assert (got[n_live:] == 7.0).all(), "rows behind the last request changed"
    L = int(pr["seq"].max(initial=1))
    prob = 2 * (D + 4) * 2.0 ** -23 * spread + 2.0 ** -20 + (2.0 ** -11 if dtype == BF16 else 2.0 ** -22) + L * 2.0 ** -23
    half = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    chunks = dtype == BF16 and D in (64, 128) and out.shape[0] > len(pr["seq"])
    low = L * 448 * (2.0 ** -32 if chunks else 2.0 ** -40) * top if D % 16 == 0 else 0 * top
    bound = half * np.abs(want) + 2 * prob[..., None] * weight + low[..., None] + 1e-30
    err = np.abs(got - want)[:n_live]
    assert np.isfinite(got).all()
    worst = float((err / bound[:n_live]).max()) if err.size else 0.0
    assert worst <= 1.0, f"worst error / bound {worst:.3g}"


CASES = [
    # B, Hq, Hkv, D, page, lens, news
    (1, 1, 1, 64, 16, [1], [1]),
    (1, 8, 8, 64, 16, [777], [1]),
    (3, 4, 4, 128, 64, [64, 65, 1], [1, 1, 1]),
    (4, 16, 2, 128, 32, [500, 33, 1, 200], [1, 1, 1, 1]),
    (2, 6, 2, 128, 16, [130, 300], [4, 1]),
    (3, 7, 1, 64, 48, [100, 60, 257], [3, 0, 20]),
    (2, 4, 4, 128, 128, [128, 400], [128, 200]),
    (5, 8, 4, 64, 16, [40, 1, 17, 0, 300], [40, 1, 5, 0, 130]),
    (2, 2, 2, 80, 16, [90, 31], [1, 7]),
    (2, 4, 2, 96, 32, [90, 200], [1, 9]),
    (2, 3, 3, 256, 64, [150, 70], [2, 1]),
    (2, 2, 1, 32, 16, [55, 20], [1, 1]),
    (2, 10, 2, 7, 16, [55, 20], [3, 1]),
    (1, 2, 1, 100, 16, [140], [5]),
    (1, 3, 1, 250, 16, [40], [2]),
    (1, 40, 1, 128, 64, [700], [1]),
    (40, 2, 2, 64, 16, list(range(1, 41)), [1] * 40),
    (1, 2, 1, 128, 64, [6000], [1]),
    (2, 8, 2, 128, 64, [1000, 700], [300, 1]),
    (3, 4, 4, 64, 16, [513, 90, 700], [257, 90, 64]),
    (1, 8, 1, 128, 16, [3000], [33]),
    (2, 14, 2, 128, 32, [600, 1300], [513, 37]),
    (1, 70, 1, 64, 16, [300], [2]),
    (2, 4, 2, 48, 16, [70, 33], [1, 1]),
    (2, 4, 4, 112, 32, [70, 333], [3, 1]),
    (1, 1, 1, 16, 16, [100], [1]),
    (2, 20, 2, 240, 16, [77, 150], [1, 2]),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:5])))
def test_attention(ctx, dtype, causal, case):
    B, Hq, Hkv, D, page, lens, news = case
    rng = np.random.default_rng(B * 1000 + D + Hq)
    pr = make_problem(rng, dtype, B, Hq, Hkv, D, page, lens, news)
    out = run_attention(ctx, pr, dtype, causal, Hkv, page)
    ctx.check()
    check_attention(pr, out, dtype, causal, page)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 40])
def test_attention_rows_that_see_nothing(ctx, dtype, D):
    """No keys at all; more new tokens than keys (the first rows lie before the cache's first token)."""
    rng = np.random.default_rng(8)
    pr = make_problem(rng, dtype, 3, 4, 2, D, 16, [0, 20, 5], [3, 50, 5])
    out = run_attention(ctx, pr, dtype, True, 2, 16)
    ctx.check()
    check_attention(pr, out, dtype, True, 16)
    got = out.double().cpu().numpy()
    assert (got[:3] == 0).all() and (got[3:33] == 0).all() and (got[33:53] != 0).any(-1).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,G,new", [(64, 1, 6), (128, 4, 6), (40, 2, 6), (128, 4, 40), (64, 8, 33)])
def test_attention_ignores_what_it_must_not_see(ctx, dtype, D, G, new):
    """NaN behind the last token of a page, and in tokens that a causal row may not see yet."""
    rng = np.random.default_rng(4)
    B, page, Hkv = 2, 16, 2
    pr = make_problem(rng, dtype, B, Hkv * G, Hkv, D, page, [37, 50], [1, new])
    clean = run_attention(ctx, pr, dtype, True, Hkv, page).clone()
    weight = ref.attention(pr["qx"], pr["kc"], pr["vc"], pr["ks"].astype(float), pr["vs"].astype(float), pr["table"],
                           pr["qs"], pr["seq"], page, True)[1]
    pr.pop("dev")

    def same(x, y, w):  # two orders of one sum of 50 terms, each rounded once more to the output's type
        return (np.abs(x - y) <= 2 * 50 * 2.0 ** -23 * w + (2.0 ** -7 if dtype == BF16 else 2.0 ** -23) * np.abs(x)).all()

    for b, L in enumerate(pr["seq"]):
        last = pr["table"][b, (L - 1) // page]
        if L % page:
            pr["kc"][last, :, L % page:] = 127
            pr["vc"][last, :, L % page:] = 127
    p49 = pr["table"][1, 49 // page]
    pr["vc"][p49, :, 49 % page, 5] = 0xFF  # the last token of request 1: only its own row sees it
    pr["kc"][pr["table"][1, 48 // page], 1, 48 % page, :] = 127  # key of token 48, head 1: the last two rows
    out = run_attention(ctx, pr, dtype, True, Hkv, page)
    ctx.check()
    a, b = clean.double().cpu().numpy(), out.double().cpu().numpy()
    rows = pr["qs"][1] + np.arange(new)
    assert np.array_equal(a[0], b[0])
    assert same(a[rows[:-2]], b[rows[:-2]], weight[rows[:-2]])
    assert same(a[rows[-2], :G], b[rows[-2], :G], weight[rows[-2], :G]) and np.isnan(b[rows[-2], G:]).all()
    assert np.isnan(b[rows[-1], :G, 5]).all() and np.isnan(b[rows[-1], G:]).all()
    keep = [d for d in range(D) if d != 5]
    assert same(a[rows[-1], :G][:, keep], b[rows[-1], :G][:, keep], weight[rows[-1], :G][:, keep])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 96])
def test_attention_scales_far_apart(ctx, dtype, D):
    """Pages whose scales differ by 2^40: the small ones still count where the scores favour them."""
    rng = np.random.default_rng(6)
    pr = make_problem(rng, dtype, 2, 4, 2, D, 16, [200, 330], [1, 3])
    pr["vs"] *= np.exp2(rng.integers(-40, 1, pr["vs"].shape)).astype(np.float32)
    out = run_attention(ctx, pr, dtype, True, 2, 16)
    ctx.check()
    check_attention(pr, out, dtype, True, 16)
    pr = make_problem(rng, dtype, 1, 2, 1, D, 16, [64], [1])
    pr["vs"][:] = np.float32(2.0 ** -64)  # pages of zeros, as append leaves them
    pr["vc"][:] = 0
    out = run_attention(ctx, pr, dtype, True, 1, 16)
    assert (out[:1] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [128, 48])
def test_attention_query_magnitudes(ctx, dtype, D):
    """Queries far from one (rows of zeros, of 1e30, of 1e-30) against keys scaled to match."""
    rng = np.random.default_rng(16)
    pr = make_problem(rng, dtype, 1, 4, 1, D, 16, [100], [3])
    f = np.array([1e30, 1e-30, 0.0])
    pr["q"], pr["qx"] = float_dev(pr["qx"] * np.concatenate([f, [1, 1]])[:, None, None], dtype)
    pr["ks"][:] = np.float32(2.0 ** -100)
    out = run_attention(ctx, pr, dtype, False, 1, 16)
    ctx.check()
    check_attention(pr, out, dtype, False, 16)


def test_attention_bad_pages_and_ranges(ctx):
    """Page ids outside the pool, lengths beyond the table, contradictory row ranges: reported, left out, and
    the other requests are right."""
    import munet_b200 as mb
    rng = np.random.default_rng(5)
    for dtype in (F32, BF16):
        for what in ("page", "negative", "long", "range", "length"):
            pr = make_problem(rng, dtype, 3, 4, 2, 64, 16, [100, 70, 90], [1, 2, 1])
            if what == "page":
                pr["table"][1, 2] = pr["kc"].shape[0]
            if what == "negative":
                pr["table"][1, 0] = -1
            if what == "long":
                pr["seq"][1] = 16 * pr["table"].shape[1] + 1
                pr["table"][1] = pr["table"][1, 0]
            if what == "range":
                pr["qs"][1:] = [1, 40, 41]
            if what == "length":
                pr["seq"][1] = -3
            out = run_attention(ctx, pr, dtype, True, 2, 16)
            with pytest.raises(mb.MuNetError) as e:
                ctx.check()
            assert e.value.code == 5
            got = out.double().cpu().numpy()
            want = ref.attention(pr["qx"], pr["kc"], pr["vc"], pr["ks"].astype(float), pr["vs"].astype(float),
                                 pr["table"][:1], [0, 1], pr["seq"][:1], 16, True)[0]
            assert np.abs(got[0] - want[0]).max() <= 0.02 * np.abs(want[0]).max()
            assert np.isfinite(got).all()
            if what == "page":  # tokens 32 .. 47 are left out
                t = pr["table"].copy()
                t[1, 2:] = np.append(t[1, 3:], -1)
                pr2 = dict(pr, table=t, seq=pr["seq"] - [0, 16, 0])
                want = ref.attention(pr["qx"], pr["kc"], pr["vc"], pr["ks"].astype(float), pr["vs"].astype(float), t,
                                     pr["qs"], pr2["seq"], 16, True)[0]
                assert np.abs(got[:4] - want[:4]).max() <= 0.02 * np.abs(want[:4]).max()


def test_attention_without_a_pool(ctx):
    import munet_b200 as mb
    rng = np.random.default_rng(14)
    for dtype, D in ((F32, 64), (BF16, 128), (BF16, 40)):
        pr = make_problem(rng, dtype, 2, 2, 1, D, 16, [20, 3], [1, 1])
        q, out = pr["q"], pr["q"].clone().fill_(7.0)
        n = ctx.attention_paged_workspace_bytes(4, 2, 2, 1, D, dtype)
        ws = dev(np.zeros(n, np.uint8))
        ctx.attention_paged(q, q.stride(0), out, out.stride(0), None, None, None, None, ints(pr["table"]),
                            pr["table"].shape[1], ints(pr["qs"]), ints(pr["seq"]), 2, 4, 2, 1, D, 0, 16, True, dtype, ws, n)
        with pytest.raises(mb.MuNetError) as e:
            ctx.check()
        assert e.value.code == 5
        assert (out[:2] == 0).all() and (out[2:] == 7).all()


@pytest.mark.parametrize("D,new", [(64, 64), (128, 200)])
def test_attention_length_far_beyond_the_table(ctx, D, new):
    """A prompt chunk whose length says a million keys where the table holds 256: those are attended to, the rest is
    reported, and no share of the work that turns out to hold no key leaves its place in the workspace unwritten."""
    import munet_b200 as mb
    import torch
    rng = np.random.default_rng(16)
    pr = make_problem(rng, BF16, 1, 4, 1, D, 16, [256], [new])
    n = ctx.attention_paged_workspace_bytes(new + 2, 1, 4, 1, D, BF16)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN, read as numbers
    out = run_attention(ctx, dict(pr, seq=np.asarray([1_000_000], np.int32)), BF16, True, 1, 16, ws=ws)
    with pytest.raises(mb.MuNetError) as e:
        ctx.check()
    assert e.value.code == 5
    check_attention(pr, out, BF16, False, 16)


def test_attention_two_calls_at_once(ctx):
    """Calls on two streams, a workspace each, among them prompt chunks and single tokens."""
    import torch
    rng = np.random.default_rng(17)
    a = make_problem(rng, BF16, 3, 8, 2, 128, 16, [1500, 700, 90], [300, 1, 40])
    b = make_problem(rng, BF16, 3, 8, 2, 128, 16, [2900, 40, 1700], [1, 1, 1])
    want = [run_attention(ctx, pr, BF16, True, 2, 16).clone() for pr in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ws = [torch.full((ctx.attention_paged_workspace_bytes(pr["n"], 3, 8, 2, 128, BF16),), 0xFF, dtype=torch.uint8,
                     device="cuda") for pr in (a, b)]
    out = [torch.full_like(w, 7.0) for w in want]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, pr in enumerate((a, b)):
            run_attention(ctx, pr, BF16, True, 2, 16, stream=streams[i], ws=ws[i], out=out[i])
    torch.cuda.synchronize()
    ctx.check()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("B,new", [(5000, 1), (3600, 2), (400, 3)])
def test_attention_many_requests(ctx, B, new):
    rng = np.random.default_rng(15)
    lens = rng.integers(new, 40, B).tolist()
    pr = make_problem(rng, BF16, B, 2, 1, 64, 16, lens, [new] * B)
    out = run_attention(ctx, pr, BF16, True, 1, 16)
    ctx.check()
    check_attention(pr, out, BF16, True, 16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_strides_streams_and_repeats(ctx, dtype):
    """Query and output as column slabs of wider tensors, on a side stream; the same bits every time."""
    import torch
    rng = np.random.default_rng(9)
    Hq, Hkv, D = 6, 2, 64
    pr = make_problem(rng, dtype, 4, Hq, Hkv, D, 16, [300, 1200, 5, 64], [1, 9, 1, 1])
    want = run_attention(ctx, pr, dtype, True, Hkv, 16)
    wide_q = torch.randn(pr["n"], 3, Hq, D, device="cuda").to(pr["q"].dtype)
    wide_q[:, 1] = pr["q"]
    wide_o = torch.zeros(pr["n"], 2 * Hq * D + 3, device="cuda", dtype=pr["q"].dtype)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    pr2 = dict(pr, q=wide_q[:, 1])
    for _ in range(3):
        out = wide_o[:, 1:1 + Hq * D].view(pr["n"], Hq, D)
        run_attention(ctx, pr2, dtype, True, Hkv, 16, stream=side, out=out)
        ctx.check(side)
        live = int(pr["qs"][-1])
        assert torch.equal(out[:live], want[:live])
        assert (wide_o[:, 0] == 0).all() and (wide_o[:, 1 + Hq * D:] == 0).all()


def test_attention_cache_beyond_32_bit_offsets(ctx):
    """A pool of more than 2^32 bytes, with the request's pages at its far end."""
    import torch
    H, D, page, dtype = 16, 128, 64, BF16
    num = (5 << 30) // (H * D * page)
    rng = np.random.default_rng(10)
    pr = make_problem(rng, dtype, 1, H, H, D, page, [150], [1])
    small = [dev(pr[k]) for k in ("kc", "vc", "ks", "vs")]
    P = small[0].shape[0]
    big = [torch.empty((num,) + tuple(t.shape[1:]), dtype=t.dtype, device="cuda") for t in small]
    for b, t in zip(big, small):
        b[num - P:] = t
    table = dev(np.where(pr["table"] >= 0, pr["table"] + num - P, -1).astype(np.int32))
    want = run_attention(ctx, dict(pr), dtype, True, H, page)
    pr["dev"] = [*big, table, dev(pr["qs"]), dev(pr["seq"])]
    pr["kc"] = np.empty((num, 0))
    got = run_attention(ctx, pr, dtype, True, H, page)
    ctx.check()
    assert torch.equal(got, want)
    # and the write to its last page
    x, xv = float_dev(rng.standard_normal((1, H, D)), dtype)
    slot = num * page - 1
    ctx.kv_cache_append(x, x, H * D, ints([slot]), 1, *big, num, page, H, D, dtype)
    ctx.check()
    c, s = ref.append(xv, [P * page - 1], small[0].cpu().numpy(), small[2].cpu().numpy(), page)
    assert np.array_equal(big[0][num - 1].cpu().numpy(), c[-1])


# ---- together -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,H,G,D", [(BF16, 2, 2, 64), (F32, 2, 1, 80), (BF16, 1, 8, 128)])
def test_generation_steps_in_a_graph(ctx, dtype, H, G, D):
    """Prompts, then single tokens: page map -> append -> attention -> head -> sample, as a decode loop runs
    them. The single-token step is captured once and replayed; every step is checked against 64 bits."""
    import torch
    rng = np.random.default_rng(12)
    B, page, V, steps = 5, 16, 257, 20
    Hq, td = H * G, torch.bfloat16 if dtype == BF16 else torch.float32
    width, pool = 8, 48
    z = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    kc, vc = z(pool, H, page, D, t=torch.uint8), z(pool, H, page, D, t=torch.uint8)
    ks, vs = z(pool, H, t=torch.float32), z(pool, H, t=torch.float32)
    table, free = z(B, width) - 1, ints(rng.permutation(pool))
    cl, nl, taken = z(B), z(B), z(1)
    cap = 64
    qs, seq, slots, pos = z(B + 1), z(B), z(cap), z(cap)
    x = z(cap, Hq + 2 * H, D, t=td)  # fused projection output: q | k | v
    out, u, idx, prob = z(cap, Hq, D, t=td), z(B, t=torch.float32), z(B), z(B, t=torch.float32)
    T, kk = torch.full((B,), 0.9, device="cuda"), ints([5, 0, 40, 1, 257])
    pp = torch.full((B,), 0.9, device="cuda")
    head = torch.randn(Hq * D, V, device="cuda").to(td) * 0.3
    logits = z(B, V, t=td)
    ws = z(ctx.attention_paged_workspace_bytes(cap, B, Hq, H, D, dtype), t=torch.uint8)
    ld = (Hq + 2 * H) * D

    def step(n):
        ctx.page_map(cl, nl, free, pool, table, width, B, page, pool, qs, seq, slots, pos, n, taken)
        ctx.kv_cache_append(x[:, Hq:Hq + H], x[:, Hq + H:], ld, slots, n, kc, vc, ks, vs, pool, page, H, D, dtype)
        ctx.attention_paged(x, ld, out, Hq * D, kc, vc, ks, vs, table, width, qs, seq, B, n, Hq, H, D, pool, page, True,
                            dtype, ws, ws.numel())
        last = (qs[1:] - 1).long()
        logits.copy_((out[last].reshape(B, -1).float() @ head.float()).to(td))
        ctx.sample(logits, V, u, T, kk, pp, None, idx, prob, B, V, dtype)

    model = dict(kc=kc.cpu().numpy(), vc=vc.cpu().numpy(), ks=ks.cpu().numpy(), vs=vs.cpu().numpy(),
                 table=table.cpu().numpy(), at=0, ctx=[0] * B)

    def verify(news):
        n = sum(news)
        t, q0, s, sl, ps, got = ref.page_map(model["ctx"], news, free.cpu().numpy().tolist(), model["table"], page, n)
        assert np.array_equal(table.cpu().numpy(), t) and qs.tolist() == q0 and slots.tolist()[:n] == sl
        assert taken.item() == got and pos.tolist()[:n] == ps
        xs = x[:n].double().cpu().numpy()
        model["kc"], model["ks"] = ref.append(xs[:, Hq:Hq + H], sl, model["kc"], model["ks"], page)
        model["vc"], model["vs"] = ref.append(xs[:, Hq + H:], sl, model["vc"], model["vs"], page)
        assert np.array_equal(kc.cpu().numpy(), model["kc"]) and np.array_equal(vc.cpu().numpy(), model["vc"])
        pr = dict(model, table=t, qx=xs[:, :Hq], qs=np.asarray(q0), seq=np.asarray(s))
        check_attention(pr, out[:n], dtype, True, page)
        lg, uu = logits.double().cpu().numpy(), u.cpu().numpy()
        for b in range(B):
            w = ref.sample(lg[b], float(uu[b]), float(T[b]), int(kk[b]), float(pp[b]))
            assert idx[b].item() == w[0] and abs(prob[b].item() - w[1]) <= 1e-6
        model["table"], model["ctx"] = t, s
        free.copy_(torch.roll(free, -got))

    def refill(news, n):
        x[:n].copy_(torch.randn(n, Hq + 2 * H, D, device="cuda") * (1 + 3 * rng.random()))
        u.copy_(torch.rand(B, device="cuda"))
        cl.copy_(ints(model["ctx"]))
        nl.copy_(ints(news))

    prompts = [9, 16, 1, 25, 7]
    refill(prompts, 58)
    step(58)
    verify(prompts)
    graph = torch.cuda.CUDAGraph()
    refill([1] * B, B)
    with torch.cuda.graph(graph):
        step(B)
    for _ in range(steps):
        refill([1] * B, B)
        graph.replay()
        verify([1] * B)
    ctx.check()


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 4, 4)])
def test_mixed_call_in_a_graph(ctx, D, Hq, Hkv):
    """Prompt chunks and single tokens in one captured call, whose kernels overlap: what follows in the graph finds
    every row, and the next replay may write the same rows and workspace again."""
    import torch
    rng = np.random.default_rng(18)
    pr = make_problem(rng, BF16, 6, Hq, Hkv, D, 16, [1300, 70, 900, 400, 33, 2100], [260, 1, 1, 200, 1, 30])
    want = run_attention(ctx, pr, BF16, True, Hkv, 16).clone()
    check_attention(pr, want, BF16, True, 16)
    ws = torch.full((ctx.attention_paged_workspace_bytes(pr["n"], 6, Hq, Hkv, D, BF16),), 0xFF, dtype=torch.uint8,
                    device="cuda")
    out, kept = torch.full_like(want, 7.0), torch.zeros(40, *want.shape, dtype=want.dtype, device="cuda")
    turn = torch.zeros(1, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_attention(ctx, pr, BF16, True, Hkv, 16, ws=ws, out=out)
        kept.index_copy_(0, turn, out[None])
        out.fill_(7.0)
        ws.fill_(0xFF)
        turn += 1
    for _ in range(40):
        graph.replay()
    torch.cuda.synchronize()
    ctx.check()
    assert all(torch.equal(k, want) for k in kept)


def test_two_graphs_that_share_a_workspace_in_turn(ctx):
    """Two captured calls with different lengths use one workspace one after the other."""
    import torch
    rng = np.random.default_rng(13)
    a = make_problem(rng, BF16, 1, 8, 2, 128, 16, [2500], [1])
    b = make_problem(rng, BF16, 3, 8, 2, 128, 16, [900, 40, 1700], [1, 1, 1])
    wa, wb = run_attention(ctx, a, BF16, True, 2, 16).clone(), run_attention(ctx, b, BF16, True, 2, 16).clone()
    ws = torch.empty(ctx.attention_paged_workspace_bytes(8, 3, 8, 2, 128, BF16), dtype=torch.uint8, device="cuda")
    oa, ob = torch.full_like(wa, 7.0), torch.full_like(wb, 7.0)
    graphs = []
    for pr, o in ((a, oa), (b, ob)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run_attention(ctx, pr, BF16, True, 2, 16, ws=ws, out=o)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(oa, wa) and torch.equal(ob, wb)
