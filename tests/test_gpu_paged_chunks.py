"""The prompt-chunk kernel of the paged attention over several works per CTA, against 64 bits.

The kernel is persistent: a CTA goes from one (request, head, row tile, key range) to the next with its barriers,
query tiles and tensor memory as the work before left them. The cases here give every CTA several works, of one and of
two query tiles, whole and split, and say so by replaying the kernel's work split."""
import math

import numpy as np
import pytest

from oracle import BF16
from tests import paged_reference as ref
from tests.test_gpu_paged_cache import make_problem, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import munet_b200 as mb
    c = mb.Context(0)
    yield c
    c.close()


def cdiv(a, b):
    return -(-a // b)


def works_of(lens, news, G, Hkv, causal, sms):
    """Per CTA the works (request, head, row tile, key tiles of it, key tiles of the item)."""
    start = 112  # units of 8 keys that beginning an item counts for
    upto, of, total = [], [], 0
    for L, n in zip(lens, news):
        if n * G >= 73:
            tokens = 255 // G + 2  # that a tile of 256 rows can span, and one
            slope = cdiv(tokens, 8) if causal else 0
            first = start + cdiv(max(L - n, 0) + tokens if causal else L, 8) + 1
            tiles = cdiv(n * G, 256)
            before = [t * first + t * (t - 1) // 2 * slope for t in range(tiles + 1)]
            total += before[-1] * Hkv
            of.append((before, first, slope))
        else:
            of.append(None)
        upto.append(total)
    ctas = min(sms, max(1, total // 64))
    out = []
    for me in range(ctas):
        u, end, mine = total * me // ctas, total * (me + 1) // ctas, []
        while u < end:
            b = next(i for i, x in enumerate(upto) if x > u)
            before, first, slope = of[b]
            head, rem = divmod(u - (upto[b - 1] if b else 0), before[-1])
            tile = max(t for t in range(len(before) - 1) if before[t] <= rem)
            cost, at = first + tile * slope, rem - before[tile]
            to = min(cost, at + end - u)
            u += to - at
            last = min((tile + 1) * 256, news[b] * G) - 1
            keys = max(0, min(lens[b], lens[b] - news[b] + last // G + 1)) if causal else lens[b]
            nc = max(1, cdiv(keys, 128))
            c0, c1 = (0 if x <= start else (x - start) * nc // (cost - start) for x in (at, to))
            if c1 > c0:
                mine.append((b, head, tile, c1 - c0, nc))
        out.append(mine)
    return out


def expect(pr, causal, page):
    """(out, bound) in 64 bits, on the GPU. The bound is the one derived beside check_attention of the general tests: per
    score 2^-23 a step over D products, which moves a probability by that much of itself; fp16 probabilities; pieces of
    2^-23 a step over the keys; an absolute quantum of fp16 weights; half a step of bfloat16 on the output."""
    import torch
    n, Hq, D = pr["q"].shape
    f64 = dict(dtype=torch.float64, device="cuda")
    table = torch.tensor(ref.TABLE, **f64)
    kc, vc, ks, vs = (torch.from_numpy(pr[k]).cuda() for k in ("kc", "vc", "ks", "vs"))
    Hkv = kc.shape[1]
    G = Hq // Hkv
    out, bound = torch.zeros(n, Hq, D, **f64), torch.zeros(n, Hq, D, **f64)
    for b, L in enumerate(pr["seq"].tolist()):
        a, e = int(pr["qs"][b]), int(pr["qs"][b + 1])
        if a == e or L == 0:
            continue
        ids = torch.from_numpy(pr["table"][b, :cdiv(L, page)].astype(np.int64)).cuda()

        def whole(cache, scale):  # [Hkv, L, D]
            x = table[cache[ids].long()] * scale[ids].double()[..., None, None]
            return x.transpose(0, 1).reshape(Hkv, -1, D)[:, :L]
        k, v = whole(kc, ks), whole(vc, vs)
        q = pr["q"][a:e].double().view(e - a, Hkv, G, D).permute(1, 2, 0, 3)  # [Hkv, G, n, D]
        seen = torch.ones(e - a, L, device="cuda", dtype=torch.bool)
        if causal:
            seen = seen.tril(L - (e - a))
        s = (q @ k.transpose(1, 2)[:, None] / math.sqrt(D)).masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        spread = (q.abs() @ k.abs().transpose(1, 2)[:, None] * seen).amax(-1) / math.sqrt(D)
        most = (w * vs[ids].double().t().repeat_interleave(page, 1)[:, None, None, :L]).amax(-1)
        o, weight = w @ v[:, None], w @ v.abs()[:, None]
        prob = 2 * (D + 4) * 2.0 ** -23 * spread + 2.0 ** -20 + 2.0 ** -11 + L * 2.0 ** -23
        lim = 2.0 ** -8 * o.abs() + 2 * prob[..., None] * weight + (L * 448 * 2.0 ** -32 * most)[..., None] + 1e-30
        back = lambda x: x.permute(2, 0, 1, 3).reshape(e - a, Hq, D)  # noqa: E731
        out[a:e], bound[a:e] = back(o), back(lim)
    return out, bound


def check(pr, out, want, bound):
    live = int(pr["qs"][-1])
    got = out.double()
    assert (got[live:] == 7.0).all(), "rows behind the last request changed"
    worst = ((got - want).abs()[:live] / bound[:live].clamp(min=1e-30)).max().item()
    assert worst <= 1.0, f"worst error / bound {worst:.3g}"  # NaN fails too


def mixture(rng, B, most):
    """Requests of 73 to `most` rows at eight heads per group, some of one token, with unlike lengths."""
    news = rng.integers(10, most // 8 + 1, B)
    news[rng.random(B) < 0.1] = 1
    lens = news + rng.integers(0, 500, B)
    lens[::7] += 900  # long ones between them
    lens[3] = news[3] - 4  # rows before the cache's first token
    return lens.tolist(), news.tolist()


RNG = np.random.default_rng(21)
CASES = {  # lens, news, G, Hkv, least number of works that some CTA does
    "80 rows": ([200 + i for i in range(64)], [10] * 64, 8, 8, 4),
    "176 rows": ([300 - i for i in range(64)], [22] * 64, 8, 8, 4),
    "one and two query tiles": (*mixture(RNG, 64, 300), 8, 8, 4),
    "80 rows over 1024 keys": ([1024] * 40, [10] * 40, 8, 8, 3),
    "several row tiles": ([700, 90, 1100, 420, 333, 901], [560, 90, 300, 410, 64, 129], 4, 16, 4),
    "one head a group": ([150 + 3 * i for i in range(40)], [73 + 3 * i for i in range(40)], 1, 12, 4),
}


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", CASES)
def test_several_works_per_cta(ctx, case, D, causal, aligned):
    """Right, and the same bits twenty times over. Rows of `out` that are not 16-byte aligned leave two bytes at a time,
    which holds the warps that have rows back against those that have none."""
    import torch
    lens, news, G, Hkv, least = CASES[case]
    works = works_of(lens, news, G, Hkv, causal, ctx.num_sms)
    assert max(len(w) for w in works) >= least
    assert any(w[3] < w[4] for mine in works for w in mine) and any(w[3] == w[4] for mine in works for w in mine)
    rng = np.random.default_rng(D + len(lens))
    pr = make_problem(rng, BF16, len(lens), G * Hkv, Hkv, D, 16, lens, news)
    want, bound = expect(pr, causal, 16)
    n, Hq = pr["n"], G * Hkv
    first = None
    for _ in range(20):
        wide = torch.full((n, Hq * D + (0 if aligned else 3)), 7.0, dtype=torch.bfloat16, device="cuda")
        out = wide[:, (0 if aligned else 1):][:, :Hq * D].view(n, Hq, D)
        run_attention(ctx, pr, BF16, causal, Hkv, 16, out=out)
        if first is None:
            check(pr, out, want, bound)
            first = out.clone()
        assert torch.equal(out, first)
        assert aligned or ((wide[:, 0] == 7).all() and (wide[:, 1 + Hq * D:] == 7).all())
    ctx.check()


@pytest.mark.parametrize("D", [64, 128])
def test_a_query_tile_that_sits_out_long_works(ctx, D):
    """Works of one query tile over many key tiles, then works of two: the second tile's warps come from far ahead of the
    keys and values, with scales that differ from page to page."""
    import torch
    B, G, page = 240, 8, 16
    news = [10 if b % 2 else 25 for b in range(B)]
    lens = [1500 + 3 * b for b in range(B)]
    works = works_of(lens, news, G, 1, True, ctx.num_sms)
    # more than two turns of the four slots with one query tile, then two of them
    assert sum(a[3] > 8 and news[a[0]] * G <= 128 and news[b[0]] * G > 128 for w in works for a, b in zip(w, w[1:])) > 20
    rng = np.random.default_rng(D)
    pr = make_problem(rng, BF16, B, G, 1, D, page, lens, news)
    pr["ks"] *= np.exp2(rng.integers(-3, 2, pr["ks"].shape)).astype(np.float32)
    pr["vs"] *= np.exp2(rng.integers(-6, 7, pr["vs"].shape)).astype(np.float32)
    want, bound = expect(pr, True, page)
    first = run_attention(ctx, pr, BF16, True, 1, page)
    check(pr, first, want, bound)
    for _ in range(10):
        assert torch.equal(run_attention(ctx, pr, BF16, True, 1, page), first)
    ctx.check()


@pytest.mark.parametrize("D", [64, 128])
def test_a_captured_call_whose_lengths_change(ctx, D):
    """Lengths, tables and row ranges are the device's: one captured call serves chunks, single tokens, an empty batch and
    padded tokens."""
    import torch
    B, G, Hkv, page, cap = 6, 4, 2, 16, 400
    rng = np.random.default_rng(D)
    steps = [([300, 40, 1, 0, 30, 1], [900, 40, 700, 0, 31, 16]), ([1] * 6, [901, 41, 701, 1, 32, 17]), ([0] * 6, [901, 41, 701, 1, 32, 17]),
             ([66, 66, 66, 66, 66, 66], [66, 1000, 300, 67, 2000, 80])]
    width = 2000 // page + 2
    pr = make_problem(rng, BF16, B, G * Hkv, Hkv, D, page, [2000] * B, [1] * B)
    num = pr["kc"].shape[0]
    pr["table"] = rng.permutation(num)[:B * (2000 // page)].reshape(B, -1).astype(np.int32)
    pr["table"] = np.concatenate([pr["table"], np.full((B, width - pr["table"].shape[1]), -1, np.int32)], 1)
    pr["q"], pr["n"] = torch.randn(cap, G * Hkv, D, device="cuda").to(torch.bfloat16), cap
    pr["dev"] = [torch.from_numpy(pr[k]).cuda() for k in ("kc", "vc", "ks", "vs", "table", "qs", "seq")]
    ws = torch.full((ctx.attention_paged_workspace_bytes(cap, B, G * Hkv, Hkv, D, BF16),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full_like(pr["q"], 7.0)
    run_attention(ctx, pr, BF16, True, Hkv, page, ws=ws, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_attention(ctx, pr, BF16, True, Hkv, page, ws=ws, out=out)
    for news, lens in steps * 3:
        pr["qs"], pr["seq"] = np.concatenate([[0], np.cumsum(news)]).astype(np.int32), np.asarray(lens, np.int32)
        pr["dev"][5].copy_(torch.from_numpy(pr["qs"]))
        pr["dev"][6].copy_(torch.from_numpy(pr["seq"]))
        out.fill_(7.0)
        graph.replay()
        ctx.check()
        if sum(news):
            check(pr, out, *expect(pr, True, page))
        assert (out[sum(news):] == 7).all()


@pytest.mark.parametrize("D,new", [(128, 40), (64, 100), (100, 2)])
def test_offsets_beyond_32_bits(ctx, D, new):
    """Pages at the far end of a pool of more than 2^32 bytes, and rows of q and out over 2^33 elements."""
    import torch
    G, Hkv, page = 4, 2, 64
    rng = np.random.default_rng(D)
    pr = make_problem(rng, BF16, 2, G * Hkv, Hkv, D, page, [300, 150], [new, 1], pad_rows=0)
    want = run_attention(ctx, pr, BF16, True, Hkv, page)
    small = pr["dev"][:4]
    P, num = small[0].shape[0], (9 << 29) // (Hkv * D * page)
    big = [torch.empty((num,) + tuple(t.shape[1:]), dtype=t.dtype, device="cuda") for t in small]
    for b, t in zip(big, small):
        b[num - P:] = t
    table = torch.from_numpy(np.where(pr["table"] >= 0, pr["table"] + num - P, -1).astype(np.int32)).cuda()
    far = dict(pr, dev=[*big, table, *pr["dev"][5:]], kc=np.empty((num, 0)))
    assert torch.equal(run_attention(ctx, far, BF16, True, Hkv, page), want)
    del big, far
    ld = 2 ** 33 // pr["n"] // 8 * 8
    q, out = (torch.empty(pr["n"] * ld, dtype=torch.bfloat16, device="cuda").view(pr["n"], ld)[:, :G * Hkv * D] for _ in range(2))
    q, out = (t.view(pr["n"], G * Hkv, D) for t in (q, out))
    q.copy_(pr["q"])
    assert torch.equal(run_attention(ctx, dict(pr, q=q), BF16, True, Hkv, page, out=out), want)
    ctx.check()
