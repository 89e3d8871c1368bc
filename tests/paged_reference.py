"""64-bit restatements of the paged-cache operators and of sampling, for the tests (numpy only)."""
import math

import numpy as np

E4M3_MAX = 448.0


def e4m3_table():
    """Value of every e4m3 code (no infinities; 0x7f and 0xff are NaN)."""
    out = np.empty(256)
    for c in range(256):
        s, e, m = -1.0 if c & 128 else 1.0, (c >> 3) & 15, c & 7
        out[c] = s * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
        if c & 127 == 127:
            out[c] = np.nan
    return out


TABLE = e4m3_table()
_POS = TABLE[:127]  # ascending, 0 .. 448


def to_e4m3(v):
    """Nearest code, ties to the even one, saturating; NaN -> 0x7f."""
    v = np.asarray(v, np.float64)
    a = np.abs(np.where(np.isnan(v), 0.0, v)).clip(max=E4M3_MAX)
    hi = np.searchsorted(_POS, a).clip(max=126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(a == _POS[hi], hi, code)
    return np.where(np.isnan(v), 127, code | (np.signbit(v).astype(np.int64) << 7)).astype(np.uint8)


def page_scale(amax):
    x = -64
    while amax > E4M3_MAX * 2.0 ** x:
        x += 1
    return 2.0 ** x


def page_map(ctx, new, free, table, page, n_slots):
    """(table, query_start, seq, slots, positions, taken) for lengths that fit."""
    table, at = table.copy(), 0
    qs, slots, pos = [0], [], []
    for r, (c, n) in enumerate(zip(ctx, new)):
        for j in range(-(-c // page), -(-(c + n) // page)):
            table[r, j] = free[at]
            at += 1
        for p in range(c, c + n):
            slots.append(table[r, p // page] * page + p % page)
            pos.append(p)
        qs.append(qs[-1] + n)
    pad = n_slots - len(slots)
    return table, qs, [c + n for c, n in zip(ctx, new)], slots + [-1] * pad, pos + [0] * pad, at


def append(x, slots, cache, scale, page):
    """cache [P,H,page,D] codes and scale [P,H], updated copies; x [n,H,D] float64."""
    cache, scale = cache.copy(), scale.astype(np.float64).copy()
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        p, e = slots[t] // page, t
        while e < len(slots) and slots[e] >= 0 and slots[e] // page == p:
            e += 1
        low = min(s % page for s in slots[t:e])
        for h in range(x.shape[1]):
            v = x[t:e, h]
            fin = np.abs(v[np.isfinite(v)])
            need = page_scale(fin.max() if fin.size else 0.0)
            now = max(scale[p, h], need) if low else need
            if low and now > scale[p, h]:
                cache[p, h, :low] = to_e4m3(TABLE[cache[p, h, :low]] * (scale[p, h] / now))
            scale[p, h] = now
            for i in range(t, e):
                cache[p, h, slots[i] % page] = to_e4m3(x[i, h] / now)
        t = e
    return cache, scale


def attention(q, kc, vc, ks, vs, table, query_start, seq, page, causal):
    """(out, weight, spread, top): the result and sum_j p_j |v_j|, [n,Hq,D]; per row max_j sum_d |q_d k_jd| / sqrt(D)
    and max_j p_j vs_j (vs: the scale of key j's page)."""
    n, Hq, D = q.shape
    Hkv = kc.shape[1]
    G = Hq // Hkv
    out, weight, spread, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, Hq)), np.zeros((n, Hq))
    for b in range(len(seq)):
        L, a, e = seq[b], query_start[b], query_start[b + 1]
        ids = table[b, :-(-L // page)]
        for h in range(Hkv):
            k = (TABLE[kc[ids, h]] * ks[ids, h][:, None, None]).reshape(-1, D)[:L]
            v = (TABLE[vc[ids, h]] * vs[ids, h][:, None, None]).reshape(-1, D)[:L]
            for i in range(a, e):
                lim = min(L, L - (e - a) + (i - a) + 1) if causal else L
                if lim <= 0:
                    continue
                for g in range(h * G, (h + 1) * G):
                    s = k[:lim] @ q[i, g] / math.sqrt(D)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[i, g], weight[i, g] = w @ v[:lim], w @ np.abs(v[:lim])
                    top[i, g] = (w * np.repeat(vs[ids, h], page)[:lim]).max()
                    spread[i, g] = (np.abs(k[:lim]) @ np.abs(q[i, g])).max() / math.sqrt(D)
    return out, weight, spread, top


def sample(x, u, T=1.0, k=0, p=1.0, min_p=0.0):
    """(token, probability) of one row of float64 logits. Weights count in multiples of 2^-42 of the largest, as
    the operator defines them: one below half of that is never drawn, not even for u = 0."""
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return -1, 0.0
    if not T > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore"):
        raw = np.where(x == m, 1.0, 0.0 if m == np.inf else np.exp((x - m) / T))
    w = np.rint(raw * 2.0 ** 42)  # whole numbers below 2^53: the sums are exact
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        order = order[:max(1, int(((c - w[order]) < np.ceil(p * c[-1])).sum()))]
    order = np.sort(order[raw[order] >= min(min_p, 1.0)])
    c = np.cumsum(w[order])
    i = min(int((c <= u * c[-1]).sum()), len(order) - 1)
    return int(order[i]), raw[order[i]] * 2.0 ** 42 / c[-1]
