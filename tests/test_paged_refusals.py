"""Argument checks of the paged-cache and sampling entry points (CPU: they come before any device call).

The checks only need a context to write their message to; a zeroed block stands in for one, so that no
device is touched. Calls that pass the checks would go on to the device and are not made here."""
import ctypes as C

import pytest

import munet_b200 as mb

F32, F16, BF16 = 0, 1, 2
INVALID, UNSUPPORTED, SIZE = 1, 2, 7
P = 4096  # some 16-byte aligned, non-null address: never dereferenced


@pytest.fixture
def ctx():
    return C.create_string_buffer(4096)


def page_map(ctx, context=P, new=P, free=P, n_free=4, table=P, stride=4, B=2, page=16, pages=8, qs=P, seq=P,
             slots=P, pos=P, n_slots=4, taken=P):
    return mb.lib().mu_page_map(ctx, context, new, free, n_free, table, stride, B, page, pages, qs, seq, slots, pos,
                                n_slots, taken, None)


def append(ctx, k=P, v=P, ld=32, slots=P, n=3, kc=P, vc=P, ks=P, vs=P, pages=8, page=16, H=2, D=16, dtype=BF16):
    return mb.lib().mu_kv_cache_append(ctx, k, v, ld, slots, n, kc, vc, ks, vs, pages, page, H, D, dtype, None)


def attend(ctx, q=P, q_ld=64, out=P, out_ld=64, kc=P, vc=P, ks=P, vs=P, table=P, stride=4, qs=P, seq=P, B=2, n=2,
           Hq=4, Hkv=2, D=16, pages=8, page=16, causal=1, dtype=BF16, ws=P, ws_bytes=1 << 30):
    return mb.lib().mu_attention_paged(ctx, q, q_ld, out, out_ld, kc, vc, ks, vs, table, stride, qs, seq, B, n, Hq,
                                       Hkv, D, pages, page, causal, dtype, ws, ws_bytes, None)


def sample(ctx, x=P, ld=10, u=P, T=None, k=None, p=None, mp=None, idx=P, prob=None, rows=2, cols=10, dtype=F32):
    return mb.lib().mu_sample(ctx, x, ld, u, T, k, p, mp, idx, prob, rows, cols, dtype, None)


REFUSED = [
    (page_map, dict(B=-1), INVALID), (page_map, dict(page=0), INVALID), (page_map, dict(n_slots=-1), INVALID),
    (page_map, dict(B=16385), SIZE), (page_map, dict(pages=1 << 27, page=16), SIZE),
    (page_map, dict(context=None), INVALID), (page_map, dict(qs=None), INVALID), (page_map, dict(taken=None), INVALID),
    (page_map, dict(free=None), INVALID), (page_map, dict(table=None), INVALID), (page_map, dict(pos=None), INVALID),
    (append, dict(n=-1), INVALID), (append, dict(H=0), INVALID), (append, dict(D=0), INVALID),
    (append, dict(ld=31), INVALID), (append, dict(k=None), INVALID), (append, dict(ks=None), INVALID),
    (append, dict(page=24), UNSUPPORTED), (append, dict(page=1040), UNSUPPORTED),
    (append, dict(D=264, ld=4096), UNSUPPORTED), (append, dict(dtype=F16), UNSUPPORTED),
    (append, dict(vc=P + 8), INVALID), (append, dict(pages=1 << 27), SIZE),
    (append, dict(n=1 << 30, H=1024, ld=1 << 20), SIZE),
    (attend, dict(B=-1), INVALID), (attend, dict(Hq=3), INVALID), (attend, dict(q_ld=63), INVALID),
    (attend, dict(out_ld=63), INVALID), (attend, dict(page=8), UNSUPPORTED), (attend, dict(D=257, q_ld=2048), UNSUPPORTED),
    (attend, dict(dtype=F16), UNSUPPORTED), (attend, dict(dtype=3), UNSUPPORTED), (attend, dict(out=None), INVALID),
    (attend, dict(table=None), INVALID), (attend, dict(ws=None), INVALID), (attend, dict(ws=P + 4), INVALID),
    (attend, dict(ws_bytes=8), INVALID), (attend, dict(kc=P + 1), INVALID), (attend, dict(pages=1 << 27), SIZE),
    (attend, dict(B=16385), SIZE), (attend, dict(n=1 << 30), SIZE),
    (sample, dict(cols=0), INVALID), (sample, dict(rows=-1), INVALID), (sample, dict(ld=9), INVALID),
    (sample, dict(x=None), INVALID), (sample, dict(u=None), INVALID), (sample, dict(idx=None), INVALID),
    (sample, dict(cols=(1 << 20) + 1, ld=1 << 21), SIZE), (sample, dict(dtype=F16), UNSUPPORTED),
]


@pytest.mark.parametrize("call,change,code", REFUSED)
def test_refused(ctx, call, change, code):
    assert call(ctx, **change) == code
    assert mb.lib().mu_last_error(ctx).decode().startswith(
        {page_map: "page_map", append: "kv_cache_append", attend: "attention_paged", sample: "sample"}[call])


def test_no_context():
    assert [f(None) for f in (page_map, append, attend, sample)] == [INVALID] * 4


def test_empty_calls_do_nothing(ctx):
    assert append(ctx, n=0, k=None) == 0
    assert attend(ctx, n=0, q=None) == 0 and attend(ctx, B=0, q=None) == 0
    assert sample(ctx, rows=0, x=None) == 0
    assert mb.lib().mu_attention_paged_workspace_bytes(ctx, 0, 1, 4, 2, 16, BF16) == 0
