"""Sampling against a 64-bit restatement: tokens are equal, probabilities to the rounding of float32."""
import numpy as np
import pytest

from oracle import BF16, F32
from tests import paged_reference as ref
from tests.test_gpu_paged_cache import dev, float_dev, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import munet_b200 as mb
    c = mb.Context(0)
    yield c
    c.close()


def run(ctx, x, u, dtype, T=None, k=None, p=None, mp=None, cols=None, stream=None):
    import torch
    rows, ld = x.shape
    idx = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -9.0, device="cuda")
    f = lambda a: None if a is None else dev(np.asarray(a, np.float32))  # noqa: E731
    ctx.sample(x, ld, f(u), f(T), None if k is None else ints(k), f(p), f(mp), idx, prob, rows, cols or ld, dtype,
               stream=stream)
    ctx.check(stream)
    return idx.cpu().numpy(), prob.cpu().numpy()


def check(ctx, xv, u, dtype, T=None, k=None, p=None, mp=None, cols=None):
    x, xd = float_dev(xv, dtype)
    idx, prob = run(ctx, x, u, dtype, T, k, p, mp, cols)
    u = np.asarray(u, np.float32).astype(float)
    at = lambda a, r, d: d if a is None else float(np.float32(a[r]))  # noqa: E731
    for r in range(len(xd)):
        w = ref.sample(xd[r, :cols], u[r], at(T, r, 1.0), int(at(k, r, 0)), at(p, r, 1.0), at(mp, r, 0.0))
        assert idx[r] == w[0], (r, idx[r], w)
        assert abs(prob[r] - w[1]) <= 2.0 ** -23 * w[1] + 1e-12
    return idx, prob


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (2, 31), (5, 33), (7, 1000), (1, 32000), (40, 4099), (300, 257),
                                       (2, 100003), (1, 262147), (1, 500009)])
def test_sample(ctx, dtype, rows, cols):
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)) * 3
    n = lambda lo, hi: rng.uniform(lo, hi, rows).astype(np.float32)  # noqa: E731
    u = n(0, 1)
    check(ctx, x, u, dtype)
    check(ctx, x, u, dtype, T=n(0.2, 2))
    check(ctx, x, u, dtype, k=rng.integers(-1, cols + 2, rows))
    check(ctx, x, u, dtype, k=rng.integers(1, 60, rows), T=n(0.5, 1.5))
    check(ctx, x, u, dtype, p=n(0, 1.1))
    check(ctx, x, u, dtype, mp=n(-0.1, 0.5))
    check(ctx, x, u, dtype, T=n(0.5, 2), k=rng.integers(1, cols + 1, rows), p=n(0.3, 1), mp=n(0, 0.2))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_go_to_the_lowest_index(ctx, dtype):
    rng = np.random.default_rng(0)
    cols = 9001
    x = rng.integers(0, 3, (12, cols)).astype(float)  # thousands of equal logits
    x[3] = 1.25
    x[4, :] = 0.0
    x[4, ::2] = -0.0  # equal values
    u = np.linspace(0, 0.9999, 12).astype(np.float32)
    check(ctx, x, u, dtype, k=np.arange(12) * 500 + 1)
    check(ctx, x, u, dtype, p=np.linspace(0, 0.99, 12))
    check(ctx, x, u, dtype, k=np.arange(12) * 700 + 1, p=np.linspace(0.99, 0.1, 12), T=np.full(12, 0.7))
    idx, _ = check(ctx, x, u, dtype, T=np.zeros(12))
    assert (idx == [int(np.argmax(r)) for r in x]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_infinite_and_nan_logits(ctx, dtype):
    inf, nan, low = np.inf, np.nan, float(np.finfo(np.float32).min) if dtype == F32 else -3.3895313892515355e38
    x = np.full((10, 50), -inf)
    x[1, 7] = 2.0
    x[2] = nan
    x[3, [4, 9]], x[3, 20] = inf, 5.0
    x[4] = low
    x[5] = low
    x[5, 13] = 0.0
    x[6, 3], x[6, 4:] = nan, 1.0
    x[7, 49] = -3.0e38
    x[8], x[8, 0] = nan, inf
    x[9, :] = np.arange(50)
    for u in (0.0, 0.3, 0.999999):
        uu = np.full(10, u, np.float32)
        for kw in ({}, dict(k=[3] * 10), dict(p=[0.5] * 10), dict(mp=[0.1] * 10), dict(T=[1e-3] * 10), dict(T=[0.0] * 10),
                   dict(T=[1e30] * 10), dict(k=[40] * 10, p=[0.7] * 10, mp=[0.01] * 10, T=[0.8] * 10)):
            idx, prob = check(ctx, x, uu, dtype, **kw)
            assert idx[0] == -1 and idx[2] == -1 and prob[0] == 0 and idx[1] == 7


def test_odd_parameters(ctx):
    """Uniform numbers at and outside their range, parameters outside theirs."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 300))
    xt, xd = float_dev(x, F32)
    idx, _ = run(ctx, xt, [1.0, 2.0, -1.0, np.nan, 0.0, 1 - 2.0 ** -24], F32)
    assert idx[0] == 299 and idx[1] == 299 and idx[2] == 0 and idx[3] == 0 and idx[4] == 0 and idx[5] == 299
    top = xd.argmax(1)
    for kw in (dict(mp=[1.0] * 6), dict(mp=[5.0] * 6), dict(p=[0.0] * 6), dict(p=[-1.0] * 6), dict(k=[1] * 6),
               dict(T=[-1.0] * 6), dict(T=[np.nan] * 6), dict(T=[1e-30] * 6)):
        idx, prob = run(ctx, xt, [0.7] * 6, F32, **kw)
        assert (idx == top).all() and (prob == 1).all(), kw
    a = run(ctx, xt, [0.7] * 6, F32)
    for kw in (dict(p=[np.nan] * 6), dict(mp=[np.nan] * 6), dict(k=[-3] * 6), dict(k=[300] * 6), dict(p=[1.0] * 6)):
        b = run(ctx, xt, [0.7] * 6, F32, **kw)
        assert (a[0] == b[0]).all() and (a[1] == b[1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_row_stride_stream_and_graph(ctx, dtype):
    import torch
    rng = np.random.default_rng(2)
    x = rng.standard_normal((9, 1003))
    x[:, 1000:] = 50.0  # behind the row's end
    u = rng.random(9).astype(np.float32)
    idx, prob = check(ctx, x, u, dtype, k=[20] * 9, p=[0.9] * 9, cols=1000)
    side = torch.cuda.Stream()
    xt, _ = float_dev(x, dtype)
    torch.cuda.synchronize()
    i2, p2 = run(ctx, xt, u, dtype, k=[20] * 9, p=[0.9] * 9, cols=1000, stream=side)
    assert (idx == i2).all() and (prob == p2).all()
    ut, kt = dev(u), ints([20] * 9)
    o = torch.zeros(9, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.sample(xt, 1003, ut, None, kt, None, None, o, None, 9, 1000, dtype)
    for _ in range(3):
        un = rng.random(9).astype(np.float32)
        ut.copy_(dev(un))
        g.replay()
        want, _ = run(ctx, xt, un, dtype, k=[20] * 9, cols=1000)
        assert (o.cpu().numpy() == want).all()


def test_follows_the_distribution(ctx):
    """Evenly spaced uniform numbers give every token its share of them, to one draw at either end."""
    rng = np.random.default_rng(3)
    x = np.repeat(rng.standard_normal((1, 64)) * 2, 4096, 0)
    u = (np.arange(4096) + 0.5) / 4096
    xt, xd = float_dev(x, F32)
    idx, _ = run(ctx, xt, u, F32)
    p = np.exp(xd[0] - xd[0].max())
    p /= p.sum()
    assert np.abs(np.bincount(idx, minlength=64) - p * 4096).max() <= 1.0 + 1e-6
