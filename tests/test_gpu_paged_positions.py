"""The positions that the page map writes, on their way into the embedding of ragged and padded tokens."""
import numpy as np
import pytest
import torch

from oracle import BF16, F32
from tests import paged_reference as ref
from tests.test_gpu_paged_cache import ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import munet_b200 as mb
    c = mb.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_positions_feed_the_embedding(ctx, dtype):
    """Token rows plus the position table's rows of the page map's positions, captured and replayed as lengths change. A
    sum of two entries is rounded once in float32 and once to its type, half a step each."""
    td = torch.bfloat16 if dtype == BF16 else torch.float32
    B, page, pool, V, longest, d, cap = 4, 16, 40, 50, 128, 96, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens, places = (torch.randn(r, d, generator=g, device="cuda").to(td) for r in (V, longest))
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    cl, nl, table, free = z(B), z(B), z(B, 8) - 1, ints(range(pool))
    qs, seq, slots, pos, taken, ids = z(B + 1), z(B), z(cap), z(cap), z(1), z(cap)
    x, p, y = (torch.zeros(cap, d, dtype=td, device="cuda") for _ in range(3))

    def step():
        ctx.page_map(cl, nl, free, pool, table, 8, B, page, pool, qs, seq, slots, pos, cap, taken)
        ctx.embedding(ids, tokens, None, x, 1, cap, V, d, dtype)
        ctx.embedding(pos, places, None, p, 1, cap, longest, d, dtype)
        ctx.eltwise(x, y, cap * d, dtype, residual=p)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    context = [0] * B
    for new in ([9, 1, 20, 3], [1, 1, 1, 1], [1, 0, 17, 1]):
        cl.copy_(ints(context)), nl.copy_(ints(new)), ids.copy_(torch.randint(0, V, (cap,), generator=g, device="cuda"))
        before = table.cpu().numpy()
        graph.replay()
        ctx.check()
        want = ref.page_map(context, new, free.tolist(), before, page, cap)
        assert pos.tolist() == want[4]
        sum64 = tokens.double()[ids.long()] + places.double()[torch.tensor(want[4], device="cuda")]
        half = torch.finfo(td).eps / 2
        assert ((y.double() - sum64).abs() <= (half * (1 + 2.0 ** -23) + 2.0 ** -24) * sum64.abs()).all()
        context = [a + b for a, b in zip(context, new)]
        free.copy_(torch.roll(free, -want[5]))
