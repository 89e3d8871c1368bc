"""The workspace of the paged attention: one that is made for a program's largest call serves its smaller ones."""
import ctypes as C
import itertools
import struct

import pytest

import munet_b200 as mb

F32, BF16 = 0, 2
TOKENS = [1, 2, 3, 8, 9, 10, 36, 37, 72, 73, 74, 256, 4096, 4097, 8192]
REQUESTS = [1, 2, 9, 10, 72, 73, 256, 3500, 3501, 4000, 4096, 16384]


@pytest.fixture
def size():
    """A zeroed block stands in for a context (no device is touched); its SM count is set."""
    ctx = C.create_string_buffer(4096)
    struct.pack_into("ii", ctx, 0, 0, 148)
    lib = mb.lib()
    assert lib.mu_ctx_num_sms(ctx) == 148
    return lambda n, B, Hq, Hkv, D, dtype: lib.mu_attention_paged_workspace_bytes(ctx, n, B, Hq, Hkv, D, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [40, 64, 80, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (16, 16), (16, 2), (80, 1)])
def test_never_shrinks_as_tokens_or_requests_grow(size, Hq, Hkv, D, dtype):
    got = {(n, B): size(n, B, Hq, Hkv, D, dtype) for n in TOKENS for B in REQUESTS}
    assert min(got.values()) > 0
    for (n, B), (m, A) in itertools.product(got, got):
        if n <= m and B <= A:
            assert got[n, B] <= got[m, A], ((n, B), (m, A))
