"""Sizes and refusals of the paged-cache ops that need no GPU."""
import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "sarathi-serve_amd", "sarathi_amd", "lib", "libsarathi_ops_hip.so")
i64, ci = ctypes.c_int64, ctypes.c_int


@pytest.fixture(scope="module")
def workspace():
    import sarathi_amd  # noqa: F401  loads torch first
    f = ctypes.CDLL(LIB).sarathi_paged_attention_workspace_bytes
    f.restype = i64
    return lambda T, R, NI, h, hk, d, page, q: f(i64(T), i64(R), i64(NI), ci(h), ci(hk), ci(d), ci(page), i64(q))


@pytest.mark.parametrize("h,hk,d", [(32, 8, 128), (32, 32, 128), (64, 64, 128), (64, 8, 128), (71, 1, 64), (12, 4, 256)])
@pytest.mark.parametrize("hint", [0, 1])
def test_workspace_does_not_grow_with_requests_that_are_not_cut(workspace, h, hk, d, hint):
    """Every cut adds parts, of which there are at most four times what fills the GPU (two workgroups per
    compute unit, shared by the key heads, 256 units), and cuts no more tiles than it adds parts.  So the
    states take at most 2 * 4 * 512 tiles of 64 rows of d + 2 floats and the chunks' at most 2 * 512 of 128
    rows, whatever the number of requests; their maps and the plan take 16 bytes a request."""
    states = (2 * 4 * 512 * 64 + 2 * 512 * 128) * (d + 2) * 4
    if hint == 1:      # tiles of 16, 32 or 64 rows, by the query heads per key head; no chunks
        states = 2 * 4 * 512 * (16 if h // hk <= 16 else 64) * (d + 2) * 4
    for R in (1, 16, 300, 600, 4096, 8192, 65536):
        size = workspace(R, R, 64 * R, h, hk, d, 16, hint)
        assert 0 < size <= states + 16 * R + 8192, (R, size)


def test_fill_of_rows_of_no_request():
    import sarathi_amd  # noqa: F401
    f = ctypes.CDLL(LIB).sarathi_paged_attention_fill
    vp, cf = ctypes.c_void_p, ctypes.c_float
    p = ctypes.cast(ctypes.create_string_buffer(4096), vp)

    def call(fill, T=1, R=1, out=p, lse=None):
        return f(p, p, p, out, vp(lse), p, p, p, p, i64(T), i64(R), i64(1), i64(1), ci(4), ci(2), ci(16), ci(16), i64(64),
                 i64(64), i64(1024), i64(32), cf(1.0), ci(1), i64(-1), i64(0), vp(None), i64(0), ci(2), ci(fill), vp(None))
    assert call(-1) == -1 and call(4) == -1
    assert call(3, T=0) == 0 and call(0, R=0) == 0 and call(1, R=0) == 0      # no lse: nothing to fill
    assert call(2, R=0, out=vp(None)) == -1


@pytest.mark.parametrize("T,R,NI,page,h,hk,hint", [
    (11620506, 11, 13441971, 339304936, 4, 1, 1), (38834252, 1, 10796720, 68632828, 8, 8, 1),
    (23899935, 151737, 38281589, 8492708, 32, 8, 1), (1787488, 8505, 2522992, 1835743780, 8, 1, 1),
    (2762704, 779143, 325257681, 148975915, 1, 1, 0), (1, 1, (1 << 31) - 2, (1 << 31) - 1, 8, 1, 1),
    (1 << 29, 1, (1 << 31) - 2, (1 << 31) - 1, 1, 1, 0),
])
def test_workspace_of_the_largest_pages(workspace, T, R, NI, page, h, hk, hint):
    """Sizes whose products pass 64 bits: the workspace stays the states of what fills the GPU a few times,
    at most 4096 tiles of 64 rows and 1024 of 128, with 16 bytes a request."""
    assert 0 < workspace(T, R, NI, h, hk, 128, page, hint) <= (4096 * 64 + 1024 * 128) * 130 * 4 + 16 * R + 8192
