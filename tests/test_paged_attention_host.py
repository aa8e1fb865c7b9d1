"""Refusals of the paged-attention ops and of the device-side metadata, before any GPU work: through
the C ABI with host pointers (nothing is launched) and through the front end with CPU tensors."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "sarathi-serve_amd", "sarathi_amd", "lib", "libsarathi_ops_hip.so")
INVALID, UNSUPPORTED, OK = -1, -2, 0
i64, ci, cf, vp = ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    import sarathi_amd  # noqa: F401  loads torch first
    return ctypes.CDLL(LIB)


@pytest.fixture(scope="module")
def p():
    return ctypes.cast(ctypes.create_string_buffer(4096), vp)


def test_paged_attention_arguments(lib, p):
    def call(**k):
        g = k.get
        return lib.sarathi_paged_attention(
            g("q", p), g("kc", p), g("vc", p), g("out", p), vp(None), g("qo", p), g("kv", p), g("ix", p),
            g("last", p), i64(g("T", 1)), i64(g("R", 1)), i64(g("NI", 1)), i64(g("pages", 1)), ci(g("h", 4)),
            ci(g("hk", 2)), ci(g("d", 16)), ci(g("page", 16)), i64(g("qs", 64)), i64(g("os", 64)),
            i64(g("ps", 1024)), i64(g("es", 32)), cf(g("scale", 1.0)), ci(1), i64(-1), i64(0), vp(None), i64(0),
            ci(g("dt", 2)), vp(None))
    null = vp(None)
    assert call(T=0) == OK and call(R=0) == OK
    assert call(T=0, q=null, out=null) == OK
    for bad in (dict(q=null), dict(out=null), dict(qo=null), dict(kv=null), dict(last=null), dict(ix=null),
                dict(kc=null), dict(vc=null), dict(T=-1), dict(R=-1), dict(NI=-1), dict(pages=-1), dict(h=0),
                dict(hk=0), dict(h=3), dict(d=0), dict(page=0), dict(T=2, qs=63), dict(T=2, os=63),
                dict(es=31), dict(ps=-1), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=3e38)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(dt=0), dict(dt=7), dict(d=257, es=2 * 257, qs=4 * 257, os=4 * 257),
                dict(T=1 << 29), dict(NI=1 << 31), dict(R=1 << 30)):
        assert call(**bad) == UNSUPPORTED, bad


def test_paged_attention_workspace(lib):
    f = lib.sarathi_paged_attention_workspace_bytes
    f.restype = i64
    size = lambda T, R, NI, h=32, hk=8, d=128, page=16, q=0: f(  # noqa: E731
        i64(T), i64(R), i64(NI), ci(h), ci(hk), ci(d), ci(page), i64(q))
    assert size(1, 1, 4096, q=1) > 0          # a long context of one token is cut
    assert size(1, 1, 4, q=1) == 0            # 64 keys are not
    assert size(0, 1, 16) == 0 and size(1, 0, 16) == 0 and size(1, 1, 0) == 0
    assert size(-1, 1, 16) == 0 and size(1, 1, 16, h=30) == 0 and size(1, 1, 16, d=300) == 0
    # what a serving batch needs stays small beside its cache
    assert size(2304, 257, 70000) < 1 << 30


def test_paged_attention_workspace_of_large_chunks(lib):
    """Chunks that fill the GPU are not cut: no room is asked for their states."""
    f = lib.sarathi_paged_attention_workspace_bytes
    f.restype = i64
    small = f(i64(1 << 14), i64(2), i64(1 << 14), ci(32), ci(8), ci(128), ci(16), i64(0))
    large = f(i64(1 << 17), i64(2), i64(1 << 14), ci(32), ci(8), ci(128), ci(16), i64(0))
    assert 0 < large == small < 1 << 24


def test_metadata_arguments(lib, p):
    def call(**k):
        g = k.get
        return lib.sarathi_build_paged_kv_metadata(
            g("ql", p), p, g("tab", p), g("qo", p), p, g("ix", p), p, g("bi", p), p, p, p, i64(g("R", 1)),
            i64(g("M", 4)), i64(g("ts", 4)), ci(g("page", 16)), i64(g("T", 1)), i64(g("P", 1)), vp(None))
    null = vp(None)
    for bad in (dict(ql=null), dict(tab=null), dict(qo=null), dict(ix=null), dict(bi=null), dict(R=-1), dict(M=-1),
                dict(ts=3), dict(page=0), dict(T=-1), dict(P=-1)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(T=1 << 31), dict(P=1 << 31), dict(R=1 << 31)):
        assert call(**bad) == UNSUPPORTED, bad


def test_merge_arguments(lib, p):
    def call(**k):
        g = k.get
        return lib.sarathi_merge_attention_states(
            g("v", p), g("lse", p), g("out", p), vp(None), i64(g("S", 2)), i64(g("T", 2)), ci(g("H", 2)),
            ci(g("D", 8)), i64(g("vs", 32)), i64(g("vt", 16)), i64(4), i64(g("lt", 2)), i64(g("ot", 16)), i64(2),
            ci(g("dt", 2)), vp(None))
    null = vp(None)
    for bad in (dict(v=null), dict(lse=null), dict(out=null), dict(S=0), dict(T=-1), dict(H=0), dict(D=0), dict(vt=15),
                dict(lt=1), dict(ot=15), dict(vs=-1)):
        assert call(**bad) == INVALID, bad
    assert call(dt=5) == UNSUPPORTED
    assert call(T=0) == OK and call(T=0, v=null, lse=null, out=null) == OK


def test_front_end_refuses_cpu_tensors_and_other_layouts(ops):
    kv = ops.kv_cache_ops
    i = torch.zeros(2, dtype=torch.int32)
    q, cache = torch.zeros((1, 4, 16), dtype=torch.bfloat16), torch.zeros((1, 2, 16, 2, 16), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        kv.paged_attention(q, cache, i, i, i, i[:1])
    with pytest.raises(ValueError, match="NHD"):
        kv.paged_attention(q, cache, i, i, i, i[:1], kv_layout="HND")
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        kv.build_paged_kv_metadata(i, i, i.reshape(2, 1), 16, 4)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        kv.merge_attention_states(torch.zeros((2, 1, 1, 8)), torch.zeros((2, 1, 1)))


def test_names_are_public(ops):
    for name in ("PagedKvMetadata", "build_paged_kv_metadata", "paged_attention", "merge_attention_states"):
        assert name in ops.kv_cache_ops.__all__ and hasattr(ops.kv_cache_ops, name)
    import sarathi_amd.layers as layers
    assert "build_append_metadata_on_device" in layers.__all__
    assert hasattr(layers.AppendMetadata, "attention")
