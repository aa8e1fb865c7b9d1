"""GPU: what the paged-cache ops do at the limits of their arguments -- batches that outgrew their index
vectors, index vectors that are no batch's, workspaces, padding and gradients."""
import ctypes

import numpy as np
import pytest
import torch

import abi_ctypes as abi
from helpers import THETA_LLAMA3, cos_sin_cache, gen, randn
from test_gpu_paged_attention import build_batch, check, reference
from test_gpu_paged_attention_use import _abi_attention, attend, to_dev

pytestmark = pytest.mark.gpu


def i32(dev, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)


# ---- more pages in use than kv_indices has room for ----------------------------------------------

@pytest.mark.parametrize("room", [1, 4, 7, 8, 11])
@pytest.mark.parametrize("fused", [False, True])
def test_append_stays_within_the_pages_that_fit(ops, dev, room, fused):
    """kv_indices is the front of a longer vector that goes on with pages which must not be written.  A
    token whose page did not fit is not appended by the lookup; by slot it still lands in its table's page."""
    page, heads, D = 4, 2, 64
    new, total = [1, 9, 0, 5, 2], [8, 11, 3, 5, 14]                  # 2 + 3 + 1 + 2 + 4 pages
    need = [-(-t // page) for t in total]
    T, M = sum(new), 4
    tables = torch.arange(5 * M, dtype=torch.int32).reshape(5, M).flip(1).to(dev)
    f = ops.kv_cache_ops
    m = f.build_paged_kv_metadata(i32(dev, new), i32(dev, total), tables, page, T, room)
    assert m.kv_indptr.tolist() == np.minimum(np.concatenate([[0], np.cumsum(need)]), room).tolist()
    longer = torch.full((room + 64,), 5 * M, dtype=torch.int32, device=dev)    # page 20 belongs to nobody
    longer[:room] = m.kv_indices
    ix = longer[:room]
    g = gen(room)
    qkv = randn((T, 6 * heads * D), g).to(dev)
    cache = randn((5 * M + 1, 2, page, heads, D), g).to(dev)
    q, k, v = qkv.split([4 * heads * D, heads * D, heads * D], dim=-1)
    table = cos_sin_cache(64, D, THETA_LLAMA3, torch.bfloat16).to(dev)
    if fused:                                                        # what the rotary embedding makes of the keys
        wq, wk = q.clone(), k.clone()
        ops.pos_encoding_ops.rotary_embedding(m.rope_positions, wq, wk, D, table, True)
    else:
        wk = k
    fits, row = [], 0
    want = cache.clone()
    want_slots = cache.clone()
    for r, (n, t) in enumerate(zip(new, total)):
        own = min(max(room - sum(need[:r]), 0), need[r])
        for j in range(n):
            x = t - n + j
            no = int(tables[r, x // page])
            fits.append(no * page + x % page if x // page < own else -1)
            for c in ([want] if fits[-1] >= 0 else []) + [want_slots]:
                c[no, 0, x % page], c[no, 1, x % page] = wk[row].view(heads, D), v[row].view(heads, D)
            row += 1
    assert min(fits) < 0                                             # 12 pages are in use
    got = f.get_kv_slot_mapping(m.batch_indices, m.positions, ix, m.kv_indptr, page)
    assert got.tolist() == fits

    def append(c, slots):
        args = (m.batch_indices, m.positions, c, ix, m.kv_indptr)
        if fused:
            f.rotary_embedding_append_paged_kv(m.rope_positions, q.clone(), k.clone(), v, D, table, True, *args,
                                               slot_mapping=slots)
        else:
            f.append_paged_kv_cache(k, v, *args, slot_mapping=slots)
        return c
    assert torch.equal(append(cache.clone(), None), want)
    assert torch.equal(append(cache.clone(), got), want)
    assert torch.equal(append(cache.clone(), m.slot_mapping), want_slots)
    # heads whose rows are no multiple of 16 bytes: the element-wise kernel
    if not fused:
        small = torch.zeros((5 * M + 1, 2, page, heads, 3), dtype=torch.bfloat16, device=dev)
        part = small.clone()
        k3, v3 = k.view(T, heads, D)[..., :3].contiguous(), v.view(T, heads, D)[..., :3].contiguous()
        f.append_paged_kv_cache(k3, v3, m.batch_indices, m.positions, part, ix, m.kv_indptr)
        for row, s in enumerate(fits):
            if s >= 0:
                small[s // page, 0, s % page], small[s // page, 1, s % page] = k3[row], v3[row]
        assert torch.equal(part, small)


@pytest.mark.parametrize("page", [1, 3, 16])
@pytest.mark.parametrize("fused", [False, True])
def test_append_of_padding_alone_and_among_tokens(ops, dev, page, fused):
    """Tokens without a request, a position or both, by the lookup, at the smallest page too (the page of
    position -1 would be 2^32 - 1 there); a batch of no request at all."""
    heads, D = 2, 64
    f, g = ops.kv_cache_ops, gen(page)
    cache = randn((20, 2, page, heads, D), g).to(dev)
    table = cos_sin_cache(64, D, THETA_LLAMA3, torch.bfloat16).to(dev)
    pages = [3, 7, 5, 11, 2, 0]
    for b, pos, indptr in (([-1] * 5, [-1] * 5, [0]), ([0, -1, 0, 1, -1, 0, 1, 1], [2, 0, -1, 0, -1, 0, -1, 2], [0, 3, 6])):
        n = len(b)
        qkv = randn((n, 4 * heads * D), g).to(dev)
        q, k, v = qkv.split([2 * heads * D, heads * D, heads * D], dim=-1)
        rope = torch.tensor([max(p, 0) for p in pos], device=dev)
        wq, wk = q.clone(), k.clone()
        if fused:
            ops.pos_encoding_ops.rotary_embedding(rope, wq, wk, D, table, True)
        want = cache.clone()
        for i, (r, x) in enumerate(zip(b, pos)):
            if r >= 0 and x >= 0:
                no = pages[indptr[r] + x // page]
                want[no, 0, x % page], want[no, 1, x % page] = wk[i].view(heads, D), v[i].view(heads, D)
        got = cache.clone()
        index = (i32(dev, b), i32(dev, pos), got, i32(dev, pages), i32(dev, indptr))
        if fused:
            f.rotary_embedding_append_paged_kv(rope, q.clone(), k.clone(), v, D, table, True, *index)
        else:
            f.append_paged_kv_cache(k, v, *index)
        assert torch.equal(got, want)
        slots = f.get_kv_slot_mapping(*index[:2], *index[3:], page).tolist()
        assert all((s < 0) == (r < 0 or x < 0) for s, r, x in zip(slots, b, pos))


# ---- index vectors that are no batch's --------------------------------------------------------------

def test_items_that_more_than_one_request_claims(ops, dev):
    """Index vectors that decrease, so that short requests name more tiles (over 100 000) than the item
    search counts in 16 bits, beside one context that is cut and sorted: an item that several requests
    claim is one request's, whole, and nothing in front of or behind `out` is written."""
    T, H, D, N, S = 2048, 16, 64, 256, 300
    qo = ([0, 1] + [500, T, 0, T] * S)[:S + 1]
    kv = [0] + [N] * S
    guard = 64
    big = torch.full((T + 2 * guard, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    q = torch.ones((T, H, D), dtype=torch.bfloat16, device=dev)
    cache = torch.ones((N, 2, 16, 2, D), dtype=torch.bfloat16, device=dev)
    for _ in range(3):
        out = ops.kv_cache_ops.paged_attention(
            q, cache, i32(dev, qo), i32(dev, kv), torch.arange(N, dtype=torch.int32, device=dev),
            torch.full((S,), 16, dtype=torch.int32, device=dev), out=big[guard:guard + T], max_query_len=1)
        torch.cuda.synchronize()
        assert bool((big[:guard] == 7).all()) and bool((big[guard + T:] == 7).all())
        # values are all 1: a row is a mean of ones, 0 (a request without keys) or as it was
        assert bool(((out == 1) | (out == 0) | (out == 7)).all())


# ---- states of cut contexts -------------------------------------------------------------------------

@pytest.mark.parametrize("new,total,heads,kv_heads,hint", [
    # cut decodes in front of, between and behind uncut ones
    ([1] * 40, [3000 if i % 13 == 0 else 30 + i for i in range(40)], 8, 2, 1),
    ([1] * 40, [3000 if i % 13 == 5 else 30 + i for i in range(40)], 8, 2, 0),
    # cut chunks and cut decodes in turn, empty requests
    ([70, 1, 0, 33, 1, 1, 64], [4200, 2900, 0, 90, 5000, 7, 3100], 8, 2, 0),
    # the same above 512 requests, where a kernel plans the launch
    ([1] * 600, [2500 if i % 97 == 0 else 1 + i % 50 for i in range(600)], 4, 2, 1),
    ([1] * 300 + [50] + [1] * 300 + [41], [1 + i % 50 for i in range(300)] + [3500] + [2100] + [9] * 299 + [2600], 8, 2, 0),
])
def test_states_of_cut_contexts_among_uncut_ones(ops, dev, new, total, heads, kv_heads, hint):
    """Only cut requests have states, and they fit the workspace asked for."""
    b = build_batch(50, 16, new, total, heads, kv_heads, 64, torch.bfloat16)
    d, lib = to_dev(b, dev), abi.load()
    need = lib.sarathi_paged_attention_workspace_bytes
    need.restype = ctypes.c_int64
    bytes_ = need(abi.i64(sum(new)), abi.i64(len(new)), abi.i64(d["kv_indices"].numel()), abi.ci(heads), abi.ci(kv_heads),
                  abi.ci(64), abi.ci(16), abi.i64(hint))
    assert bytes_ > 0
    guard = 1 << 20
    ws = torch.full((bytes_ + 2 * guard,), 77, dtype=torch.uint8, device=dev)
    out = torch.empty_like(d["query"])
    abi.check(lib, _abi_attention(lib, d, out, abi.vp(ws.data_ptr() + guard), bytes_, 64 ** -0.5, hint))
    check(b, out, None, reference(b))
    assert bool((ws[:guard] == 77).all()) and bool((ws[guard + bytes_:] == 77).all())
    # and through the front end, twice: nothing depends on the order of workgroups
    for _ in range(2):
        assert torch.equal(attend(ops, d, max_query_len=hint), out)


# ---- gradients --------------------------------------------------------------------------------------

def test_inputs_that_require_a_gradient_are_refused(ops, dev):
    """Nothing is differentiated here, and results without a graph would drop the gradient in silence."""
    b = build_batch(51, 16, [3, 1], [40, 9], 4, 2, 64, torch.bfloat16, poison=False)
    d = to_dev(b, dev)
    f, merge = ops.kv_cache_ops.paged_attention, ops.kv_cache_ops.merge_attention_states
    index = (d["qo_indptr"], d["kv_indptr"], d["kv_indices"], d["last"])
    want, lse = attend(ops, d, return_lse=True)
    kc, vc = d["cache"][:, 0].contiguous(), d["cache"][:, 1].contiguous()
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    for args, kw, name in (((grad(d["query"]), d["cache"]), {}, "query"), ((d["query"], grad(d["cache"])), {}, "paged_kv_cache"),
                           ((d["query"], (grad(kc), vc)), {}, "k_cache"), ((d["query"], (kc, grad(vc))), {}, "v_cache"),
                           ((d["query"], d["cache"]), dict(out=grad(want)), "out")):
        with pytest.raises(RuntimeError, match=name + " requires a gradient"):
            f(*args, *index, **kw)
        with torch.no_grad():
            assert torch.equal(f(*args, *index, **kw), want)
        with torch.inference_mode():
            if "out" not in kw:
                assert torch.equal(f(*args, *index, **kw), want)
    # a value that was computed from a parameter, not a leaf
    with pytest.raises(RuntimeError, match="query requires a gradient"):
        f(grad(d["query"]) * 1.0, d["cache"], *index)
    v, z = torch.stack((want, want)), torch.stack((lse, lse))
    for args, name in (((grad(v), z), "v"), ((v, grad(z)), "lse")):
        with pytest.raises(RuntimeError, match=name + " requires a gradient"):
            merge(*args)
        with torch.no_grad():
            assert torch.equal(merge(*args)[0], want)


# ---- rows of no request -------------------------------------------------------------------------------

def dirty(dev, *shapes):
    """Leaves NaN in the memory that the next tensors of these shapes are made of."""
    held = [torch.full(s, float("nan"), dtype=t, device=dev) for s, t in shapes]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("front,behind", [(0, 5), (3, 0), (2, 300)])
@pytest.mark.parametrize("new,total,heads,kv_heads,head_size,hint", [
    ([1] * 5, [40, 3000, 1, 77, 300], 8, 2, 128, 1),                    # few rows, a cut context
    ([70, 1, 9], [70, 500, 2000], 8, 1, 64, 0),                         # chunks beside single tokens
    ([40, 2], [40, 90], 4, 2, 256, 0),
    ([3, 1], [30, 9], 5, 1, 20, 0),                                     # the plain kernel
    ([1] * 600, [1 + i % 40 for i in range(600)], 4, 2, 64, 1),         # planned
    ([0, 0], [9, 0], 4, 2, 64, 0),                                      # requests without a new token
])
def test_rows_of_no_request_are_defined(ops, dev, front, behind, new, total, heads, kv_heads, head_size, hint):
    """New outputs hold 0 and -inf in front of and behind the requests, whatever the queries there hold;
    an output that was passed in is left alone there, and the new lse beside it is -inf."""
    b = build_batch(52, 16, new, total, heads, kv_heads, head_size, torch.bfloat16)
    d = to_dev(b, dev)
    n = sum(new)
    T = front + n + behind
    q = torch.full((T, heads, head_size), float("nan"), dtype=torch.bfloat16, device=dev)
    q[front:front + n] = d["query"]
    index = (d["qo_indptr"] + front, d["kv_indptr"], d["kv_indices"], d["last"])
    f, want = ops.kv_cache_ops.paged_attention, reference(b)
    outside = torch.ones(T, dtype=torch.bool, device=dev)
    outside[front:front + n] = False
    for flat in (False, True):
        dirty(dev, (q.shape, q.dtype), (q.shape[:2], torch.float32))
        out, lse = f(q.flatten(1) if flat else q, d["cache"], *index, max_query_len=hint, return_lse=True)
        assert bool((out[outside] == 0).all()) and bool((lse[outside] == -torch.inf).all())
        check(b, out[front:front + n], lse[front:front + n], want)
        dirty(dev, (q.shape, q.dtype))
        only = f(q, d["cache"], *index, max_query_len=hint)
        assert torch.equal(only.view_as(out), out)
    given = torch.full((T, heads + 1, head_size), 3.0, dtype=torch.bfloat16, device=dev)
    dirty(dev, (q.shape[:2], torch.float32))
    res, lse2 = f(q, d["cache"], *index, max_query_len=hint, return_lse=True, out=given[:, :heads])
    assert bool((given[outside] == 3).all()) and bool((given[:, heads] == 3).all())
    assert torch.equal(res[~outside], out.view_as(q)[~outside]) and torch.equal(lse2, lse)


def test_rows_without_any_request(ops, dev):
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    cache = torch.zeros((2, 2, 16, 2, 64), dtype=torch.float16, device=dev)
    q = torch.full((37, 6, 64), float("nan"), dtype=torch.float16, device=dev)
    dirty(dev, (q.shape, q.dtype), (q.shape[:2], torch.float32))
    out, lse = ops.kv_cache_ops.paged_attention(q, cache, zero, zero, none, none, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -torch.inf).all())
    given = torch.full_like(q, 3.0)
    ops.kv_cache_ops.paged_attention(q, cache, zero, zero, none, none, out=given)
    assert bool((given == 3).all())


def test_a_captured_padded_step_returns_defined_rows(ops, dev):
    """Metadata and attention into new outputs, captured once: at every replay the rows behind the batch are
    0 and -inf, whatever the replay before left in them."""
    import sarathi_amd.layers as layers
    heads, kv_heads, D, page, R, M = 8, 2, 64, 16, 6, 40
    g = gen(53)
    cache = randn((R * M, 2, page, kv_heads, D), g).to(dev)
    tables = torch.randperm(R * M, generator=g).to(torch.int32).reshape(R, M).to(dev)
    query_lens, seq_lens = (torch.zeros(R, dtype=torch.int32, device=dev) for _ in range(2))
    q = torch.full((R, heads, D), float("nan"), dtype=torch.bfloat16, device=dev)

    def step():
        meta = layers.build_append_metadata_on_device(query_lens, seq_lens, tables, page, R, max_query_len=1)
        return meta.attention(q, cache, return_lse=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = step()
    for lens in ([600, 1, 16, 17, 300, 64], [5, 400], [], [640, 2, 1]):
        n = len(lens)
        query_lens.copy_(torch.tensor([1] * n + [0] * (R - n), dtype=torch.int32))
        seq_lens.copy_(torch.tensor(lens + [0] * (R - n), dtype=torch.int32))
        q[:n] = randn((n, heads, D), g).to(dev)
        graph.replay()
        torch.cuda.synchronize()
        got, z = out.clone(), lse.clone()
        assert bool((got[n:] == 0).all()) and bool((z[n:] == -torch.inf).all())
        assert bool(got[:n].isfinite().all()) and bool(z[:n].isfinite().all())
        eager, eager_z = step()
        torch.cuda.synchronize()
        assert torch.equal(eager, got) and torch.equal(eager_z, z)
