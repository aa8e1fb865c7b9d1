"""GPU: paged attention, device-built metadata and merged states as a serving program uses them --
chunked prefill against one pass, captured and replayed steps with padding, streams, caches beyond
4 GiB, cut contexts, odd arguments -- and the tokens that the append ops skip."""
import ctypes

import numpy as np
import pytest
import torch

import abi_ctypes as abi
from helpers import THETA_LLAMA3, cos_sin_cache, gen, randn
from test_gpu_paged_attention import build_batch, call, check, reference

pytestmark = pytest.mark.gpu


def to_dev(b, dev):
    d = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in b.items()}
    d["query"] = b["query"].contiguous().to(dev).unflatten(1, (b["heads"], b["head_size"]))
    return d


def attend(ops, d, **kw):
    return ops.kv_cache_ops.paged_attention(d["query"], d["cache"], d["qo_indptr"], d["kv_indptr"], d["kv_indices"],
                                            d["last"], **kw)


# ---- shapes at which the launch changes ---------------------------------------------------------

@pytest.mark.parametrize("new,total,heads,kv_heads,head_size,page,dtype,kw", [
    # contexts cut into parts, few and many tokens, the wide and the narrow join
    ([1], [9000], 8, 2, 128, 16, torch.bfloat16, {}),
    ([1] * 3, [5000, 1, 2600], 6, 1, 64, 16, torch.float16, {}),
    ([1] * 70, [700 + 37 * i for i in range(70)], 2, 1, 128, 16, torch.bfloat16, {}),
    ([2, 4], [3000, 4100], 4, 4, 80, 32, torch.float16, {}),
    ([1], [6001], 71, 1, 64, 16, torch.bfloat16, dict(window_left=2500)),
    ([3], [2049], 20, 1, 256, 16, torch.bfloat16, {}),
    ([1], [2500], 4, 2, 128, 1, torch.float16, {}),
    # a chunk whose few tiles are cut as well
    ([70], [4200], 4, 1, 128, 16, torch.bfloat16, {}),
    ([33, 1, 40], [2100, 900, 3000], 8, 1, 64, 16, torch.float16, dict(window_left=1500)),
    # large tiles: ragged, windows inside a chunk, pages that are no multiple of 16
    ([1100, 1, 900, 1], [1100, 300, 1500, 17], 16, 16, 64, 16, torch.bfloat16, {}),
    ([700], [1700], 32, 16, 128, 16, torch.bfloat16, dict(window_left=130)),
    ([513], [600], 64, 8, 128, 24, torch.float16, {}),
    ([400, 0, 1], [450, 12, 77], 48, 8, 96, 16, torch.bfloat16, dict(causal=False)),
    # a head size between those of the tiles
    ([150, 1], [260, 700], 6, 2, 192, 16, torch.bfloat16, {}),
    # query heads per key head above 16 and above 64
    ([1, 9, 1], [300, 200, 2], 34, 2, 128, 16, torch.bfloat16, {}),
    ([5, 1], [50, 1030], 65, 1, 128, 16, torch.float16, {}),
])
@pytest.mark.parametrize("hint", [False, True])
def test_every_launch_form(ops, dev, new, total, heads, kv_heads, head_size, page, dtype, kw, hint):
    b = build_batch(3, page, new, total, heads, kv_heads, head_size, dtype)
    got, lse = call(ops, dev, b, return_lse=True, max_query_len=max(new) if hint else None, **kw)
    check(b, got, lse, reference(b, kw.get("causal", True), kw.get("window_left", -1)))
    again = call(ops, dev, b, max_query_len=max(new) if hint else None, **kw)
    assert torch.equal(again, got)               # no result depends on the order of workgroups


def test_many_requests(ops, dev):
    """More requests than a workgroup has threads, with empty ones among them."""
    rng = np.random.default_rng(5)
    new = [int(v) for v in rng.choice([0, 1, 1, 1, 2, 6], 1300)]
    total = [n + int(rng.integers(0, 60)) if n else int(rng.integers(0, 60)) for n in new]
    b = build_batch(4, 16, new, total, 4, 2, 64, torch.bfloat16)
    want = reference(b)
    for hint in (None, 6):
        got, lse = call(ops, dev, b, return_lse=True, max_query_len=hint)
        check(b, got, lse, want)


def test_a_wrong_upper_bound_costs_time_only(ops, dev):
    b = build_batch(8, 16, [40, 1, 300], [64, 2000, 300], 8, 2, 128, torch.bfloat16)
    got, lse = call(ops, dev, b, return_lse=True, max_query_len=1)
    check(b, got, lse, reference(b))


def test_scale_and_large_scores(ops, dev):
    """Scores far from zero and scales other than the default: the running maximum moves."""
    b = build_batch(9, 16, [30, 1], [200, 900], 4, 2, 128, torch.bfloat16)
    k = b["cache"][:, 0]
    b["cache"][:, 0] = torch.where(k.isnan(), k, k * 6)
    for scale in (0.4, 1e-3):
        got, lse = call(ops, dev, b, return_lse=True, sm_scale=scale)
        check(b, got, lse, reference(b, scale=scale))


def test_scores_that_grow_along_the_context(ops, dev):
    """Every block of keys raises the maximum, by more and by less than the threshold of rescaling."""
    D = 64
    for step in (0.02, 0.6):
        b = build_batch(10, 16, [20, 1], [400, 1200], 2, 1, D, torch.float16)
        q = b["query"]
        q.zero_()
        q[:, 0::D] = 1.0
        for r, t in enumerate(b["total"]):
            pages = b["kv_indices"][b["kv_indptr"][r]:b["kv_indptr"][r + 1]].long()
            ramp = torch.zeros(len(pages) * 16)
            ramp[:t] = torch.arange(t, dtype=torch.float32) * step
            b["cache"][pages, 0, :, 0, 0] = ramp.reshape(-1, 16).half()
        got, lse = call(ops, dev, b, return_lse=True, sm_scale=1.0)
        check(b, got, lse, reference(b, scale=1.0))


def test_infinite_scores_stay_in_their_rows(ops, dev):
    """A key of -inf is never chosen; a NaN query poisons its own rows only."""
    b = build_batch(12, 16, [20, 1, 1], [150, 40, 700], 4, 2, 64, torch.bfloat16)
    page = int(b["kv_indices"][b["kv_indptr"][2]])
    b["cache"][page, 0, 3] = 0.0
    b["cache"][page, 0, 3, :, 0] = float("-inf")
    b["query"].view(22, 4, 64)[21, :, 0] = 1.0
    b["query"].view(22, 4, 64)[5, 2] = float("nan")
    got, lse = call(ops, dev, b, return_lse=True)
    got, lse = got.cpu(), lse.cpu()
    assert bool(got[5, 2].isnan().all()) and bool(lse[5, 2].isnan())
    b["query"].view(22, 4, 64)[5, 2] = 0.0
    clean, clean_lse = call(ops, dev, b, return_lse=True)
    out, z, mag = reference(b)
    ok = torch.ones((22, 4), dtype=torch.bool)
    ok[5, 2] = False
    assert torch.equal(got[ok], clean.cpu()[ok]) and torch.equal(lse[ok], clean_lse.cpu()[ok])
    check(b, clean, clean_lse, (out, z, mag))


# ---- tensors ------------------------------------------------------------------------------------

def test_strides_pairs_and_out(ops, dev):
    b = build_batch(13, 16, [19, 1, 1], [100, 31, 257], 8, 2, 128, torch.bfloat16)
    d = to_dev(b, dev)
    want = attend(ops, d)
    check(b, want, None, reference(b))
    # a (K, V) pair of separate tensors; 2-D query rows; a strided out
    kc, vc = d["cache"][:, 0].contiguous(), d["cache"][:, 1].contiguous()
    args = (d["qo_indptr"], d["kv_indptr"], d["kv_indices"], d["last"])
    f = ops.kv_cache_ops.paged_attention
    assert torch.equal(f(d["query"], (kc, vc), *args), want)
    flat = f(d["query"].flatten(1), d["cache"], *args)
    assert flat.shape == (21, 8 * 128) and torch.equal(flat.view_as(want), want)
    wide = torch.full((21, 9 * 128), 7.0, dtype=torch.bfloat16, device=dev)
    res = f(d["query"], d["cache"], *args, out=wide[:, :8 * 128].unflatten(1, (8, 128)))
    assert res.data_ptr() == wide.data_ptr() and torch.equal(res, want) and bool((wide[:, 8 * 128:] == 7).all())
    # one layer of a cache that holds several: entries far apart
    layers = torch.zeros((d["cache"].shape[0], 2, 16, 3, 2, 128), dtype=torch.bfloat16, device=dev)
    layers[:, :, :, 1] = d["cache"]
    assert torch.equal(f(d["query"], layers[:, :, :, 1], *args), want)
    # rows that are no multiple of 16 bytes apart, and unaligned ones: the plain kernel
    for pad, shift in ((4, 0), (8, 1)):
        rows = torch.zeros((21, 8 * 128 + pad), dtype=torch.bfloat16, device=dev)
        rows[:, shift:shift + 8 * 128] = d["query"].flatten(1)
        odd = f(rows[:, shift:shift + 8 * 128], d["cache"], *args)
        check(b, odd, None, reference(b))
    # no request, no token
    empty = torch.zeros(1, dtype=torch.int32, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    out, lse = f(d["query"][:0], d["cache"], empty, empty, none, none, return_lse=True)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)


def test_rows_behind_the_last_request_are_left_alone(ops, dev):
    for new, total in (([9, 1], [30, 2000]), ([200, 1], [260, 90])):
        b = build_batch(14, 16, new, total, 8, 2, 64, torch.float16)
        d = to_dev(b, dev)
        n = sum(new)
        q = torch.cat((d["query"], torch.full((5, 8, 64), float("nan"), dtype=torch.float16, device=dev)))
        out = torch.full_like(q, 3.0)
        ops.kv_cache_ops.paged_attention(q, d["cache"], d["qo_indptr"], d["kv_indptr"], d["kv_indices"], d["last"], out=out)
        assert bool((out[n:] == 3.0).all())
        check(b, out[:n], None, reference(b))


def test_index_vectors_past_their_tensors_touch_nothing(ops, dev):
    """Whatever the index vectors say, reads stay inside the tensors; requests with sound ones get
    their results."""
    b = build_batch(15, 16, [3, 1, 40, 1], [40, 33, 90, 50], 4, 2, 64, torch.bfloat16, poison=False)
    d = to_dev(b, dev)
    bad = d["kv_indices"].clone()
    p0, p1 = int(b["kv_indptr"][1]), int(b["kv_indptr"][2])
    bad[p0] = 1 << 30
    bad[p1 - 1] = -7
    good = attend(ops, d)
    d["kv_indices"] = bad
    got = attend(ops, d)
    rows = torch.ones(45, dtype=torch.bool, device=dev)
    rows[3] = False
    assert torch.equal(got[rows], good[rows])
    # more tokens and more pages than there are, and lengths out of range
    d = to_dev(b, dev)
    d["qo_indptr"] = torch.tensor([0, 3, 4, 44, 4000], dtype=torch.int32, device=dev)
    d["kv_indptr"] = torch.tensor([0, 3, 6, 12, 90000], dtype=torch.int32, device=dev)
    d["last"] = torch.tensor([8, 1, 10, 1 << 20], dtype=torch.int32, device=dev)
    got = attend(ops, d)
    torch.cuda.synchronize()
    assert torch.equal(got[:44], good[:44])


def test_cache_beyond_four_gib(ops, dev):
    """Pages whose byte offsets pass 32 bits, from both ends of a 6 GiB cache."""
    pages, page, hk, D = 98304, 16, 8, 128
    cache = torch.zeros((pages, 2, page, hk, D), dtype=torch.bfloat16, device=dev)
    assert cache.nbytes > 6e9
    small = build_batch(16, page, [20, 1], [70, 900], 32, hk, D, torch.bfloat16, poison=False)
    n = small["kv_indices"].numel()
    far = torch.cat((torch.arange(pages - n + n // 2, pages), torch.arange(n // 2))).to(torch.int32)
    cache[far.long().to(dev)] = small["cache"][small["kv_indices"].long()].to(dev)
    d = to_dev(small, dev)
    want = attend(ops, d)
    d["cache"], d["kv_indices"] = cache, far.to(dev)
    assert torch.equal(attend(ops, d), want)


def test_refusals(ops, dev):
    b = build_batch(17, 16, [2], [20], 4, 2, 64, torch.bfloat16)
    d = to_dev(b, dev)
    f = ops.kv_cache_ops.paged_attention
    a = [d["query"], d["cache"], d["qo_indptr"], d["kv_indptr"], d["kv_indices"], d["last"]]

    def refused(match, **change):
        names = ["query", "cache", "qo", "kv", "ix", "last"]
        args = [change.pop(n, v) for n, v in zip(names, a)]
        with pytest.raises(RuntimeError, match=match):
            f(*args, **change)

    refused("bfloat16 and float16", query=d["query"].float(), cache=d["cache"].float())
    refused("share a dtype", cache=d["cache"].half())
    refused("multiple of the cache's", query=d["query"][:, :3])
    refused("int32 vector", qo=d["qo_indptr"].long())
    refused("expected qo_indptr", qo=d["qo_indptr"][:1])
    refused("must be \\[num_pages, 2", cache=d["cache"][:, 0])
    refused("contiguous", cache=d["cache"].transpose(3, 4).contiguous().transpose(3, 4))
    refused("at most 256", query=torch.zeros((2, 4, 512), dtype=torch.bfloat16, device=dev),
            cache=torch.zeros((2, 2, 16, 2, 512), dtype=torch.bfloat16, device=dev))
    refused("dtype and shape", out=torch.zeros((3, 4, 64), dtype=torch.bfloat16, device=dev))
    refused("must not be negative", max_query_len=-1)
    for scale in (0.0, -0.3, float("nan"), float("inf"), 1e300):
        refused("positive and finite", sm_scale=scale)
    refused("must not overlap", query=d["query"][:1].expand(2, 4, 64))
    m = ops.kv_cache_ops.merge_attention_states
    v, z = torch.zeros((2, 3, 4, 8), device=dev), torch.zeros((2, 3, 4), device=dev)
    for bad_v, bad_z, match in ((v[0], z, "expected v"), (v, z[:1], "expected v"), (v, z.half(), "float32"),
                                (v.transpose(2, 3).contiguous().transpose(2, 3), z, "contiguous"),
                                (v[:0], z[:0], "there must be")):
        with pytest.raises(RuntimeError, match=match):
            m(bad_v, bad_z)
    i = torch.ones(3, dtype=torch.int32, device=dev)
    t = torch.zeros((3, 4), dtype=torch.int32, device=dev)
    g = ops.kv_cache_ops.build_paged_kv_metadata
    for args, kw, match in (((i, i[:2], t, 16), {}, "one length"), ((i, i, t[:2], 16), {}, "block_tables"),
                            ((i, i, t.long(), 16), {}, "block_tables"), ((i, i, t, 0), {}, "page_size"),
                            ((i.long(), i, t, 16), {}, "int32"), ((i, i, t, 16), dict(num_tokens=-1), "negative"),
                            ((i, i, t.t().contiguous().t(), 16), {}, "contiguous rows")):
        with pytest.raises(RuntimeError, match=match):
            g(*args, **{"num_tokens": 3, **kw})


# ---- the C ABI ----------------------------------------------------------------------------------

def _abi_attention(lib, d, out, ws, ws_bytes, scale, hint=0):
    q, c = d["query"], d["cache"]
    return lib.sarathi_paged_attention(
        abi.ptr(q), abi.ptr(c), abi.vp(c.data_ptr() + c.stride(1) * 2), abi.ptr(out), abi.vp(None),
        abi.ptr(d["qo_indptr"]), abi.ptr(d["kv_indptr"]), abi.ptr(d["kv_indices"]), abi.ptr(d["last"]),
        abi.i64(q.shape[0]), abi.i64(d["last"].numel()), abi.i64(d["kv_indices"].numel()), abi.i64(c.shape[0]),
        abi.ci(q.shape[1]), abi.ci(c.shape[3]), abi.ci(c.shape[4]), abi.ci(c.shape[2]), abi.i64(q.stride(0)),
        abi.i64(out.stride(0)), abi.i64(c.stride(0)), abi.i64(c.stride(2)), abi.cf(scale), abi.ci(1), abi.i64(-1),
        abi.i64(hint), ws, abi.i64(ws_bytes), abi.ci(abi.DT[q.dtype]), abi.stream())


def test_without_a_workspace_nothing_is_cut(ops, dev):
    lib = abi.load()
    for new, total in (([1, 1], [5000, 700]), ([50, 1], [3000, 40])):
        b = build_batch(18, 16, new, total, 4, 1, 128, torch.bfloat16)
        d = to_dev(b, dev)
        want = reference(b)
        need = lib.sarathi_paged_attention_workspace_bytes
        need.restype = ctypes.c_int64
        bytes_ = need(abi.i64(sum(new)), abi.i64(2), abi.i64(d["kv_indices"].numel()), abi.ci(4), abi.ci(1), abi.ci(128),
                      abi.ci(16), abi.i64(0))
        assert bytes_ > 0
        ws = torch.full((bytes_,), 255, dtype=torch.uint8, device=dev)    # contents do not matter
        for p, n in ((abi.ptr(ws), bytes_), (abi.vp(None), 0), (abi.ptr(ws), bytes_ - 1)):
            out = torch.empty_like(d["query"])
            abi.check(lib, _abi_attention(lib, d, out, p, n, 128 ** -0.5))
            check(b, out, None, want)


# ---- as a serving program runs them ---------------------------------------------------------------

def _model_step(ops, dev, meta, qkv, positions, cache, cos_sin, heads, kv_heads, D):
    q, k, v = qkv.split([heads * D, kv_heads * D, kv_heads * D], dim=-1)
    meta.rotary_embedding_append(positions, q, k, v, D, cos_sin, True, cache)
    return meta.attention(q, cache).unflatten(1, (heads, D))


@pytest.mark.parametrize("on_device", [False, True])
def test_chunked_prefill_and_decodes_match_one_pass(ops, dev, on_device):
    """A prompt processed in chunks beside decode steps of another request: the cache ends up with the
    bits of one pass, and attention agrees with the definition over what the cache holds."""
    import sarathi_amd.layers as layers
    heads, kv_heads, D, page = 8, 2, 128, 16
    g = gen(21)
    prompt, other = 300, 40
    width = (heads + 2 * kv_heads) * D
    rows = randn((prompt, width), g).to(dev)
    other_rows = randn((other + 8, width), g).to(dev)
    cos_sin = cos_sin_cache(4096, D, THETA_LLAMA3, torch.bfloat16).to(dev)
    tables = torch.randperm(40, generator=g).to(torch.int32)[:2 * 20].reshape(2, 20)
    tab_dev = tables.to(dev)

    def step(cache, reqs):
        """reqs: (row of the table, rows of qkv, tokens in all afterwards)"""
        new, total = [r[1].shape[0] for r in reqs], [r[2] for r in reqs]
        if on_device:
            meta = layers.build_append_metadata_on_device(
                torch.tensor(new, dtype=torch.int32, device=dev), torch.tensor(total, dtype=torch.int32, device=dev),
                tab_dev[[r[0] for r in reqs]].contiguous(), page, sum(new), max_query_len=max(new))
            positions = meta.rope_positions
        else:
            meta = layers.build_append_metadata(
                [layers.SequenceSlice(True, n, t, tables[r[0]].tolist()) for n, t, r in zip(new, total, reqs)], page, dev)
            positions = meta.append_positions.long()
        return _model_step(ops, dev, meta, torch.cat([r[1].clone() for r in reqs]), positions, cache, cos_sin, heads,
                           kv_heads, D)

    whole = torch.zeros((40, 2, page, kv_heads, D), dtype=torch.bfloat16, device=dev)
    want = step(whole, [(0, rows, prompt)])
    step(whole, [(1, other_rows[:other], other)])
    want_other = torch.cat([step(whole, [(1, other_rows[other + i:other + i + 1], other + i + 1)]) for i in range(8)])

    cache = torch.zeros_like(whole)
    step(cache, [(1, other_rows[:other], other)])
    got, got_other, at = [], [], 0
    for i, n in enumerate([100, 1, 37, 64, 5, 60, 30, 3]):
        o = step(cache, [(0, rows[at:at + n], at + n), (1, other_rows[other + i:other + i + 1], other + i + 1)])
        got.append(o[:n])
        got_other.append(o[n:])
        at += n
    assert at == prompt
    assert torch.equal(cache, whole)
    # both are within the rounding of the same sums; two roundings of half a step each way
    half = torch.finfo(torch.bfloat16).eps / 2
    for a, b in ((torch.cat(got), want), (torch.cat(got_other), want_other)):
        a, b = a.float(), b.float()
        assert bool(((a - b).abs() <= 2 * half * b.abs() + 2 * half * 4.0).all())   # |v| <= 4 nearly everywhere
        assert (a - b).abs().mean().item() < half


def test_shared_prefix_joins_with_suffixes(ops, dev):
    """One prefix for all requests: non-causal attention of all tokens over it as ONE request, causal
    attention over the suffixes, joined; against attention over the whole contexts."""
    heads, kv_heads, D, page = 8, 2, 128, 16
    prefix, suffix, new = 320, [5, 33, 17, 1], [1, 1, 3, 1]
    b = build_batch(22, page, new, [prefix + s for s in suffix], heads, kv_heads, D, torch.bfloat16, poison=False)
    first = b["kv_indices"][:prefix // page]
    for r in range(1, 4):          # the same prefix under other page numbers
        at = int(b["kv_indptr"][r])
        b["cache"][b["kv_indices"][at:at + prefix // page].long()] = b["cache"][first.long()]
    want = reference(b)
    d = to_dev(b, dev)
    T = sum(new)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    f = ops.kv_cache_ops.paged_attention
    states = torch.empty((2, T, heads, D), dtype=torch.bfloat16, device=dev)
    lses = torch.empty((2, T, heads), dtype=torch.float32, device=dev)
    _, lses[0] = f(d["query"], d["cache"], i32([0, T]), i32([0, prefix // page]), first.to(dev), i32([page]),
                   causal=False, out=states[0], return_lse=True)
    ix = torch.cat([b["kv_indices"][int(b["kv_indptr"][r]) + prefix // page:int(b["kv_indptr"][r + 1])] for r in range(4)])
    kv = np.concatenate([[0], np.cumsum([(s + page - 1) // page for s in suffix])])
    _, lses[1] = f(d["query"], d["cache"], d["qo_indptr"], i32(kv.tolist()), ix.to(dev),
                   i32([(s - 1) % page + 1 for s in suffix]), out=states[1], return_lse=True)
    out, z = ops.kv_cache_ops.merge_attention_states(states, lses)
    half = torch.finfo(torch.bfloat16).eps / 2
    ref, ref_z, mag = want
    # each state is rounded to the dtype once more than in one pass
    assert bool(((out.cpu().double() - ref).abs() <= half * (2 * mag + ref.abs()) + 1e-4 * mag).all())
    assert bool(((z.cpu().double() - ref_z).abs() <= 2e-6 * ref_z.abs() + 1e-5).all())


def test_captured_step_follows_lengths_and_padding(ops, dev):
    """Metadata, append and attention of a padded decode batch captured once, replayed on other lengths
    (with eager work in between); padding tokens write nothing."""
    import sarathi_amd.layers as layers
    heads, kv_heads, D, page, R, M = 8, 2, 128, 16, 6, 64
    g = gen(23)
    cache = randn((R * M, 2, page, kv_heads, D), g).to(dev)
    tables = torch.randperm(R * M, generator=g).to(torch.int32).reshape(R, M).to(dev)
    query_lens, seq_lens = (torch.zeros(R, dtype=torch.int32, device=dev) for _ in range(2))
    q = torch.zeros((R, heads, D), dtype=torch.bfloat16, device=dev)
    k, v = (torch.zeros((R, kv_heads, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    out = torch.zeros_like(q)

    def step():
        meta = layers.build_append_metadata_on_device(query_lens, seq_lens, tables, page, R, max_query_len=1)
        meta.append(k, v, cache)
        meta.attention(q, cache, out=out)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()                                # all padding: nothing happens
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for lens in ([1000, 1, 16, 17, 300, 64], [5, 900], [], [700, 2, 1]):
        n = len(lens)
        query_lens.copy_(torch.tensor([1] * n + [0] * (R - n), dtype=torch.int32))
        seq_lens.copy_(torch.tensor(lens + [0] * (R - n), dtype=torch.int32))
        for t in (q, k, v):
            t.copy_(randn(t.shape, g))
        before = cache.clone()
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        eager_cache, eager_out = cache.clone(), out.clone()
        # the cache: each request's last entry, nothing else
        want = before.clone()
        for r, t in enumerate(lens):
            page_no = int(tables[r, (t - 1) // page])
            want[page_no, 0, (t - 1) % page], want[page_no, 1, (t - 1) % page] = k[r], v[r]
        assert torch.equal(cache, want)
        assert bool((out[n:] == 9.0).all())
        if n:
            b = dict(query=q[:n].cpu().flatten(1), cache=cache.cpu(), new=[1] * n, total=lens, page_size=page, heads=heads,
                     kv_heads=kv_heads, head_size=D, dtype=torch.bfloat16,
                     kv_indices=torch.cat([tables[r, :(t + page - 1) // page] for r, t in enumerate(lens)]).cpu(),
                     kv_indptr=torch.tensor(np.concatenate([[0], np.cumsum([(t + page - 1) // page for t in lens])])))
            check(b, out[:n], None, reference(b))
        step()                                # the program's own eager call between the replays
        torch.cuda.synchronize()
        assert torch.equal(cache, eager_cache) and torch.equal(out, eager_out)


def test_two_streams_and_two_graphs_do_not_share_scratch(ops, dev):
    """Cut contexts on two streams at once, eager and as two graphs replayed together."""
    b = [build_batch(24 + i, 16, [1] * 4, [3000 + 500 * i, 2000, 900, 4000], 8, 2, 128, torch.bfloat16) for i in range(2)]
    d = [to_dev(x, dev) for x in b]
    want = [attend(ops, x, max_query_len=1) for x in d]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, x in zip(streams, d):
            with torch.cuda.stream(s):
                got.append([attend(ops, x, max_query_len=1) for _ in range(4)])
        torch.cuda.synchronize()
        for w, outs in zip(want, got):
            assert all(torch.equal(o, w) for o in outs)
    graphs, outs = [], []
    for s, x in zip(streams, d):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append([attend(ops, x, max_query_len=1) for _ in range(4)])
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(t, w) for t in o)


# ---- metadata ------------------------------------------------------------------------------------

def _metadata(new, total, tables, page, T, P):
    """The definition, request by request."""
    M = tables.shape[1]
    new, total = [max(n, 0) for n in new], [max(t, 0) for t in total]
    pages = [min(-(-t // page), M) for t in total]
    qo, kv = np.concatenate([[0], np.cumsum(new)]), np.concatenate([[0], np.cumsum(pages)])
    ix = [int(tables[r, i]) for r, p in enumerate(pages) for i in range(p)]
    last = [min(t - (p - 1) * page, page) if p else 0 for t, p in zip(total, pages)]
    bi, pos, slot = [], [], []
    for r, (n, t) in enumerate(zip(new, total)):
        for j in range(n):
            x = t - n + j
            ok = x >= 0 and x // page < pages[r]
            pg = int(tables[r, x // page]) if ok else -1
            bi.append(r)
            pos.append(x if ok else -1)
            slot.append(pg * page + x % page if ok and pg >= 0 else -1)
    fit = lambda v, n: (v + [-1] * n)[:n]  # noqa: E731
    return (np.minimum(qo, T).tolist(), np.minimum(kv, P).tolist(), fit(ix, P), last, fit(bi, T), fit(pos, T), fit(slot, T),
            [max(v, 0) for v in fit(pos, T)])


@pytest.mark.parametrize("R", [1, 2, 7, 300, 4096, 4097, 5000])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_metadata_over_sizes_and_odd_lengths(ops, dev, R, page):
    rng = np.random.default_rng(R + page)
    M = 9
    tables = torch.from_numpy(rng.integers(-1, 1000, (R, M + 3)).astype(np.int32))
    new = rng.integers(-1, 7, R)
    total = np.where(rng.random(R) < 0.1, rng.integers(-3, 4, R), rng.integers(0, M * page + 5, R))
    if R <= 7:
        new[0], total[0] = 3000, M * page            # a chunk that begins before its sequence does
    T, P = int(np.maximum(new, 0).sum()), int(sum(min(-(-max(int(t), 0) // page), M) for t in total))
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)  # noqa: E731
    view = tables.to(dev)[:, :M]                      # rows further apart than they are long
    for dt, dp in ((0, 0), (37, 5), (-min(3, T), -min(2, P))):
        m = ops.kv_cache_ops.build_paged_kv_metadata(i32(new), i32(total), view, page, T + dt, P + dp)
        want = _metadata(new.tolist(), total.tolist(), tables[:, :M], page, T + dt, P + dp)
        for name, g, w in zip(m._fields, m, want):
            assert g.tolist() == w, name
            assert g.dtype == (torch.int64 if name == "rope_positions" else torch.int32)


def test_metadata_without_requests_or_pages(ops, dev):
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    m = ops.kv_cache_ops.build_paged_kv_metadata(none, none, torch.zeros((0, 4), dtype=torch.int32, device=dev), 16, 3, 2)
    assert m.qo_indptr.tolist() == [0] and m.kv_indptr.tolist() == [0] and m.kv_indices.tolist() == [-1, -1]
    assert m.slot_mapping.tolist() == [-1] * 3 and m.rope_positions.tolist() == [0] * 3
    two = torch.tensor([2, 0], dtype=torch.int32, device=dev)
    m = ops.kv_cache_ops.build_paged_kv_metadata(two, two, torch.zeros((2, 0), dtype=torch.int32, device=dev), 16, 2)
    assert m.qo_indptr.tolist() == [0, 2, 2] and m.kv_indptr.tolist() == [0, 0, 0]
    assert m.slot_mapping.tolist() == [-1, -1] and m.kv_last_page_len.tolist() == [0, 0]


# ---- tokens that go nowhere -------------------------------------------------------------------------

@pytest.mark.parametrize("heads,head_size,dtype,nnz", [(8, 128, torch.bfloat16, 70), (2, 64, torch.float16, 3000),
                                                       (16, 160, torch.bfloat16, 40), (1, 3, torch.float32, 33)])
@pytest.mark.parametrize("use_slots", [False, True])
def test_append_skips_negative_destinations(ops, dev, heads, head_size, dtype, nnz, use_slots):
    g = gen(nnz)
    page = 16
    pages = (nnz + page - 1) // page
    k, v = (randn((nnz, heads, head_size), g, dtype).to(dev) for _ in range(2))
    cache = randn((pages, 2, page, heads, head_size), g, dtype).to(dev)
    slots = torch.arange(nnz, dtype=torch.int32, device=dev)
    skip = torch.rand(nnz, generator=g).to(dev) < 0.4
    skip[-1] = True
    want = cache.clone().permute(0, 2, 1, 3, 4).reshape(-1, 2, heads, head_size)
    keep = ~skip
    want[slots.long()[keep], 0], want[slots.long()[keep], 1] = k[keep], v[keep]
    bi = torch.where(skip, -1, 0).to(torch.int32)
    pos = torch.where(skip, -1, slots).to(torch.int32)
    ix = torch.arange(pages, dtype=torch.int32, device=dev)
    indptr = torch.tensor([0, pages], dtype=torch.int32, device=dev)
    mapped = torch.where(skip, -1, slots).to(torch.int32)
    assert torch.equal(ops.kv_cache_ops.get_kv_slot_mapping(bi, pos, ix, indptr, page), mapped)
    ops.kv_cache_ops.append_paged_kv_cache(k, v, bi, pos, cache, ix, indptr, slot_mapping=mapped if use_slots else None)
    assert torch.equal(cache.permute(0, 2, 1, 3, 4).reshape(-1, 2, heads, head_size), want)


@pytest.mark.parametrize("nq,nkv,D,rot,T", [(32, 8, 128, 128, 40), (32, 8, 128, 128, 1500), (71, 1, 64, 64, 33),
                                            (4, 2, 64, 32, 20)])
@pytest.mark.parametrize("use_slots", [False, True])
def test_fused_rotary_append_skips_negative_destinations(ops, dev, nq, nkv, D, rot, T, use_slots):
    g = gen(T)
    page, pages = 16, (T + 15) // 16
    qkv = randn((T, (nq + 2 * nkv) * D), g).to(dev)
    cache = randn((pages, 2, page, nkv, D), g).to(dev)
    table = cos_sin_cache(2048, rot, THETA_LLAMA3, torch.bfloat16).to(dev)
    positions = torch.arange(T, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    skip = torch.rand(T, generator=g).to(dev) < 0.4
    bi, pos = torch.where(skip, -1, 0).to(torch.int32), torch.where(skip, -1, slots).to(torch.int32)
    ix = torch.arange(pages, dtype=torch.int32, device=dev)
    indptr = torch.tensor([0, pages], dtype=torch.int32, device=dev)
    split = [nq * D, nkv * D, nkv * D]
    want_qkv, before = qkv.clone(), cache.clone()
    wq, wk, wv = want_qkv.split(split, dim=-1)
    ops.pos_encoding_ops.rotary_embedding(positions, wq, wk, D, table, True)
    flat = before.permute(0, 2, 1, 3, 4).reshape(-1, 2, nkv, D)
    keep = ~skip
    flat[slots.long()[keep], 0] = wk.reshape(T, nkv, D)[keep]
    flat[slots.long()[keep], 1] = wv.reshape(T, nkv, D)[keep]
    q, k, v = qkv.split(split, dim=-1)
    old_k = k.clone()
    ops.kv_cache_ops.rotary_embedding_append_paged_kv(
        positions, q, k, v, D, table, True, bi, pos, cache, ix, indptr,
        slot_mapping=torch.where(skip, -1, slots).to(torch.int32) if use_slots else None)
    assert torch.equal(q, wq) and torch.equal(k, old_k)
    assert torch.equal(cache.permute(0, 2, 1, 3, 4).reshape(-1, 2, nkv, D), flat)


@pytest.mark.parametrize("states", [2, 5])
def test_merge_strides(ops, dev, states):
    """States next to each other per token, and per state; a state is a view of a larger tensor."""
    g = gen(states)
    v = randn((7, states, 6, 64), g).to(dev)
    z = torch.randn((7, states, 6), generator=g).to(dev)
    a, az = ops.kv_cache_ops.merge_attention_states(v.transpose(0, 1), z.transpose(0, 1))
    b, bz = ops.kv_cache_ops.merge_attention_states(v.transpose(0, 1).contiguous(), z.transpose(0, 1).contiguous())
    assert torch.equal(a, b) and torch.equal(az, bz)
    wide = torch.zeros((states, 7, 8, 64), dtype=torch.bfloat16, device=dev)
    wide[:, :, :6] = v.transpose(0, 1)
    c, _ = ops.kv_cache_ops.merge_attention_states(wide[:, :, :6], z.transpose(0, 1))
    assert torch.equal(c, b)
    # unaligned rows: the element-wise kernel
    odd = torch.zeros((states, 7, 6 * 64 + 3), dtype=torch.bfloat16, device=dev)
    odd[:, :, 3:] = v.transpose(0, 1).flatten(2)
    e, _ = ops.kv_cache_ops.merge_attention_states(odd[:, :, 3:].unflatten(2, (6, 64)), z.transpose(0, 1))
    assert bool(((e.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-6).all())


# ---- what reviews of the kernels asked for --------------------------------------------------------

@pytest.mark.parametrize("hint", [0, 8])
def test_decreasing_index_vectors_stay_inside_the_workspace(ops, dev, hint):
    """Index vectors that decrease name more tiles than the tensors' sizes allow for: the states that
    cutting leaves in the workspace stay within it (the memory on both sides is left as it was)."""
    lib = abi.load()
    T, N, D, S = 64, 300, 64, 33
    d = dict(query=torch.ones((T, 8, D), dtype=torch.bfloat16, device=dev),
             cache=torch.ones((N, 2, 16, 1, D), dtype=torch.bfloat16, device=dev),
             qo_indptr=torch.tensor([0, T] * ((S + 1) // 2), dtype=torch.int32, device=dev),
             kv_indptr=torch.tensor([0, N] * ((S + 1) // 2), dtype=torch.int32, device=dev),
             kv_indices=torch.arange(N, dtype=torch.int32, device=dev),
             last=torch.full((S,), 16, dtype=torch.int32, device=dev))
    need = lib.sarathi_paged_attention_workspace_bytes
    need.restype = ctypes.c_int64
    bytes_ = need(abi.i64(T), abi.i64(S), abi.i64(N), abi.ci(8), abi.ci(1), abi.ci(D), abi.ci(16), abi.i64(hint))
    assert bytes_ > 0
    guard = 1 << 24
    ws = torch.full((bytes_ + 2 * guard,), 77, dtype=torch.uint8, device=dev)
    out = torch.empty_like(d["query"])
    abi.check(lib, _abi_attention(lib, d, out, abi.vp(ws.data_ptr() + guard), bytes_, D ** -0.5, hint))
    torch.cuda.synchronize()
    assert bool((ws[:guard] == 77).all()) and bool((ws[guard + bytes_:] == 77).all())


@pytest.mark.parametrize("new", [1, 40])
def test_small_probabilities_keep_their_share_in_float16(ops, dev, new):
    """One key far above all others: theirs are 2^-25.5 of it, below half of float16's least step, and
    only they have values.  They are held 2^7 higher, where a step is 2^-24 / 2^-18.5 = 2.2 % of one:
    half of it, and half a step of the result (2^-25), is the bound."""
    keys, D = 1500, 64
    d = dict(query=torch.zeros((new, 4, D), dtype=torch.float16, device=dev),
             cache=torch.zeros((94, 2, 16, 1, D), dtype=torch.float16, device=dev),
             qo_indptr=torch.tensor([0, new], dtype=torch.int32, device=dev),
             kv_indptr=torch.tensor([0, 94], dtype=torch.int32, device=dev),
             kv_indices=torch.arange(94, dtype=torch.int32, device=dev),
             last=torch.tensor([keys - 93 * 16], dtype=torch.int32, device=dev))
    d["query"][..., 0] = 25.5
    d["cache"][:, 1] = 1024.0
    d["cache"][:4, 0, :, :, 0] = 1.0       # the 64 first keys, one block of every wave
    d["cache"][:4, 1] = 0.0
    out = ops.kv_cache_ops.paged_attention(d["query"], d["cache"], d["qo_indptr"], d["kv_indptr"], d["kv_indices"],
                                           d["last"], sm_scale=float(np.log(2.0)), causal=False)
    small = (keys - 64) * 2.0 ** -25.5
    want = 1024 * small / (64 + small)
    got = out.cpu().double()
    assert bool(((got - want).abs() <= 2.0 ** -6.5 * want + 2.0 ** -25).all()), (got.min().item(), want)


@pytest.mark.parametrize("new,heads,D,page", [(1, 8, 128, 16), (60, 8, 128, 16), (1, 4, 64, 5), (70, 4, 64, 24)])
def test_pages_behind_the_window_may_be_gone(ops, dev, new, heads, D, page):
    """Keys that the window hides from every token are not read: their pages may hold anything, or no
    longer be named."""
    total, window = 1333, 300
    b = build_batch(41, page, [new], [total], heads, 1, D, torch.bfloat16)
    want = reference(b, window=window)
    first = total - new - window                                  # first key that any token sees
    flat = b["cache"][b["kv_indices"].long()].clone()             # pages in order
    for t in range(first):
        flat[t // page, :, t % page] = float("nan")
    b["cache"][b["kv_indices"].long()] = flat
    b["kv_indices"][:first // page] = -1
    got, lse = call(ops, dev, b, window_left=window, return_lse=True)
    check(b, got, lse, want)


@pytest.mark.parametrize("new,total,heads,kv_heads,head_size,page,dtype,kw", [
    ([300], [1700], 12, 4, 256, 16, torch.bfloat16, {}),
    ([300, 1, 40], [300, 2000, 1999], 8, 1, 256, 7, torch.float16, {}),                 # cut, odd pages
    ([129, 1], [900, 64], 40, 2, 192, 32, torch.bfloat16, dict(window_left=200)),
    ([70, 2, 1], [70, 1, 90], 3, 3, 136, 16, torch.float16, dict(causal=False)),
    ([40], [2600], 2, 1, 200, 5, torch.bfloat16, {}),
])
def test_chunks_of_long_heads(ops, dev, new, total, heads, kv_heads, head_size, page, dtype, kw):
    b = build_batch(43, page, new, total, heads, kv_heads, head_size, dtype)
    got, lse = call(ops, dev, b, return_lse=True, **kw)
    check(b, got, lse, reference(b, kw.get("causal", True), kw.get("window_left", -1)))
    assert torch.equal(call(ops, dev, b, **kw), got)


@pytest.mark.parametrize("new,total,heads,kv_heads,head_size,page,dtype,kw", [
    # more items than the GPU takes at once, of all lengths: sorted into bins
    ([1] * 70, [1 + (i * 619) % 2600 for i in range(70)], 16, 8, 64, 16, torch.bfloat16, {}),
    ([1] * 150, [1 + (i * 619) % 1900 for i in range(150)], 8, 8, 64, 16, torch.float16, {}),
    ([2] * 90, [2 + (i * 431) % 2100 for i in range(90)], 8, 8, 128, 32, torch.bfloat16, dict(window_left=1500)),
    # beside a chunk
    ([200, 1, 90] + [1] * 90, [700, 1500, 90] + [(i * 619) % 2300 for i in range(90)], 16, 8, 64, 16, torch.bfloat16, {}),
    # several tiles per request (the hint of the second run is too small for them)
    ([7] * 40, [7 + (i * 619) % 2400 for i in range(40)], 64, 16, 64, 16, torch.bfloat16, {}),
])
@pytest.mark.parametrize("hint", [None, 1])
def test_ragged_batches_sorted_by_length(ops, dev, new, total, heads, kv_heads, head_size, page, dtype, kw, hint):
    b = build_batch(44, page, new, total, heads, kv_heads, head_size, dtype)
    got, lse = call(ops, dev, b, return_lse=True, max_query_len=hint, **kw)
    check(b, got, lse, reference(b, True, kw.get("window_left", -1)))
    assert torch.equal(call(ops, dev, b, max_query_len=hint, **kw), got)


def test_windows_of_nothing_and_everything_and_large_pages(ops, dev):
    for page in (4096, 48):
        b = build_batch(45, page, [40, 1, 3], [300, 4500, 3], 8, 2, 64, torch.bfloat16, spare=1)
        for window in (0, 1, 5000, 1 << 40):
            got, lse = call(ops, dev, b, return_lse=True, window_left=window)
            check(b, got, lse, reference(b, window=min(window, 1 << 20)))
    d = to_dev(b, dev)                                  # a cache without a page: nobody sees a key
    d["cache"] = d["cache"][:0]
    out, lse = attend(ops, d, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -torch.inf).all())


@pytest.mark.parametrize("new,total,heads,kv_heads,head_size,page,dtype", [
    ([1] * 700, [1 + (i * 619) % 150 for i in range(700)], 4, 2, 64, 16, torch.bfloat16),            # nothing to cut
    ([1] * 699 + [1], [1 + (i * 619) % 150 for i in range(699)] + [4000], 4, 1, 64, 16, torch.float16),
    ([i % 3 for i in range(1100)] + [170, 90], [(i * 37) % 90 for i in range(1100)] + [900, 1700], 8, 2, 64, 16,
     torch.bfloat16),                                                                            # chunks and empty requests
    ([0] * 513, [0] * 513, 4, 2, 64, 16, torch.bfloat16),
])
@pytest.mark.parametrize("hint", [None, 1])
def test_batches_of_many_requests_are_planned(ops, dev, new, total, heads, kv_heads, head_size, page, dtype, hint):
    """Above 512 requests a kernel plans the launch; without its workspace every workgroup looks at all."""
    b = build_batch(46, page, new, total, heads, kv_heads, head_size, dtype)
    want = reference(b)
    got, lse = call(ops, dev, b, return_lse=True, max_query_len=hint)
    check(b, got, lse, want)
    if sum(new) == 0:
        return
    d, lib = to_dev(b, dev), abi.load()
    out = torch.empty_like(d["query"])
    abi.check(lib, _abi_attention(lib, d, out, abi.vp(None), 0, head_size ** -0.5, hint or 0))
    check(b, out, None, want)


def test_decreasing_index_vectors_stay_inside_a_planned_workspace(ops, dev):
    lib = abi.load()
    T, N, D, S = 64, 300, 64, 701
    d = dict(query=torch.ones((T, 8, D), dtype=torch.bfloat16, device=dev),
             cache=torch.ones((N, 2, 16, 1, D), dtype=torch.bfloat16, device=dev),
             qo_indptr=torch.tensor([0, T] * ((S + 1) // 2), dtype=torch.int32, device=dev),
             kv_indptr=torch.tensor([0, N] * ((S + 1) // 2), dtype=torch.int32, device=dev),
             kv_indices=torch.arange(N, dtype=torch.int32, device=dev),
             last=torch.full((S,), 16, dtype=torch.int32, device=dev))
    need = lib.sarathi_paged_attention_workspace_bytes
    need.restype = ctypes.c_int64
    bytes_ = need(abi.i64(T), abi.i64(S), abi.i64(N), abi.ci(8), abi.ci(1), abi.ci(D), abi.ci(16), abi.i64(0))
    guard = 1 << 24
    ws = torch.full((bytes_ + 2 * guard,), 77, dtype=torch.uint8, device=dev)
    out = torch.empty_like(d["query"])
    abi.check(lib, _abi_attention(lib, d, out, abi.vp(ws.data_ptr() + guard), bytes_, D ** -0.5))
    torch.cuda.synchronize()
    assert bool((ws[:guard] == 77).all()) and bool((ws[guard + bytes_:] == 77).all())
