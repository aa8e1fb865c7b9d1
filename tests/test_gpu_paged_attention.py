"""GPU: index vectors built from lengths, attention over the paged cache and the join of attention
states, against plain evaluations in 64 bits.

Tolerance of an attention output: the kernels round each probability to the tensor dtype (half a
step, eps / 2 of it), multiply by v in 32 bits and round the result once (another eps / 2).  The
first kind adds up to at most eps / 2 * sum_i p_i |v_i| / sum_i p_i, so
|got - want| <= eps / 2 * (sum_i w_i |v_i| + |want|) with w the exact weights; 32-bit sums and the
scores' own error (products of 16-bit values are exact in 32 bits, sums of up to 256 of them and the
exponent are off by a few 2^-24 relative to |q| |k| scale) stay below 5e-5 of sum_i w_i |v_i| for the
sizes here."""
import numpy as np
import pytest
import torch

from helpers import gen, randn

pytestmark = pytest.mark.gpu


def build_batch(seed, page_size, new, total, heads, kv_heads, head_size, dtype, spare=3, poison=True):
    """CPU tensors of a batch: packed qkv rows, a cache whose unused entries hold NaN."""
    g = gen(seed)
    need = [(t + page_size - 1) // page_size for t in total]
    num_pages = sum(need) + spare
    order = torch.randperm(num_pages, generator=g)[:sum(need)].to(torch.int32)
    cache = randn((num_pages, 2, page_size, kv_heads, head_size), g, dtype)
    used = torch.zeros((num_pages, page_size), dtype=torch.bool)
    at = 0
    for t, n in zip(total, need):
        slots = order[at:at + n].long()
        for i in range(n):
            used[slots[i], :min(page_size, t - i * page_size)] = True
        at += n
    if poison:
        cache.permute(0, 2, 1, 3, 4)[~used] = float("nan")
    qkv = randn((sum(new), (heads + 2 * kv_heads) * head_size), g, dtype)
    starts = lambda v: torch.tensor(np.concatenate([[0], np.cumsum(v)]), dtype=torch.int32)  # noqa: E731
    last = [t - (n - 1) * page_size if n else 0 for t, n in zip(total, need)]
    return dict(query=qkv[:, :heads * head_size], cache=cache, qo_indptr=starts(new), kv_indptr=starts(need),
                kv_indices=order, last=torch.tensor(last, dtype=torch.int32), new=new, total=total,
                page_size=page_size, heads=heads, kv_heads=kv_heads, head_size=head_size, dtype=dtype)


def reference(b, causal=True, window=-1, scale=None):
    """out, lse and sum_i w_i |v_i| in 64 bits, request by request."""
    H, K, D, P = b["heads"], b["kv_heads"], b["head_size"], b["page_size"]
    scale = D ** -0.5 if scale is None else scale
    T = b["query"].shape[0]
    out, mag = torch.zeros((T, H, D), dtype=torch.float64), torch.zeros((T, H, D), dtype=torch.float64)
    lse = torch.full((T, H), -torch.inf, dtype=torch.float64)
    row = 0
    for r, (n, t) in enumerate(zip(b["new"], b["total"])):
        pages = b["kv_indices"][b["kv_indptr"][r]:b["kv_indptr"][r + 1]].long()
        kv = b["cache"][pages].permute(0, 2, 1, 3, 4).reshape(-1, 2, K, D)[:t].double()
        q = b["query"][row:row + n].reshape(n, K, H // K, D).double()
        pos = torch.arange(t - n, t)[:, None]
        key = torch.arange(t)[None]
        see = torch.ones((n, t), dtype=torch.bool)
        if causal:
            see &= key <= pos
        if window >= 0:
            see &= key >= pos - window
        s = torch.einsum("nkgd,tkd->nkgt", q, kv[:, 0]) * scale
        s = s.masked_fill(~see[:, None, None, :], -torch.inf)
        if t and n:
            z = s.logsumexp(-1)
            w = torch.where(z[..., None] == -torch.inf, 0.0, (s - z[..., None]).exp())
            out[row:row + n] = torch.einsum("nkgt,tkd->nkgd", w, kv[:, 1]).reshape(n, H, D)
            mag[row:row + n] = torch.einsum("nkgt,tkd->nkgd", w, kv[:, 1].abs()).reshape(n, H, D)
            lse[row:row + n] = z.reshape(n, H)
        row += n
    return out, lse, mag


def call(ops, dev, b, **kw):
    to = lambda t: t.to(dev)  # noqa: E731
    qkv = to(b["query"]._base if b["query"]._base is not None else b["query"])
    q = qkv[:, :b["heads"] * b["head_size"]].unflatten(1, (b["heads"], b["head_size"]))
    return ops.kv_cache_ops.paged_attention(q, to(b["cache"]), to(b["qo_indptr"]), to(b["kv_indptr"]),
                                            to(b["kv_indices"]), to(b["last"]), **kw)


def check(b, got, lse, want):
    out, z, mag = want
    half = torch.finfo(b["dtype"]).eps / 2
    tiny = torch.finfo(b["dtype"]).smallest_normal if b["dtype"] == torch.float16 else 1e-30
    bound = half * (mag + out.abs()) + 5e-5 * mag + tiny
    diff = (got.cpu().double().reshape(out.shape) - out).abs()
    assert bool((diff <= bound).all()), "off by %.3g where %.3g is allowed" % (
        diff.max().item(), bound.flatten()[(diff - bound).argmax()].item())
    if lse is not None:
        dead = z == -torch.inf
        lse = lse.cpu().double()
        assert torch.equal(lse == -torch.inf, dead)
        # scores: 32-bit sums of up to 256 exact products; z itself rounds once
        assert bool(((lse - z).abs()[~dead] <= 2e-6 * z.abs()[~dead] + 1e-5).all())


BATCHES = {
    "one token, one key": ([1], [1]),
    "one long": ([1], [1537]),
    "decodes": ([1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 700]),
    "chunk": ([37], [37]),
    "chunk in context": ([53, 2], [400, 1030]),
    "hybrid": ([40, 1, 3, 1, 1], [40, 33, 9, 16, 200]),
    "empty requests": ([0, 5, 0, 1, 0], [0, 7, 30, 1, 0]),
    "no key at all": ([3, 1], [0, 4]),
    "more new tokens than keys": ([6, 2], [4, 9]),
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("heads,kv_heads,head_size,page_size,dtype", [
    (32, 8, 128, 16, torch.bfloat16),
    (4, 4, 128, 7, torch.float16),
    (71, 1, 64, 16, torch.bfloat16),
    (6, 2, 80, 5, torch.float16),
    (4, 1, 256, 16, torch.bfloat16),
    (5, 1, 20, 3, torch.float16),      # rows of 40 bytes: the plain kernel
    (8, 8, 64, 1, torch.float16),
])
def test_attention_matches_definition(ops, dev, batch, heads, kv_heads, head_size, page_size, dtype):
    new, total = BATCHES[batch]
    b = build_batch(7, page_size, new, total, heads, kv_heads, head_size, dtype)
    for kw in (dict(), dict(causal=False), dict(window_left=0), dict(window_left=20),
               dict(causal=False, window_left=9)):
        got, lse = call(ops, dev, b, return_lse=True, max_query_len=max(new), **kw)
        check(b, got, lse, reference(b, kw.get("causal", True), kw.get("window_left", -1)))


def test_metadata_matches_definition(ops, dev):
    from oracle import paged_kv
    page, tables = 16, torch.arange(40, dtype=torch.int32).reshape(4, 10).flip(1)
    new, total = [3, 0, 1, 7], [20, 5, 33, 7]
    m = ops.kv_cache_ops.build_paged_kv_metadata(torch.tensor(new, dtype=torch.int32, device=dev),
                                                 torch.tensor(total, dtype=torch.int32, device=dev),
                                                 tables.to(dev), page, num_tokens=13, num_kv_pages=9)
    assert m.qo_indptr.tolist() == [0, 3, 3, 4, 11]
    assert m.kv_indptr.tolist() == [0, 2, 3, 6, 7]
    assert m.kv_indices.tolist() == [9, 8, 19, 29, 28, 27, 39, -1, -1]
    assert m.kv_last_page_len.tolist() == [4, 5, 1, 7]
    b, p = paged_kv.get_batch_indices_positions(m.qo_indptr.cpu().numpy(), np.array(total), 13)
    assert m.batch_indices.tolist() == b.tolist() and m.positions.tolist() == p.tolist()
    assert m.rope_positions.tolist() == [max(v, 0) for v in p.tolist()]
    assert m.slot_mapping.tolist()[-2:] == [-1, -1]
    assert m.slot_mapping.tolist()[:3] == [8 * 16 + 1, 8 * 16 + 2, 8 * 16 + 3]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("states,tokens,heads,head_size", [(2, 16, 32, 128), (3, 5, 3, 20), (4, 33, 8, 80),
                                                           (1, 1, 1, 1), (9, 2, 5, 64)])
def test_merge_matches_definition(ops, dev, dtype, states, tokens, heads, head_size):
    g = gen(states)
    v = randn((states, tokens, heads, head_size), g, dtype)
    lse = torch.randn((states, tokens, heads), generator=g) * 3
    lse[torch.rand(lse.shape, generator=g) < 0.3] = -torch.inf
    v[lse == -torch.inf] = float("nan")          # a state without keys: not looked at
    out, z = ops.kv_cache_ops.merge_attention_states(v.to(dev), lse.to(dev))
    want_z = lse.double().logsumexp(0)
    w = torch.where(want_z == -torch.inf, 0.0, (lse.double() - want_z).exp())
    x = torch.where(w[..., None] == 0, 0.0, v.double())
    want, mag = (w[..., None] * x).sum(0), (w[..., None] * x.abs()).sum(0)
    # one rounding to the dtype, 32-bit weights and sums
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 4e-6 * mag + 1e-7 * (dtype == torch.float16)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    dead = want_z == -torch.inf
    assert torch.equal(z.cpu() == -torch.inf, dead)
    assert bool(((z.cpu().double() - want_z).abs()[~dead] <= 1e-6 * want_z.abs()[~dead] + 1e-6).all())


@pytest.mark.parametrize("new,total", [
    ([129], [129]), ([256], [900]), ([130, 1, 77, 1], [130, 64, 500, 3]), ([300], [2111]),
    ([65, 64, 63, 1], [65, 640, 63, 1000]),
])
@pytest.mark.parametrize("heads,kv_heads,head_size,page_size,dtype", [
    (8, 2, 128, 16, torch.bfloat16),
    (4, 4, 128, 7, torch.float16),
    (7, 1, 64, 32, torch.bfloat16),
    (3, 1, 96, 16, torch.float16),
    (2, 2, 40, 48, torch.bfloat16),
])
def test_chunks_match_definition(ops, dev, new, total, heads, kv_heads, head_size, page_size, dtype):
    b = build_batch(11, page_size, new, total, heads, kv_heads, head_size, dtype)
    for kw in (dict(), dict(causal=False), dict(window_left=100)):
        got, lse = call(ops, dev, b, return_lse=True, **kw)
        check(b, got, lse, reference(b, kw.get("causal", True), kw.get("window_left", -1)))
