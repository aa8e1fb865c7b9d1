"""Workloads of the paged-attention operators: the batch metadata built on the GPU, attention of a
hybrid batch (chunks of new tokens and single decode tokens) over the paged KV cache, and the join
of attention states computed over disjoint parts of a context.

``listed()`` names the fixed cases, ``draw(rng)`` gives another case of the same ranges,
``prepare(case, seed)`` makes what a serving program holds before the call, ``run(state)`` makes one
pass -- through the package where ``own`` is true, as elementary tensor operations otherwise --
``exact(case, seed)`` evaluates the definition in 64 bits and ``work(case)`` counts what a pass
cannot do without.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PHI = 0.6180339887498949      # spreads lengths evenly over a range, the same for every seed


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sarathi-serve_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import sarathi_amd
    return sarathi_amd.kv_cache_ops


# ---- cases -------------------------------------------------------------------------------------

def _batch(name, op, chunks, chunk_len, context, decodes, dec_lo, dec_hi, page, **kw):
    """``chunks`` prompt chunks of up to ``chunk_len`` new tokens after up to ``context`` cached
    ones, then ``decodes`` requests with one new token and dec_lo..dec_hi tokens in all."""
    return dict(name=name, op=op, chunks=chunks, chunk_len=chunk_len, context=context,
                decodes=decodes, dec_lo=dec_lo, dec_hi=dec_hi, page=page, **kw)


def listed():
    return [
        # a small decode step: the latency of building the indices of the batch
        _batch("metadata_16_decodes", "metadata", 0, 0, 0, 16, 1, 8191, 16),
        # a step of a large deployment: eight chunks and a thousand running requests
        _batch("metadata_1008_requests", "metadata", 8, 2048, 4096, 1000, 1, 32767, 16),
        # one user, one token: nothing but latency (Llama-3-8B heads)
        _batch("decode_1_request", "attention", 0, 0, 0, 1, 4096, 4096, 16,
               heads=32, kv_heads=8, head_size=128, dtype="bf16", window=-1, lse=False),
        # the running requests of the 2304-token batch, ragged contexts (Llama-3-8B heads)
        _batch("decode_256_requests", "attention", 0, 0, 0, 256, 1, 8191, 16,
               heads=32, kv_heads=8, head_size=128, dtype="bf16", window=-1, lse=False),
        # few requests of very long contexts: the work has to be split over the context (70B heads)
        _batch("decode_8_long", "attention", 0, 0, 0, 8, 40000, 65536, 16,
               heads=64, kv_heads=8, head_size=128, dtype="fp16", window=-1, lse=True),
        # a short odd chunk, a key head per query head, pages that divide nothing, a sliding window
        _batch("chunk_333_window", "attention", 1, 333, 1001, 0, 0, 0, 7,
               heads=32, kv_heads=32, head_size=128, dtype="fp16", window=512, lse=False),
        # Falcon-7B heads: 71 query heads share one key head of 64
        _batch("hybrid_71_heads_of_64", "attention", 1, 512, 0, 64, 1, 2048, 16,
               heads=71, kv_heads=1, head_size=64, dtype="bf16", window=-1, lse=True),
        # the 2304-token hybrid batch: a 2048-token chunk at 4096 and 256 decodes (Llama-3-8B heads)
        _batch("hybrid_2304", "attention", 1, 2048, 4096, 256, 1, 8191, 16,
               heads=32, kv_heads=8, head_size=128, dtype="bf16", window=-1, lse=False),
        # several prompts of one step, ragged, 70B heads
        _batch("chunks_4_ragged", "attention", 4, 1024, 4096, 0, 0, 0, 16,
               heads=64, kv_heads=8, head_size=128, dtype="bf16", window=-1, lse=False),
        # a large chunk deep in a long prompt
        _batch("chunk_4096_at_12288", "attention", 1, 4096, 12288, 0, 0, 0, 16,
               heads=32, kv_heads=8, head_size=128, dtype="bf16", window=-1, lse=False),
        # shared prefix + own suffix of a small decode batch
        dict(name="merge_2_of_16", op="merge", tokens=16, states=2, heads=32, head_size=128, dtype="bf16"),
        # a 2304-token batch whose context was attended to in four parts
        dict(name="merge_4_of_2304", op="merge", tokens=2304, states=4, heads=64, head_size=128, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["metadata", "attention", "attention", "attention", "attention", "merge"])
    if op == "merge":
        return dict(op=op, tokens=_log(rng, 1, 2304), states=rng.randint(2, 4), heads=rng.choice([8, 12, 32, 64]),
                    head_size=rng.choice([64, 80, 128]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    page = rng.choice([1, 7, 16, 16, 16, 32, 64])
    if op == "metadata":
        c = _batch("", op, rng.randint(0, 8), _log(rng, 2, 2048), _log(rng, 1, 4096), _log(rng, 1, 1000), 1,
                   _log(rng, 16, 32767), page)
        del c["name"]
        return c
    heads, kv_heads, size = rng.choice([(32, 8, 128), (64, 8, 128), (32, 32, 128), (128, 8, 64), (71, 1, 64),
                                        (56, 8, 128), (24, 8, 96), (40, 10, 80), (12, 4, 256)])
    kind = rng.choice(["decode", "chunk", "hybrid"])
    chunks = 0 if kind == "decode" else rng.randint(1, 3)
    decodes = 0 if kind == "chunk" else _log(rng, 1, 128)
    hi = _log(rng, 1, 8191) if decodes > 8 else _log(rng, 1, 40000)
    c = _batch("", op, chunks, _log(rng, 2, 1024) if chunks else 0, _log(rng, 1, 4096) - 1 if chunks else 0,
               decodes, min(hi, rng.choice([1, hi])) if decodes else 0, hi if decodes else 0, page,
               heads=heads, kv_heads=kv_heads, head_size=size, dtype=rng.choice(["bf16", "fp16"]),
               window=rng.choice([-1, -1, _log(rng, 1, 2048)]), lse=rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, tokens in all) of every request: a matter of the case, not of the seed."""
    new, total = [], []
    for i in range(case["chunks"]):
        f = 1.0 if i == 0 else (i * PHI) % 1.0
        n = max(1, int(case["chunk_len"] * (0.25 + 0.75 * f)))
        new.append(n)
        total.append(n + int(case["context"] * (1.0 if i == 0 else (i * PHI * PHI) % 1.0)))
    for i in range(case["decodes"]):
        f = 1.0 if i == 0 else (i * PHI) % 1.0
        new.append(1)
        total.append(case["dec_lo"] + int((case["dec_hi"] - case["dec_lo"]) * f))
    return new, total


def _visible(case):
    """How many (new token, key) pairs the mask leaves."""
    w, pairs = case["window"], 0
    for n, t in zip(*_lengths(case)):
        first = t - n + 1                                  # keys up to and with the first new token
        if w < 0 or t <= w + 1:
            pairs += n * (first + t) // 2
        else:
            pairs += sum(min(k, w + 1) for k in range(first, t + 1))
    return pairs


def _keys_read(case):
    """How many keys at least one new token sees."""
    w = case["window"]
    return sum(t if w < 0 else t - max(0, t - n - w) for n, t in zip(*_lengths(case)))


def work(case):
    if case["op"] == "merge":
        rows = case["tokens"] * case["heads"]
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        return {"bytes": rows * (case["states"] + 1) * (case["head_size"] * size + 4),
                "flops": rows * case["states"] * (2 * case["head_size"] + 4)}
    new, total = _lengths(case)
    pages = sum(-(-t // case["page"]) for t in total)
    if case["op"] == "metadata":
        # lengths and pages in; two prefix arrays, last-page lengths, pages and four words per token out
        # (one of them 8 bytes wide)
        return {"bytes": 4 * (2 * len(new) + pages + 3 * len(new) + 2 + pages) + 20 * sum(new),
                "flops": sum(new) + pages}
    rows = sum(new) * case["heads"]
    kv = 2 * _keys_read(case) * case["kv_heads"] * case["head_size"] * 2
    return {"bytes": 2 * rows * case["head_size"] * 2 + kv + 4 * pages + (4 * rows if case["lse"] else 0),
            "flops": 4 * _visible(case) * case["heads"] * case["head_size"]}


# ---- inputs ------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "merge":
        s, t, h, d = (case[k] for k in ("states", "tokens", "heads", "head_size"))
        v = torch.randn((s, t, h, d), generator=g, device=dev, dtype=torch.float32).to(DTYPES[case["dtype"]])
        lse = torch.randn((s, t, h), generator=g, device=dev, dtype=torch.float32) * 2 + 7
        # a part in which a token sees nothing: now and then all but the first state
        lse[1:] = torch.where(torch.rand((s - 1, t, h), generator=g, device=dev) < 0.05, -math.inf, lse[1:])
        return {"case": case, "v": v, "lse": lse}
    new, total = _lengths(case)
    page = case["page"]
    need = [-(-t // page) for t in total]
    spare = 5
    order = torch.randperm(sum(need) + spare, generator=g, device=dev)[:sum(need)].to(torch.int32)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def starts(values):
        out = [0]
        for v in values:
            out.append(out[-1] + v)
        return out

    st = {"case": case, "num_tokens": sum(new), "num_pages": sum(need)}
    if case["op"] == "metadata":
        # what a scheduler that lives on the GPU holds: lengths and a dense table, pages of a request in a row
        table = torch.zeros((len(new), max(need)), dtype=torch.int32, device=dev)
        col = torch.arange(max(need), device=dev)
        table[col[None, :] < ints(need)[:, None]] = order
        st.update(query_lens=ints(new), seq_lens=ints(total), block_tables=table)
        return st
    h, hk, d, dt = case["heads"], case["kv_heads"], case["head_size"], DTYPES[case["dtype"]]
    cache = torch.empty((sum(need) + spare, 2, page, hk, d), device=dev, dtype=dt)
    cache.normal_(generator=g)
    # the query lies in a packed row of query, key and value, as the projection leaves it
    qkv = torch.empty((sum(new), (h + 2 * hk) * d), device=dev, dtype=dt)
    qkv.normal_(generator=g)
    st.update(query=qkv[:, :h * d].unflatten(1, (h, d)), cache=cache, qo_indptr=ints(starts(new)),
              kv_indptr=ints(starts(need)), kv_indices=order,
              last_page_len=ints([t - (n - 1) * page for t, n in zip(total, need)]),
              max_query_len=max(new), new=new, total=total)
    return st


# ---- one pass ----------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        ops = _ops()
        if op == "metadata":
            return tuple(ops.build_paged_kv_metadata(
                state["query_lens"], state["seq_lens"], state["block_tables"], state["case"]["page"],
                num_tokens=state["num_tokens"], num_kv_pages=state["num_pages"]))
        if op == "merge":
            return ops.merge_attention_states(state["v"], state["lse"])
        return ops.paged_attention(
            state["query"], state["cache"], state["qo_indptr"], state["kv_indptr"], state["kv_indices"],
            state["last_page_len"], causal=True, window_left=state["case"]["window"],
            max_query_len=state["max_query_len"], return_lse=state["case"]["lse"])
    return {"metadata": _metadata, "attention": _attention, "merge": _merge}[op](state)


def _metadata(st):
    page, dev = st["case"]["page"], st["seq_lens"].device
    new, total = st["query_lens"].long(), st["seq_lens"].long()
    pages = (total + page - 1) // page
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    qo = torch.cat((zero, new.cumsum(0)))
    kv = torch.cat((zero, pages.cumsum(0)))
    # the request a page, resp. a token, belongs to: how many requests end at or before it
    i = torch.arange(st["num_pages"], device=dev)
    r = torch.searchsorted(kv[1:].contiguous(), i, right=True)
    indices = st["block_tables"][r, i - kv[r]]
    t = torch.arange(st["num_tokens"], device=dev)
    b = torch.searchsorted(qo[1:].contiguous(), t, right=True)
    pos = total[b] - new[b] + t - qo[b]
    slot = st["block_tables"][b, pos // page].long() * page + pos % page
    last = total - (pages - 1).clamp_min(0) * page
    return (qo.int(), kv.int(), indices, last.int(), b.int(), pos.int(), slot.int(), pos)


def _attention(st):
    c = st["case"]
    q, n = st["query"], c["chunks"]
    out = torch.empty((q.shape[0] + 1,) + tuple(q.shape[1:]), dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[0] + 1, q.shape[1]), dtype=torch.float32, device=q.device)
    # requests padded to the longest of their kind: chunks together, single tokens together
    if n:
        _padded(st, slice(0, n), out, lse)
    if c["decodes"]:
        _padded(st, slice(n, n + c["decodes"]), out, lse)
    return (out[:-1], lse[:-1]) if c["lse"] else out[:-1]


def _padded(st, part, out, lse):
    c, q, cache = st["case"], st["query"], st["cache"]
    dev, page, h, hk, d = q.device, c["page"], c["heads"], c["kv_heads"], c["head_size"]
    rows, keys = max(st["new"][part]), max(st["total"][part])
    first = st["qo_indptr"][:-1][part].long()
    new = st["qo_indptr"][1:][part].long() - first
    kv0 = st["kv_indptr"][:-1][part].long()
    total = (st["kv_indptr"][1:][part].long() - kv0 - 1) * page + st["last_page_len"][part].long()
    tok = torch.arange(rows, device=dev)
    real = tok[None, :] < new[:, None]
    row = torch.where(real, first[:, None] + tok, out.shape[0] - 1)          # padding goes to a row of its own
    x = q[row.clamp_max(q.shape[0] - 1)].float()                             # [b, rows, h, d]
    x = x.reshape(-1, rows, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(-1, hk, rows * (h // hk), d)
    key = torch.arange(keys, device=dev)
    near = torch.minimum(key[None, :], total[:, None] - 1)                   # past the end: the last key again
    at = st["kv_indices"][kv0[:, None] + near // page].long()
    k = cache[at, 0, near % page].float().permute(0, 2, 3, 1)                # [b, hk, d, keys]
    v = cache[at, 1, near % page].float().permute(0, 2, 1, 3)                # [b, hk, keys, d]
    pos = total[:, None] - new[:, None] + tok                                # [b, rows]
    see = key[None, None, :] <= pos[:, :, None]
    if c["window"] >= 0:
        see &= key[None, None, :] >= pos[:, :, None] - c["window"]
    see = see[:, None, :, None, :].expand(-1, 1, -1, h // hk, -1).reshape(-1, 1, rows * (h // hk), keys)
    s = torch.matmul(x, k.contiguous()) * d ** -0.5
    s = s.masked_fill_(~see, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.contiguous()) / l.clamp_min(torch.finfo(torch.float32).tiny)
    o = o.reshape(-1, hk, rows, h // hk, d).permute(0, 2, 1, 3, 4).reshape(-1, rows, h, d)
    out[row] = o.to(out.dtype)
    lse[row] = (m + l.log()).reshape(-1, hk, rows, h // hk).permute(0, 2, 1, 3).reshape(-1, rows, h)


def _merge(st):
    v, lse = st["v"], st["lse"]
    m = lse.amax(0).clamp_min(torch.finfo(torch.float32).min)
    w = (lse - m).exp()
    l = w.sum(0)
    out = (v.float() * w[..., None]).sum(0) / l.clamp_min(torch.finfo(torch.float32).tiny)[..., None]
    return out.to(v.dtype), m + l.log()


# ---- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "metadata":
        return None                       # whole numbers
    st = prepare(case, seed)
    if case["op"] == "merge":
        z = st["lse"].double().logsumexp(0)
        share = (st["lse"].double() - z).exp()
        return torch.einsum("sth,sthd->thd", share, st["v"].double()), z
    h, hk, d, page, w = (case[k] for k in ("heads", "kv_heads", "head_size", "page", "window"))
    out = torch.zeros(st["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["query"].shape[:2], dtype=torch.float64, device="cuda")
    begin, pages = 0, 0
    for n, t in zip(*_lengths(case)):
        mine = st["kv_indices"][pages:pages + -(-t // page)].long()
        lo = max(0, t - n - w) if w >= 0 else 0
        for j in range(hk):
            k = st["cache"][mine, 0, :, j].reshape(-1, d)[lo:t].double()
            v = st["cache"][mine, 1, :, j].reshape(-1, d)[lo:t].double()
            for a in range(0, n, 512):
                b = min(n, a + 512)
                x = st["query"][begin + a:begin + b, j * (h // hk):(j + 1) * (h // hk)].double()
                dist = torch.arange(t - n + a, t - n + b, device="cuda")[:, None] - torch.arange(lo, t, device="cuda")
                hide = (dist < 0) | (dist > w) if w >= 0 else dist < 0
                s = (x.reshape(-1, d) @ k.T / math.sqrt(d)).reshape(b - a, h // hk, -1).masked_fill(hide[:, None], -math.inf)
                heads = slice(j * (h // hk), (j + 1) * (h // hk))
                lse[begin + a:begin + b, heads] = s.logsumexp(-1)
                out[begin + a:begin + b, heads] = (s.softmax(-1).reshape(-1, t - lo) @ v).reshape(b - a, h // hk, d)
        begin, pages = begin + n, pages + -(-t // page)
    return (out, lse) if case["lse"] else out
