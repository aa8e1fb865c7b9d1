"""Paged KV-cache append ops with the signatures of the flashinfer functions the reference's
attention wrapper calls (sarathi/model_executor/attention/flashinfer_attention_wrapper.py:213-226
and :262-273; flashinfer-python==0.4.1), plus the rotary-embedding + append fusion, the index
vectors of a batch built on the GPU, attention over the cache and the join of attention states.

The cache is flashinfer's NHD layout: one tensor ``[num_pages, 2, page_size, num_kv_heads,
head_size]`` (K plane, V plane) or a ``(k_cache, v_cache)`` pair of
``[num_pages, page_size, num_kv_heads, head_size]`` tensors.
"""
from typing import NamedTuple, Optional, Tuple, Union

import torch

from ._ext import C as _C

PagedCache = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _split_cache(paged_kv_cache: PagedCache, kv_layout: str):
    if kv_layout != "NHD":
        raise ValueError("only the NHD page layout is supported, got %r" % (kv_layout,))
    if isinstance(paged_kv_cache, (tuple, list)):
        k_cache, v_cache = paged_kv_cache
        return k_cache, v_cache
    if paged_kv_cache.dim() != 5 or paged_kv_cache.shape[1] != 2:
        raise ValueError("paged_kv_cache must be [num_pages, 2, page_size, num_kv_heads, head_size]")
    return paged_kv_cache[:, 0], paged_kv_cache[:, 1]


def get_seq_lens(kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor,
                 page_size: int) -> torch.Tensor:
    """Length of every request's kv sequence: full pages * page_size + entries of the last page."""
    seq_lens = torch.empty_like(kv_last_page_len)
    _C.get_seq_lens(kv_indptr, kv_last_page_len, seq_lens, page_size)
    return seq_lens


def get_batch_indices_positions(append_indptr: torch.Tensor, seq_lens: torch.Tensor,
                                nnz: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """For each of the ``nnz`` appended tokens: the request it belongs to and its index in that
    request's kv sequence (the request's last appended token is the sequence's last entry)."""
    batch_indices = torch.empty((nnz,), dtype=torch.int32, device=append_indptr.device)
    positions = torch.empty((nnz,), dtype=torch.int32, device=append_indptr.device)
    _C.get_batch_indices_positions(append_indptr, seq_lens, batch_indices, positions)
    return batch_indices, positions


def get_kv_slot_mapping(batch_indices: torch.Tensor, positions: torch.Tensor,
                        kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                        page_size: int) -> torch.Tensor:
    """``page * page_size + entry`` of every appended token.  The page table of a batch is the
    same for all layers: compute this once per batch and pass it as ``slot_mapping`` to the append
    ops, which then resolve a token's destination with one index load instead of three.  -1 for a
    token that goes nowhere: a negative request or position, or one past its request's pages."""
    slot_mapping = torch.empty_like(batch_indices)
    _C.get_kv_slot_mapping(batch_indices, positions, kv_indices, kv_indptr, slot_mapping, page_size)
    return slot_mapping


def append_paged_kv_cache(append_key: torch.Tensor, append_value: torch.Tensor,
                          batch_indices: torch.Tensor, positions: torch.Tensor,
                          paged_kv_cache: PagedCache, kv_indices: torch.Tensor,
                          kv_indptr: torch.Tensor, kv_last_page_len: Optional[torch.Tensor] = None,
                          kv_layout: str = "NHD",
                          slot_mapping: Optional[torch.Tensor] = None) -> None:
    """Copy ``append_key`` / ``append_value`` ``[nnz, num_kv_heads, head_size]`` into the cache.
    ``kv_last_page_len`` is accepted for signature compatibility; the destination of a token
    follows from ``positions`` alone."""
    k_cache, v_cache = _split_cache(paged_kv_cache, kv_layout)
    _C.append_paged_kv_cache(append_key, append_value, batch_indices, positions, k_cache, v_cache,
                             kv_indices, kv_indptr, slot_mapping)


def rotary_embedding_append_paged_kv(positions: torch.Tensor, query: torch.Tensor,
                                     key: torch.Tensor, value: torch.Tensor, head_size: int,
                                     cos_sin_cache: torch.Tensor, is_neox: bool,
                                     batch_indices: torch.Tensor, append_positions: torch.Tensor,
                                     paged_kv_cache: PagedCache, kv_indices: torch.Tensor,
                                     kv_indptr: torch.Tensor,
                                     num_append_tokens: Optional[int] = None,
                                     write_key: bool = False, kv_layout: str = "NHD",
                                     slot_mapping: Optional[torch.Tensor] = None) -> None:
    """``pos_encoding_ops.rotary_embedding(positions, query, key, ...)`` followed by
    ``append_paged_kv_cache(key[:n], value[:n], ...)`` in one launch (n = ``num_append_tokens``,
    default all tokens).  ``query`` is rotated in place; the rotated keys go to the cache and, only
    with ``write_key=True``, also back into ``key``."""
    k_cache, v_cache = _split_cache(paged_kv_cache, kv_layout)
    n = positions.shape[0] if num_append_tokens is None else int(num_append_tokens)
    _C.rotary_embedding_append_paged_kv(positions, query, key, value, head_size, cos_sin_cache,
                                        is_neox, batch_indices, append_positions, k_cache, v_cache,
                                        kv_indices, kv_indptr, n, write_key, slot_mapping)


class PagedKvMetadata(NamedTuple):
    """What ``build_paged_kv_metadata`` returns; the names of the append's and the attention's
    arguments.  int32 but for ``rope_positions``."""
    qo_indptr: torch.Tensor         # [num_seqs + 1] start of each sequence's new tokens
    kv_indptr: torch.Tensor         # [num_seqs + 1] start of each sequence's pages
    kv_indices: torch.Tensor        # [num_kv_pages] used pages of all sequences in a row, then -1
    kv_last_page_len: torch.Tensor  # [num_seqs]
    batch_indices: torch.Tensor     # [num_tokens] sequence of every new token
    positions: torch.Tensor         # [num_tokens] its index in the sequence
    slot_mapping: torch.Tensor      # [num_tokens] page * page_size + entry
    rope_positions: torch.Tensor    # [num_tokens] int64, for the rotary embedding


def build_paged_kv_metadata(query_lens: torch.Tensor, seq_lens: torch.Tensor,
                            block_tables: torch.Tensor, page_size: int, num_tokens: int,
                            num_kv_pages: Optional[int] = None) -> PagedKvMetadata:
    """The index vectors of a batch from lengths that live on the GPU, without a copy or a
    synchronisation: the device-side counterpart of FlashinferAttentionWrapper.begin_forward's
    bookkeeping (sarathi/model_executor/attention/flashinfer_attention_wrapper.py:84-229).

    ``query_lens`` / ``seq_lens`` int32 ``[num_seqs]``: new tokens, and tokens in all after the
    append.  ``block_tables`` int32 ``[num_seqs, max_pages]``: each sequence's pages in order;
    entries past ``ceil(seq_len / page_size)`` are not read.  ``num_tokens`` and ``num_kv_pages``
    (default: the size of ``block_tables``, which every batch fits) are the lengths of the per-token
    vectors and of ``kv_indices``, and have to hold the batch's new tokens and used pages: requests that
    do not fit are not served (nothing outside the vectors is touched, but attention sees them without
    what was cut off, and their tokens past it are appended only by ``slot_mapping``).  Room beyond
    the batch, as a captured graph needs, is filled with -1 (``rope_positions``: 0), and the append ops
    skip negative slots and positions."""
    if num_kv_pages is None:
        num_kv_pages = block_tables.numel()
    return PagedKvMetadata._make(_C.build_paged_kv_metadata(query_lens, seq_lens, block_tables, page_size,
                                                            num_tokens, num_kv_pages))


def paged_attention(query: torch.Tensor, paged_kv_cache: PagedCache, qo_indptr: torch.Tensor,
                    kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                    kv_last_page_len: torch.Tensor, sm_scale: Optional[float] = None,
                    causal: bool = True, window_left: int = -1,
                    max_query_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, kv_layout: str = "NHD"):
    """Attention of a batch's new tokens over their sequences in the cache, prompt chunks and single
    decode tokens in one call (the two wrappers that the reference plans and runs at
    sarathi/model_executor/attention/flashinfer_attention_wrapper.py:169-209 and :275-304).

    ``query`` ``[num_tokens, num_heads, head_size]`` (or 2-D rows, possibly a view of a packed qkv
    buffer), bfloat16 or float16; the tokens of request r are ``[qo_indptr[r], qo_indptr[r + 1])``
    and are the last ones of its sequence, whose keys the four kv vectors describe as for the append.
    With ``causal`` a token sees the keys up to its own, with ``window_left >= 0`` only that many
    before it.  ``sm_scale``, positive, defaults to ``head_size ** -0.5``.  ``max_query_len``, where the caller
    knows an upper bound of the requests' new tokens, picks the kernel (1: a pure decode batch).

    Returns ``out`` (shaped like ``query``), with ``return_lse`` also the natural-log sums
    ``[num_tokens, num_heads]`` (float32) that ``merge_attention_states`` joins.  A token that sees no
    key gets 0 and -inf, and so do rows behind the last request, except that those of an ``out`` that
    was passed in are left as they were.  ``out`` must not overlap ``query`` or the cache.  A value that
    a mask hides from some of a request's tokens only must be finite.
    No gradients: inputs that require one are refused unless gradients are switched off."""
    if kv_layout != "NHD":
        raise ValueError("only the NHD page layout is supported, got %r" % (kv_layout,))
    if isinstance(paged_kv_cache, (tuple, list)):
        k_cache, v_cache = paged_kv_cache
    else:
        k_cache, v_cache = paged_kv_cache, None
    result = _C.paged_attention(query, k_cache, v_cache, qo_indptr, kv_indptr, kv_indices, kv_last_page_len,
                                out, return_lse, sm_scale, causal, window_left,
                                0 if max_query_len is None else max_query_len)
    return tuple(result) if return_lse else result[0]


def merge_attention_states(v: torch.Tensor, lse: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Joins ``paged_attention`` states over disjoint parts of a context, e.g. a prefix that requests
    share and each request's own suffix: ``v`` ``[states, tokens, heads, head_size]``, ``lse``
    ``[states, tokens, heads]`` (natural log, float32).  The state and token dimensions may have any
    strides.  Returns the joined output and its lse; states with lse -inf are left out.  No gradients:
    inputs that require one are refused unless gradients are switched off."""
    out, out_lse = _C.merge_attention_states(v, lse)
    return out, out_lse


__all__ = ["get_seq_lens", "get_batch_indices_positions", "get_kv_slot_mapping", "append_paged_kv_cache",
           "rotary_embedding_append_paged_kv", "PagedKvMetadata", "build_paged_kv_metadata",
           "paged_attention", "merge_attention_states"]
