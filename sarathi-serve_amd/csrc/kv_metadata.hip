// Index vectors of a hybrid batch over a paged KV cache, built on the GPU from the requests'
// lengths: what FlashinferAttentionWrapper.begin_forward collects with host loops and copies
// (sarathi/model_executor/attention/flashinfer_attention_wrapper.py:84-229).
//
// With n_r new tokens, s_r tokens in all and a dense table of pages per request, of which
// p_r = ceil(s_r / page_size) are in use:
//   qo_indptr = exclusive prefix sums of n, kv_indptr = those of p,
//   kv_indices = the used pages of all requests in a row,
//   last_page_len[r] = s_r - (p_r - 1) * page_size,
//   and for the j-th new token of request r: batch index r, position s_r - n_r + j, the slot
//   page * page_size + entry of that position, and the position again as the rotary embedding's
//   64-bit index.
//
// The work is a prefix sum over the requests and then one lookup per token and per page: a few
// hundred KiB at the most, so what bounds it is latency.  Up to kMetaLdsSeqs requests it is ONE
// launch of independent workgroups: each of them adds up all the lengths itself (they come out of
// L2; 1008 requests cost about a microsecond), keeps both prefix arrays in LDS and looks its own
// tokens and pages up there.  More requests take two launches, a scan by one workgroup and then
// the lookups against the prefix arrays in global memory.
#include "launch.h"
#include "vec16.h"

namespace sarathi_hip {

constexpr int kMetaLdsSeqs = 4096;   // two prefix arrays of 16 KiB
constexpr int kMetaPerThread = 4;    // tokens or pages a thread looks up

struct KvMetaArgs {
  const int32_t* query_lens;
  const int32_t* seq_lens;
  const int32_t* tables;
  int32_t *qo_indptr, *kv_indptr, *kv_indices, *last_page_len;
  int32_t *batch_indices, *positions, *slots;
  int64_t* rope_positions;
  int64_t table_stride;   // entries between the rows of the table
  int32_t seqs, max_pages, page_size;
  int64_t num_tokens, num_pages;   // room in the per-token vectors, resp. in kv_indices
  uint32_t token_groups;           // workgroups that work on tokens; the others work on pages
};

SK_DEV int32_t meta_new(const KvMetaArgs& a, int32_t r) {
  const int32_t n = a.query_lens[r];
  return n > 0 ? n : 0;
}
// pages of request r in use, never more than its row of the table holds
SK_DEV int32_t meta_pages(const KvMetaArgs& a, int32_t r) {
  const int32_t s = a.seq_lens[r];
  if (s <= 0) return 0;
  const int32_t p = (int32_t)(((uint32_t)s + (uint32_t)a.page_size - 1u) / (uint32_t)a.page_size);
  return p < a.max_pages ? p : a.max_pages;
}
SK_DEV int32_t meta_clip(int64_t v, int64_t most) { return (int32_t)(v < most ? v : most); }

// Exclusive prefix sums of both lengths over all requests by one workgroup of 256, each thread a
// run of consecutive requests; emit(r, tokens before r, pages before r) for every r in [0, seqs].
// The sums are held in 64 bits: they may pass 32 bits where the lengths are not a batch's.
template <typename F> SK_DEV void meta_scan(const KvMetaArgs& a, F emit) {
  __shared__ int64_t wave_q[4], wave_p[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t run = (a.seqs + 255) / 256;
  const int64_t first = (int64_t)tid * run;
  const int32_t r0 = first < a.seqs ? (int32_t)first : a.seqs;
  const int32_t r1 = first + run < a.seqs ? (int32_t)(first + run) : a.seqs;
  int64_t q = 0, p = 0;
  for (int32_t r = r0; r < r1; ++r) {
    q += meta_new(a, r);
    p += meta_pages(a, r);
  }
  const int64_t my_q = q, my_p = p;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t uq = __shfl_up(q, d, 64), up = __shfl_up(p, d, 64);
    if (lane >= d) {
      q += uq;
      p += up;
    }
  }
  if (lane == 63) {
    wave_q[wave] = q;
    wave_p[wave] = p;
  }
  __syncthreads();
  q -= my_q;
  p -= my_p;
  for (int w = 0; w < wave; ++w) {
    q += wave_q[w];
    p += wave_p[w];
  }
  for (int32_t r = r0; r < r1; ++r) {
    emit(r, q, p);
    q += meta_new(a, r);
    p += meta_pages(a, r);
  }
  if (tid == 255) emit(a.seqs, q, p);  // the last thread's sums run over everything
}

// The prefix arrays and the per-request vector, written by one workgroup.
SK_DEV void meta_write_request(const KvMetaArgs& a, int32_t r, int64_t q, int64_t p) {
  a.qo_indptr[r] = meta_clip(q, a.num_tokens);
  a.kv_indptr[r] = meta_clip(p, a.num_pages);
  if (r == a.seqs) return;
  const int32_t pages = meta_pages(a, r);
  int32_t last = 0;
  if (pages > 0) {
    const int64_t in_last = (int64_t)a.seq_lens[r] - (int64_t)(pages - 1) * a.page_size;
    last = meta_clip(in_last, a.page_size);  // a sequence longer than its row of the table: full
  }
  a.last_page_len[r] = last;
}

// The request whose range of `starts` holds i: starts[lo] <= i < starts[hi].  Empty requests
// (repeated entries) are stepped over.  i lies below starts[seqs].
SK_DEV int32_t meta_find(const int32_t* starts, int32_t seqs, int64_t i) {
  int32_t lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int32_t mid = (int32_t)(((uint32_t)lo + (uint32_t)hi) >> 1);
    if (starts[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

SK_DEV void meta_lookups(const KvMetaArgs& a, const int32_t* qo, const int32_t* kv) {
  const bool is_token = blockIdx.x < a.token_groups;  // uniform over the workgroup
  const int64_t group = is_token ? blockIdx.x : blockIdx.x - a.token_groups;
  const int64_t base = group * (256 * kMetaPerThread) + threadIdx.x;
  if (is_token) {
    const int32_t total = qo[a.seqs];
#pragma unroll
    for (int k = 0; k < kMetaPerThread; ++k) {
      const int64_t i = base + k * 256;
      if (i >= a.num_tokens) break;
      int32_t b = -1, pos = -1, slot = -1;
      if (i < total) {
        b = meta_find(qo, a.seqs, i);
        const int64_t at = (int64_t)a.seq_lens[b] - meta_new(a, b) + (i - qo[b]);
        const int32_t pg = at >= 0 ? (int32_t)((uint32_t)at / (uint32_t)a.page_size) : 0;
        if (at >= 0 && pg < meta_pages(a, b)) {
          pos = (int32_t)at;
          const int32_t page = a.tables[(int64_t)b * a.table_stride + pg];
          if (page >= 0) slot = page * a.page_size + (pos - pg * a.page_size);
        }
      }
      a.batch_indices[i] = b;
      a.positions[i] = pos;
      a.slots[i] = slot;
      a.rope_positions[i] = pos >= 0 ? pos : 0;
    }
    return;
  }
  const int32_t total = kv[a.seqs];
#pragma unroll
  for (int k = 0; k < kMetaPerThread; ++k) {
    const int64_t i = base + k * 256;
    if (i >= a.num_pages) break;
    int32_t page = -1;
    if (i < total) {
      const int32_t r = meta_find(kv, a.seqs, i);
      page = a.tables[(int64_t)r * a.table_stride + (i - kv[r])];
    }
    a.kv_indices[i] = page;
  }
}

__global__ __launch_bounds__(256) void kv_metadata_kernel(KvMetaArgs a) {
  extern __shared__ int32_t meta_lds[];  // two prefix arrays of seqs + 1 entries
  int32_t* const qo = meta_lds;
  int32_t* const kv = meta_lds + a.seqs + 1;
  const bool writer = blockIdx.x == 0;
  meta_scan(a, [&](int32_t r, int64_t q, int64_t p) {
    qo[r] = meta_clip(q, a.num_tokens);
    kv[r] = meta_clip(p, a.num_pages);
    if (writer) meta_write_request(a, r, q, p);
  });
  __syncthreads();
  meta_lookups(a, qo, kv);
}

__global__ __launch_bounds__(256) void kv_metadata_scan_kernel(KvMetaArgs a) {
  meta_scan(a, [&](int32_t r, int64_t q, int64_t p) { meta_write_request(a, r, q, p); });
}
__global__ __launch_bounds__(256) void kv_metadata_lookup_kernel(KvMetaArgs a) {
  meta_lookups(a, a.qo_indptr, a.kv_indptr);
}

}  // namespace sarathi_hip

using namespace sarathi_hip;

extern "C" int sarathi_build_paged_kv_metadata(
    const int32_t* query_lens, const int32_t* seq_lens, const int32_t* block_tables,
    int32_t* qo_indptr, int32_t* kv_indptr, int32_t* kv_indices, int32_t* kv_last_page_len,
    int32_t* batch_indices, int32_t* positions, int32_t* slot_mapping, int64_t* rope_positions,
    int64_t num_seqs, int64_t max_pages_per_seq, int64_t table_stride, int page_size,
    int64_t num_tokens, int64_t num_kv_pages, void* stream) {
  if (num_seqs < 0 || max_pages_per_seq < 0 || page_size <= 0 || num_tokens < 0 ||
      num_kv_pages < 0 || table_stride < max_pages_per_seq || !qo_indptr || !kv_indptr)
    return SARATHI_ERR_INVALID_ARG;
  if (num_seqs > 0 && (!query_lens || !seq_lens || !kv_last_page_len ||
                       (max_pages_per_seq > 0 && !block_tables)))
    return SARATHI_ERR_INVALID_ARG;
  if ((num_tokens > 0 && (!batch_indices || !positions || !slot_mapping || !rope_positions)) ||
      (num_kv_pages > 0 && !kv_indices))
    return SARATHI_ERR_INVALID_ARG;
  if (num_seqs >= 0x7fffffffLL || num_tokens >= 0x7fffffffLL || num_kv_pages >= 0x7fffffffLL ||
      max_pages_per_seq >= 0x7fffffffLL)
    return SARATHI_ERR_UNSUPPORTED;
  const int64_t per_group = 256 * kMetaPerThread;
  const int64_t tok_groups = (num_tokens + per_group - 1) / per_group;
  const int64_t groups = tok_groups + (num_kv_pages + per_group - 1) / per_group;
  KvMetaArgs a{query_lens,    seq_lens,          block_tables,      qo_indptr,
               kv_indptr,     kv_indices,        kv_last_page_len,  batch_indices,
               positions,     slot_mapping,      rope_positions,    table_stride,
               (int32_t)num_seqs, (int32_t)max_pages_per_seq, (int32_t)page_size,
               num_tokens,    num_kv_pages,      (uint32_t)tok_groups};
  hipStream_t st = (hipStream_t)stream;
  if (num_seqs <= kMetaLdsSeqs) {
    hipLaunchKernelGGL(kv_metadata_kernel, dim3((unsigned)(groups > 0 ? groups : 1)), dim3(256),
                       (unsigned)(2 * (num_seqs + 1) * sizeof(int32_t)), st, a);
    return launch_status();
  }
  hipLaunchKernelGGL(kv_metadata_scan_kernel, dim3(1), dim3(256), 0, st, a);
  if (groups > 0)
    hipLaunchKernelGGL(kv_metadata_lookup_kernel, dim3((unsigned)groups), dim3(256), 0, st, a);
  return launch_status();
}
