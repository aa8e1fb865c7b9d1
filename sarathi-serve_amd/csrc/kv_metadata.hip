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
// The work is a sum over the requests in front of one's own and then one lookup per token and per
// page; what bounds it is latency, then the bytes of the page table.  Up to kMetaOneLaunch requests it
// is ONE launch of independent workgroups, each of one request (or of a piece of a long one): it adds
// up the lengths of the requests before its own (all of them come out of L2), and then its tokens and
// pages lie side by side, so nothing is searched for.  The additions grow with the square of the
// requests; beyond the limit one workgroup writes the prefix sums first.  Measured: 16 decodes 4.4 us,
// eight chunks and 1000 decodes with tables of up to 2048 pages 6.8 us, an empty launch 1.6 of them;
// the call costs 8 us of host time (eight tensors out of one allocation).
#include "launch.h"
#include "vec16.h"

namespace sarathi_hip {

constexpr int kMetaOneLaunch = 4096;
constexpr int kMetaPiece = 2048;  // tokens or pages of a request that one workgroup takes
constexpr int kMetaFill = 16;     // workgroups that fill the room behind the batch

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
  uint32_t pieces;                 // workgroups per request
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

// Sums over the workgroup's 256 threads; every thread returns them.
SK_DEV void meta_block_sum(int64_t& q, int64_t& p) {
  __shared__ int64_t sums[4][2];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    q += __shfl_xor(q, d, 64);
    p += __shfl_xor(p, d, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6][0] = q;
    sums[threadIdx.x >> 6][1] = p;
  }
  __syncthreads();
  q = (sums[0][0] + sums[1][0]) + (sums[2][0] + sums[3][0]);
  p = (sums[0][1] + sums[1][1]) + (sums[2][1] + sums[3][1]);
}

// SCANNED: the prefix sums are in qo_indptr / kv_indptr already.
template <bool SCANNED>
__global__ __launch_bounds__(256) void kv_metadata_kernel(KvMetaArgs a) {
  const int tid = threadIdx.x;
  const int64_t work = (int64_t)a.seqs * a.pieces;
  const bool fill = (int64_t)blockIdx.x >= work;
  const int32_t r = fill ? a.seqs : (int32_t)(blockIdx.x / a.pieces);
  const int32_t piece = fill ? 0 : (int32_t)(blockIdx.x - (uint32_t)r * a.pieces);
  int32_t n = 0, pages = 0;
  if (!fill) {
    n = meta_new(a, r);
    pages = meta_pages(a, r);
    if (piece > 0 && (int64_t)piece * kMetaPiece >= (n > pages ? n : pages)) return;
  }
  int64_t q = 0, p = 0;
  if constexpr (SCANNED) {
    q = a.qo_indptr[r];
    p = a.kv_indptr[r];
  } else {
    for (int32_t i = tid; i < r; i += 256) {
      q += meta_new(a, i);
      p += meta_pages(a, i);
    }
    meta_block_sum(q, p);
    if (tid == 0 && piece == 0) {
      if (!fill) meta_write_request(a, r, q, p);
      else if ((int64_t)blockIdx.x == work) meta_write_request(a, a.seqs, q, p);
    }
  }
  if (fill) {  // behind the batch
    const int64_t at = ((int64_t)blockIdx.x - work) * 256 + tid, step = (int64_t)kMetaFill * 256;
    for (int64_t i = q + at; i < a.num_tokens; i += step) {
      a.batch_indices[i] = -1;
      a.positions[i] = -1;
      a.slots[i] = -1;
      a.rope_positions[i] = 0;
    }
    for (int64_t i = p + at; i < a.num_pages; i += step) a.kv_indices[i] = -1;
    return;
  }
  const int32_t* const table = a.tables + (int64_t)r * a.table_stride;
  const int64_t before = (int64_t)a.seq_lens[r] - n;  // position of the first new token
  const int64_t most = n > pages ? n : pages, stride = (int64_t)a.pieces * kMetaPiece;
  for (int64_t j0 = (int64_t)piece * kMetaPiece; j0 < most; j0 += stride) {
#pragma unroll 4
    for (int k = 0; k < kMetaPiece / 256; ++k) {
      const int64_t j = j0 + k * 256 + tid;
      if (j < pages && p + j < a.num_pages) a.kv_indices[p + j] = table[j];
    }
    for (int k = 0; k < kMetaPiece / 256; ++k) {
      const int64_t j = j0 + k * 256 + tid;
      if (j >= n || q + j >= a.num_tokens) break;
      const int64_t at = before + j;
      const int64_t pg = at >= 0 ? (int64_t)((uint32_t)at / (uint32_t)a.page_size) : 0;
      int32_t pos = -1, slot = -1;
      if (at >= 0 && pg < pages) {
        pos = (int32_t)at;
        const int32_t page = table[pg];
        if (page >= 0) slot = page * a.page_size + (pos - (int32_t)pg * a.page_size);
      }
      a.batch_indices[q + j] = r;
      a.positions[q + j] = pos;
      a.slots[q + j] = slot;
      a.rope_positions[q + j] = pos >= 0 ? pos : 0;
    }
  }
}

__global__ __launch_bounds__(256) void kv_metadata_scan_kernel(KvMetaArgs a) {
  meta_scan(a, [&](int32_t r, int64_t q, int64_t p) { meta_write_request(a, r, q, p); });
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
  // pieces of the longest request there can be, while the requests alone are few workgroups
  const int64_t longest = num_tokens > max_pages_per_seq ? num_tokens : max_pages_per_seq;
  int64_t pieces = (longest + kMetaPiece - 1) / kMetaPiece;
  if (pieces > 1024 / (num_seqs + 1)) pieces = 1024 / (num_seqs + 1);
  if (pieces < 1) pieces = 1;
  const int64_t groups = num_seqs * pieces + kMetaFill;
  if (groups > 0x7fffffffLL) return SARATHI_ERR_UNSUPPORTED;
  KvMetaArgs a{query_lens,    seq_lens,          block_tables,      qo_indptr,
               kv_indptr,     kv_indices,        kv_last_page_len,  batch_indices,
               positions,     slot_mapping,      rope_positions,    table_stride,
               (int32_t)num_seqs, (int32_t)max_pages_per_seq, (int32_t)page_size,
               num_tokens,    num_kv_pages,      (uint32_t)pieces};
  hipStream_t st = (hipStream_t)stream;
  if (num_seqs <= kMetaOneLaunch) {
    hipLaunchKernelGGL((kv_metadata_kernel<false>), dim3((unsigned)groups), dim3(256), 0, st, a);
    return launch_status();
  }
  hipLaunchKernelGGL(kv_metadata_scan_kernel, dim3(1), dim3(256), 0, st, a);
  hipLaunchKernelGGL((kv_metadata_kernel<true>), dim3((unsigned)groups), dim3(256), 0, st, a);
  return launch_status();
}
