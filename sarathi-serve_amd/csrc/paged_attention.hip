// Attention of the new tokens of a hybrid batch over their requests' pages (paged_attn.h has the
// formulas).  Stands for the two flashinfer wrappers that the reference plans and runs per batch
// (sarathi/model_executor/attention/flashinfer_attention_wrapper.py:169-209, 262-304): one entry
// for chunks of new tokens and for single decode tokens alike.
//
// This file holds the entry point, the plan of a launch, the plain kernel for any head size and
// alignment and the kernel that joins the parts of a cut context; the matrix-core kernels are in
// paged_attention_few.hip and paged_attention_mixed_*.hip.
#include "launch.h"
#include "paged_attn.h"
#include "paged_attn_launch.h"

namespace sarathi_hip {

// ---- any head size, any alignment: one wave per token and query head ---------------------------
//
// 64 keys at a time: every lane takes one key's whole dot product, the wave agrees on the maximum,
// and then every lane owns the head's elements lane, lane + 64, ...  Everything in 32 bits.  It is
// the form that is right for every shape; it runs where the vector kernels cannot (heads or strides
// that are no multiple of 16 bytes).
template <int DT>
__global__ __launch_bounds__(64) void paged_attn_plain_kernel(PagedAttnArgs a) {
  __shared__ float qrow[kAttnMaxHead];
  __shared__ float prob[64];
  const int lane = threadIdx.x;
  const int32_t tok = (int32_t)blockIdx.x, head = (int32_t)blockIdx.y;
  if (a.seqs == 0 || tok >= clamp_i32(a.qo_indptr[a.seqs], 0, a.tokens) || tok < a.qo_indptr[0]) {
    const int64_t row = (int64_t)tok * a.out_stride + (int64_t)head * a.head_size;
    if (a.fill & 2)
      for (int d = lane; d < a.head_size; d += 64) store_elem<DT>(a.out, row + d, 0.f);
    if ((a.fill & 1) && lane == 0) a.lse[(int64_t)tok * a.heads + head] = -INFINITY;
    return;
  }
  int32_t lo_r = 0, hi_r = a.seqs;
  while (hi_r - lo_r > 1) {
    const int32_t mid = (lo_r + hi_r) >> 1;
    if (a.qo_indptr[mid] <= tok) lo_r = mid; else hi_r = mid;
  }
  const AttnSeq x = attn_seq(a, lo_r);
  if (tok < x.q0 || tok >= x.q0 + x.n) return;
  int32_t lo, hi;
  attn_span(a, x, tok - x.q0, lo, hi);
  const int D = a.head_size;
  const int64_t kv_head = (int64_t)(head / a.group) * D;
  const int64_t qbase = (int64_t)tok * a.q_stride + (int64_t)head * D;
  for (int d = lane; d < D; d += 64) qrow[d] = load_elem<DT>(a.q, qbase + d);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[kAttnMaxHead / 64] = {};
  for (int32_t t0 = lo; t0 < hi; t0 += 64) {
    const int32_t t = t0 + lane;
    float s = -INFINITY;
    if (t < hi) {
      const char* k = reinterpret_cast<const char*>(a.k_cache) + attn_entry(a, x, t);
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(qrow[d], load_elem<DT>(k, kv_head + d), dot);
      s = dot * a.scale_log2;
    }
    const float top = fmaxf(m, wave64_max(s));
    const float ref = top == -INFINITY ? 0.f : top;
    const float p = t < hi ? __builtin_amdgcn_exp2f(s - ref) : 0.f;
    const float keep = __builtin_amdgcn_exp2f(m - ref);
    l = l * keep + p;
    m = top;
    __syncthreads();
    prob[lane] = p;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAttnMaxHead / 64; ++i) o[i] *= keep;
    const int32_t cnt = hi - t0 < 64 ? hi - t0 : 64;
    for (int32_t j = 0; j < cnt; ++j) {
      const char* v = reinterpret_cast<const char*>(a.v_cache) + attn_entry(a, x, t0 + j);
#pragma unroll
      for (int i = 0; i < kAttnMaxHead / 64; ++i) {
        const int d = lane + 64 * i;
        if (d < D) o[i] = fmaf(prob[j], load_elem<DT>(v, kv_head + d), o[i]);
      }
    }
  }
  l = wave64_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t obase = (int64_t)tok * a.out_stride + (int64_t)head * D;
#pragma unroll
  for (int i = 0; i < kAttnMaxHead / 64; ++i) {
    const int d = lane + 64 * i;
    if (d < D) store_elem<DT>(a.out, obase + d, o[i] * inv);
  }
  if (a.lse && lane == 0) a.lse[(int64_t)tok * a.heads + head] = attn_lse(m, l);
}

// ---- joins the parts of cut contexts -------------------------------------------------------------
//
// WPT waves per token and four query heads of a key head: sixteen where there are few tokens (a
// workgroup of their own), else one (four tokens in a workgroup).  Half-waves of 32 lanes share the
// rows and their parts: with few rows several take turns at one row's parts, and each has eight of them on
// their way at once, so that the time hardly grows with the parts.  A part whose sum is zero has no
// output.  Parts are added in a fixed order: results do not depend on which workgroup ran when.
// Nothing to join (the attention kernel leaves word) costs a launch and one load.  Bound by latency: 4 to
// 7 us from one request to 256, of which up to 4 hide behind the kernel before.
constexpr int kJoinRows = 4;

template <int DT, int VALS, int WPT>  // VALS elements of the head per lane
__global__ __launch_bounds__(WPT == 1 ? 256 : WPT * 64) void paged_attn_join_kernel(PagedAttnArgs a) {
  constexpr int U = 2 * WPT;  // half-waves of a token
  typedef float vals_t __attribute__((ext_vector_type(VALS)));
  __shared__ float box[WPT == 1 ? 1 : WPT][32 * VALS + 2];
  const int lane = threadIdx.x & 63, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = WPT == 1 ? lane >> 5 : (int)threadIdx.x >> 5;
  const int32_t tok = (int32_t)blockIdx.x * (WPT == 1 ? 4 : 1) + (WPT == 1 ? wave : 0);
  const int32_t quads = (a.group + kJoinRows - 1) / kJoinRows;
  const int32_t h = (int32_t)blockIdx.y / quads, g_first = ((int32_t)blockIdx.y - h * quads) * kJoinRows;
  const int32_t g_end = g_first + kJoinRows < a.group ? g_first + kJoinRows : a.group;
  // one trip to memory for everything, where 64 lanes hold all requests
  const bool small = a.seqs < 64;
  const int32_t any = a.part_map[2 * a.seqs];
  const int32_t li = lane <= a.seqs ? lane : a.seqs, lr = lane < a.seqs ? lane : a.seqs - 1;
  int32_t qo_l = 0, row_l = 0, parts_l = 0;
  if (small) {
    qo_l = a.qo_indptr[li];
    row_l = a.part_map[lr];
    parts_l = a.part_map[a.seqs + lr];
  }
  if (any == 0 || tok >= a.tokens) return;
  // request of the token, the last whose first token is not past it
  int32_t r = 0, parts, first_row, q0, n;
  if (small) {
    const int cnt = __popcll(__builtin_amdgcn_ballot_w64(lane < a.seqs && qo_l <= tok));
    if (cnt == 0) return;  // before the first request
    r = cnt - 1;
    parts = __builtin_amdgcn_readlane(parts_l, r);
    first_row = __builtin_amdgcn_readlane(row_l, r);
    q0 = clamp_i32(__builtin_amdgcn_readlane(qo_l, r), 0, a.tokens);
    n = clamp_i32(__builtin_amdgcn_readlane(qo_l, r + 1), q0, a.tokens) - q0;
  } else {
    int32_t width = a.seqs;
    while (true) {  // 64 candidates at a time
      const int32_t step = (width + 63) / 64;
      const bool ok = lane * step < width && a.qo_indptr[r + lane * step] <= tok;
      const int cnt = __popcll(__builtin_amdgcn_ballot_w64(ok));
      if (cnt == 0) return;
      r += (cnt - 1) * step;
      if (step == 1) break;
      width = width - (cnt - 1) * step < step ? width - (cnt - 1) * step : step;
    }
    r = __builtin_amdgcn_readfirstlane(r);
    parts = a.part_map[a.seqs + r];
    first_row = a.part_map[r];
    q0 = clamp_i32(a.qo_indptr[r], 0, a.tokens);
    n = clamp_i32(a.qo_indptr[r + 1], q0, a.tokens) - q0;
  }
  if (parts <= 1 || tok < q0 || tok >= q0 + n) return;
  const int64_t rows_all = (int64_t)n * a.group;
  const bool tiled = a.few.rows_log2 < 0 || (a.tile.rows_log2 >= 0 && rows_all > a.few.max_rows);
  const int32_t lg = tiled ? a.tile.rows_log2 : a.few.rows_log2;
  int share = U;  // half-waves per row
  while (share > 1 && U / share < g_end - g_first) share >>= 1;
  const int rows_at_once = U / share;
  const int d0 = l32 * VALS;
  const bool on = d0 < a.head_size;
  for (int32_t g0 = g_first; g0 < g_end; g0 += rows_at_once) {
    const int32_t gq = g0 + unit / share;
    const bool live = gq < g_end;
    const int32_t row = (tok - q0) * a.group + (live ? gq : g_first);
    const int32_t tile = row >> lg, in_tile = row & ((1 << lg) - 1);
    const int64_t row0 = first_row + ((int64_t)(tile * parts * a.kv_heads + h) << lg) + in_tile;
    const int64_t per_part = (int64_t)a.kv_heads << lg;
    float ref = kRefStart, l = 0.f;
    vals_t o = 0.f;
    for (int32_t p0 = unit % share; p0 < parts; p0 += 8 * share) {
      f32x2 ml[8];
      vals_t po[8];
      float pr[8], pl[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int32_t p = p0 + i * share;
        const int64_t at = row0 + (p < parts ? p : parts - 1) * per_part;
        ml[i] = *reinterpret_cast<const f32x2*>(a.part_ml + at * 2);
        // heads are multiples of 8 elements: whole vectors; lanes past the head read its first
        po[i] = *reinterpret_cast<const vals_t*>(a.part_o + at * a.head_size + (on ? d0 : 0));
      }
      __builtin_amdgcn_sched_barrier(0);  // every load is issued before anything waits
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        pr[i] = ml[i].x;
        pl[i] = p0 + i * share < parts ? ml[i].y : 0.f;
      }
      float top = ref;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = pl[i] != 0.f ? fmaxf(top, pr[i]) : top;
      const float keep = __builtin_amdgcn_exp2f(ref - top);
      ref = top;
      l *= keep;
      o *= keep;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = pl[i] != 0.f ? __builtin_amdgcn_exp2f(pr[i] - ref) : 0.f;
        l += pl[i] * w;
#pragma unroll
        for (int v = 0; v < VALS; ++v) {
          const float x = po[i][v];
          o[v] = pl[i] != 0.f ? fmaf(x, w, o[v]) : o[v];
        }
      }
    }
    if (share > 1) {  // the two halves of a wave have the same row
      const float ref2 = __shfl_xor(ref, 32, 64), l2 = __shfl_xor(l, 32, 64);
      const float top = fmaxf(ref, ref2);
      const float w1 = __builtin_amdgcn_exp2f(ref - top), w2 = __builtin_amdgcn_exp2f(ref2 - top);
      l = l * w1 + l2 * w2;
#pragma unroll
      for (int v = 0; v < VALS; ++v) {
        const float x = o[v];
        o[v] = x * w1 + __shfl_xor(x, 32, 64) * w2;
      }
      ref = top;
    }
    if constexpr (WPT > 1) {
      if (share > 2) {  // uniform over the workgroup
        __syncthreads();  // the last round's boxes are read
        if (lane < 32) {
          box[wave][32 * VALS] = ref;
          box[wave][32 * VALS + 1] = l;
#pragma unroll
          for (int v = 0; v < VALS; ++v) box[wave][d0 + v] = o[v];
        }
        __syncthreads();
        if (unit % share == 0) {
          float top = kRefStart;
          for (int s = 0; s < share / 2; ++s) top = fmaxf(top, box[wave + s][32 * VALS]);
          l = 0.f;
          o = 0.f;
          for (int s = 0; s < share / 2; ++s) {
            const float w = __builtin_amdgcn_exp2f(box[wave + s][32 * VALS] - top);
            l += box[wave + s][32 * VALS + 1] * w;
#pragma unroll
            for (int v = 0; v < VALS; ++v) o[v] += box[wave + s][d0 + v] * w;
          }
          ref = top;
        }
      }
    }
    if (unit % share != 0 || !live) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int32_t head = h * a.group + gq;
    if (on) {
      const int64_t base = (int64_t)tok * a.out_stride + (int64_t)head * a.head_size + d0;
#pragma unroll
      for (int v = 0; v < VALS; v += 2) {
        const float x = o[v], y = o[v + 1];
        *reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(a.out) + (base + v) * 2) = pack2<DT>(x * inv, y * inv);
      }
    }
    if (a.lse && l32 == 0) a.lse[(int64_t)tok * a.heads + head] = attn_lse(ref, l);
  }
}

template <int DT, int VALS> static int launch_join_head(const PagedAttnArgs& a, hipStream_t st) {
  // sixteen waves per token while that leaves the GPU room
  const unsigned heads4 = (unsigned)(a.kv_heads * ((a.group + kJoinRows - 1) / kJoinRows));
  if ((int64_t)a.tokens * heads4 <= 2 * compute_units())
    hipLaunchKernelGGL((paged_attn_join_kernel<DT, VALS, 16>), dim3((unsigned)a.tokens, heads4),
                       dim3(1024), 0, st, a);
  else
    hipLaunchKernelGGL((paged_attn_join_kernel<DT, VALS, 1>), dim3((unsigned)((a.tokens + 3) / 4), heads4),
                       dim3(256), 0, st, a);
  return launch_status();
}
template <int DT> static int launch_join(const PagedAttnArgs& a, hipStream_t st) {
  if (a.head_size <= 64) return launch_join_head<DT, 2>(a, st);
  if (a.head_size <= 128) return launch_join_head<DT, 4>(a, st);
  return launch_join_head<DT, 8>(a, st);
}

// ---- plans batches of many requests ---------------------------------------------------------------
//
// One workgroup, bound by latency: a run of requests per thread, three times over.
__global__ __launch_bounds__(1024) void paged_attn_plan_kernel(PagedAttnArgs a) {
  attn_find_item<16, true>(a, 0, a.part_map != nullptr);
}

// ---- what a call launches ------------------------------------------------------------------------

// The requests of a batch fall into two classes by their rows (new tokens times query heads per key
// head): few rows, and chunks, which are taken in large tiles.  All sizes here are known on the host.
struct AttnPlan {
  AttnClass few, tile;
  int64_t state_room;  // rows of states per key head
  int64_t items;       // at most so many work items per key head, with contexts cut and without
  int64_t uncut_items;
  int64_t plan_bytes;                    // of the workspace; 0: workgroups look at all requests
  int64_t map_bytes, ml_bytes, o_bytes;  // 0: nothing is cut
  int64_t bytes() const { return plan_bytes + map_bytes + ml_bytes + o_bytes; }
};
constexpr int kPlanSeqs = 512;   // two per thread of a workgroup
constexpr int kFillGroups = 64;  // workgroups that fill the rows of no request
static int64_t round256(int64_t v) { return (v + 255) & ~(int64_t)255; }
static int log2_of(int v) {
  int n = 0;
  while ((1 << n) < v) ++n;
  return n;
}

static AttnPlan plan_attention(int64_t tokens, int64_t seqs, int64_t indices, int heads,
                               int kv_heads, int head_size, int page_size, int64_t max_query_len) {
  AttnPlan p{};
  const int group = heads / kv_heads;
  const int64_t longest = max_query_len > 0 && max_query_len < tokens ? max_query_len : tokens;
  const int64_t most_rows = longest * group, all_rows = tokens * group;
  // All sequences together have no more keys.  Beyond 2^36 a smaller number only makes parts longer, and
  // the products below stay within 64 bits.
  int64_t capacity = indices * page_size;
  if (capacity > (int64_t)1 << 36) capacity = (int64_t)1 << 36;
  const int64_t units = compute_units();
  const int few_limit = head_size > 128 ? 32 : 64;
  int64_t few_tiles = 0, chunk_tiles = 0, few_target = 0, chunk_target = 0;
  // Two workgroups per compute unit; one where a chunk's tile has long heads.  Few rows of heads above
  // 128 fit once as well, but count as two: their parts are half as long as filling the GPU once asks for.
  const int64_t room = 2 * units, tile_room = head_size > 128 ? units : room;
  p.few.fill = room / kv_heads > 0 ? (int32_t)(room / kv_heads) : 1;
  p.tile.fill = tile_room / kv_heads > 0 ? (int32_t)(tile_room / kv_heads) : 1;
  p.few.rows_log2 = p.tile.rows_log2 = -1;
  if (most_rows <= few_limit) {
    // all requests in tiles of few rows (max_query_len may be wrong: any number of tiles each)
    const int rows = most_rows <= 16 ? 16 : most_rows <= 32 ? 32 : few_limit;
    p.few.rows_log2 = log2_of(rows);
    p.few.max_rows = 0x7fffffff;
    few_tiles = all_rows / rows + seqs;
  } else {
    // Single tokens in one tile each, longer requests in large tiles; with more than 32 query heads
    // per key head a single token is a large tile.
    const int big = 128, rows = group <= 16 ? 16 : group <= 32 ? 32 : 0;
    if (rows > 0) {
      p.few.rows_log2 = log2_of(rows);
      p.few.max_rows = rows;
      few_tiles = seqs;
    }
    p.tile.rows_log2 = log2_of(big);
    const int64_t chunks = seqs < all_rows / (rows + 1) ? seqs : all_rows / (rows + 1);
    chunk_tiles = all_rows / big + chunks;
    // cut only where the tiles leave a quarter of the GPU idle: a part costs its state's way to
    // memory and back
    if (all_rows / big * kv_heads < tile_room * 3 / 4) chunk_target = p.tile.fill;
    p.tile.min_part = 512;
  }
  if (few_tiles > all_rows) few_tiles = all_rows;
  p.few.min_part = 128;
  // beside chunks, their tiles even out what is left over
  few_target = p.few.rows_log2 < 0 ? 0 : (p.tile.rows_log2 < 0 ? 4 : 1) * (int64_t)p.few.fill;
  // Cutting yields no more parts than the pages can fill, and where parts are as long as filling the
  // GPU once allows, no more than that takes: the fewer workgroups find nothing to do, the better.
  auto bound = [&](int64_t target, const AttnClass& c, int64_t tiles) {
    const int64_t keys = ((most_rows >> c.rows_log2) + 1) * capacity;  // at most so many, times tiles
    int64_t most = keys / kPartKeys > c.fill ? keys / kPartKeys : c.fill;
    if (most > tiles * (capacity / c.min_part)) most = tiles * (capacity / c.min_part);
    return target < most ? target : most;
  };
  if (few_target > 0) few_target = bound(few_target, p.few, few_tiles);
  if (capacity <= kCutKeys + 128) few_target = 0;
  if (chunk_target > 0) chunk_target = bound(chunk_target, p.tile, chunk_tiles);
  // every request is of one class: the tiles that are there at most
  int64_t tiles = p.tile.rows_log2 < 0 ? few_tiles : (all_rows >> p.tile.rows_log2) + seqs;
  if (tiles > all_rows) tiles = all_rows;
  p.uncut_items = tiles;
  p.items = tiles + few_target + chunk_target;
  if (seqs > kPlanSeqs) p.plan_bytes = round256((4 + 2 * seqs) * 4);
  // Only cut tiles leave states.  All cuts together add at most `target` parts and every cut tile has at
  // least one of them, so no more than `target` tiles are cut.
  auto states = [](int64_t tiles, int64_t target, const AttnClass& c) {
    return target == 0 ? 0 : ((tiles < target ? tiles : target) + target) << c.rows_log2;
  };
  p.state_room = states(few_tiles, few_target, p.few) + states(chunk_tiles, chunk_target, p.tile);
  const int64_t state_rows = p.state_room * kv_heads;
  if (few_target + chunk_target == 0 || state_rows >= 0x7fffffffLL) return p;
  p.few.target = (int32_t)few_target;
  p.tile.target = (int32_t)chunk_target;
  p.few.most = (int32_t)(few_tiles + few_target);
  p.map_bytes = round256((2 * seqs + 1) * 4);
  p.ml_bytes = round256(state_rows * 8);
  p.o_bytes = round256(state_rows * head_size * 4);
  return p;
}

}  // namespace sarathi_hip

using namespace sarathi_hip;

// Batches that may hold chunks take the kernel that does both classes; the others have few rows only.
static int launch_paged_attn(const PagedAttnArgs& a, int dtype, bool page16, int64_t groups,
                             hipStream_t st) {
  if (groups == 0) return SARATHI_OK;
  if (a.tile.rows_log2 < 0) return launch_attn_few(a, dtype, page16, groups, st);
  if (dtype == kBF16)
    return a.head_size <= 64    ? launch_attn_mixed_bf16_64(a, page16, groups, st)
           : a.head_size <= 128 ? launch_attn_mixed_bf16_128(a, page16, groups, st)
                                : launch_attn_mixed_bf16_256(a, page16, groups, st);
  return a.head_size <= 64    ? launch_attn_mixed_f16_64(a, page16, groups, st)
         : a.head_size <= 128 ? launch_attn_mixed_f16_128(a, page16, groups, st)
                              : launch_attn_mixed_f16_256(a, page16, groups, st);
}

static bool attn_sizes_ok(int64_t tokens, int64_t seqs, int64_t indices, int heads, int kv_heads,
                          int head_size, int page_size) {
  return tokens >= 0 && seqs >= 0 && indices >= 0 && heads > 0 && kv_heads > 0 &&
         heads % kv_heads == 0 && head_size > 0 && page_size > 0;
}
static bool attn_sizes_fit(int64_t tokens, int64_t seqs, int64_t indices, int heads, int head_size) {
  return head_size <= kAttnMaxHead && heads <= 65535 && tokens * heads < 0x40000000LL &&
         seqs < 0x40000000LL && indices < 0x7fffffffLL;
}

extern "C" int64_t sarathi_paged_attention_workspace_bytes(int64_t num_tokens, int64_t num_seqs,
                                                           int64_t num_kv_indices, int num_heads,
                                                           int num_kv_heads, int head_size,
                                                           int page_size, int64_t max_query_len) {
  if (!attn_sizes_ok(num_tokens, num_seqs, num_kv_indices, num_heads, num_kv_heads, head_size,
                     page_size) ||
      !attn_sizes_fit(num_tokens, num_seqs, num_kv_indices, num_heads, head_size) ||
      num_tokens == 0 || num_seqs == 0)
    return 0;
  const AttnPlan p = plan_attention(num_tokens, num_seqs, num_kv_indices, num_heads, num_kv_heads,
                                    head_size, page_size, max_query_len);
  return p.bytes();
}

extern "C" int sarathi_paged_attention_fill(
    const void* query, const void* k_cache, const void* v_cache, void* out, float* lse,
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t num_tokens, int64_t num_seqs, int64_t num_kv_indices,
    int64_t num_pages, int num_heads, int num_kv_heads, int head_size, int page_size,
    int64_t query_stride, int64_t out_stride, int64_t page_stride, int64_t entry_stride,
    float sm_scale, int causal, int64_t window_left, int64_t max_query_len, void* workspace,
    int64_t workspace_bytes, int dtype, int fill_rows, void* stream) {
  if (fill_rows < 0 || fill_rows > 3) return SARATHI_ERR_INVALID_ARG;
  if (!attn_sizes_ok(num_tokens, num_seqs, num_kv_indices, num_heads, num_kv_heads, head_size,
                     page_size) || num_pages < 0)
    return SARATHI_ERR_INVALID_ARG;
  // maxima are taken before scaling, and masked scores are -inf: the scale is positive and finite
  if (!(sm_scale > 0.f) || !(sm_scale * kLog2e < INFINITY)) return SARATHI_ERR_INVALID_ARG;
  const int64_t row = (int64_t)num_heads * head_size, kv_row = (int64_t)num_kv_heads * head_size;
  if ((num_tokens > 1 && (query_stride < row || out_stride < row)) || entry_stride < kv_row ||
      page_stride < 0)
    return SARATHI_ERR_INVALID_ARG;
  if (num_tokens > 0 && num_seqs > 0 &&
      (!query || !out || !qo_indptr || !kv_indptr || !kv_last_page_len ||
       (num_kv_indices > 0 && !kv_indices) || (num_pages > 0 && (!k_cache || !v_cache))))
    return SARATHI_ERR_INVALID_ARG;
  if ((dtype != kF16 && dtype != kBF16) ||
      !attn_sizes_fit(num_tokens, num_seqs, num_kv_indices, num_heads, head_size) ||
      num_pages >= 0x7fffffffLL)
    return SARATHI_ERR_UNSUPPORTED;
  const int fill = lse ? fill_rows : fill_rows & 2;
  if (num_tokens == 0 || (num_seqs == 0 && fill == 0)) return SARATHI_OK;
  if (num_seqs == 0 && (fill & 2) && !out) return SARATHI_ERR_INVALID_ARG;
  const AttnPlan p = plan_attention(num_tokens, num_seqs, num_kv_indices, num_heads, num_kv_heads,
                              head_size, page_size, max_query_len);
  PagedAttnArgs a{};
  a.q = query;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.out = out;
  a.lse = lse;
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.last_page_len = kv_last_page_len;
  a.q_stride = query_stride;
  a.out_stride = out_stride;
  a.page_stride = page_stride * 2;
  a.entry_stride = entry_stride * 2;
  int up = 0;
  while (((int64_t)1 << up) < page_size) ++up;
  a.page_shift = 31 + up;  // exact for positions below 2^31, and the factor stays below 2^32
  a.page_magic = (uint32_t)((((uint64_t)1 << a.page_shift) + page_size - 1) / page_size);
  a.seqs = (int32_t)num_seqs;
  a.tokens = (int32_t)num_tokens;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.head_size = head_size;
  a.page_size = page_size;
  a.num_pages = (int32_t)num_pages;
  a.num_indices = num_pages > 0 ? (int32_t)num_kv_indices : 0;  // no page: no key
  a.causal = causal != 0;
  a.window = window_left < 0 ? -1 : window_left < 0x3fffffff ? (int32_t)window_left : 0x3fffffff;
  a.fill = fill;
  a.scale_log2 = sm_scale * kLog2e;
  hipStream_t st = (hipStream_t)stream;
  const bool vec = head_size % 8 == 0 && aligned16(query) && aligned16(k_cache) &&
                   aligned16(v_cache) && aligned16(out) && query_stride % 8 == 0 &&
                   out_stride % 4 == 0 && page_stride % 8 == 0 && entry_stride % 8 == 0;
  if (!vec || num_seqs == 0) {
    const dim3 grid((unsigned)num_tokens, (unsigned)num_heads);
    if (dtype == kBF16)
      hipLaunchKernelGGL((paged_attn_plain_kernel<kBF16>), grid, dim3(64), 0, st, a);
    else
      hipLaunchKernelGGL((paged_attn_plain_kernel<kF16>), grid, dim3(64), 0, st, a);
    return launch_status();
  }
  // a workspace that is missing or too small means no cutting and no plan, not an error
  const bool have = workspace && aligned16(workspace) && workspace_bytes >= p.bytes();
  const bool cut = have && p.map_bytes > 0;
  a.few = p.few;
  a.tile = p.tile;
  char* w = reinterpret_cast<char*>(workspace);
  if (have && p.plan_bytes > 0) {
    a.plan = reinterpret_cast<uint32_t*>(w);
    w += p.plan_bytes;
  }
  if (cut) {
    a.part_map = reinterpret_cast<int32_t*>(w);
    a.part_ml = reinterpret_cast<float*>(w + p.map_bytes);
    a.part_o = reinterpret_cast<float*>(w + p.map_bytes + p.ml_bytes);
    a.state_room = (int32_t)p.state_room;
  } else {
    a.few.target = a.tile.target = 0;
  }
  int64_t groups = (cut ? p.items : p.uncut_items) * num_kv_heads;
  a.item_groups = (uint32_t)groups;
  if (fill) groups += num_tokens < kFillGroups ? num_tokens : kFillGroups;
  if (groups > 0x7fffffffLL) return SARATHI_ERR_UNSUPPORTED;
  // offsets inside a share of sixteen keys are 32-bit
  const bool page16 = page_size % 16 == 0 && a.entry_stride < (1 << 26);
  if (a.plan) {
    hipLaunchKernelGGL(paged_attn_plan_kernel, dim3(1), dim3(1024), 0, st, a);
    if (const int rc = launch_status(); rc != SARATHI_OK) return rc;
  }
  const int rc = launch_paged_attn(a, dtype, page16, groups, st);
  if (rc != SARATHI_OK || !cut) return rc;
  return dtype == kBF16 ? launch_join<kBF16>(a, st) : launch_join<kF16>(a, st);
}

extern "C" int sarathi_paged_attention(
    const void* query, const void* k_cache, const void* v_cache, void* out, float* lse,
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t num_tokens, int64_t num_seqs, int64_t num_kv_indices,
    int64_t num_pages, int num_heads, int num_kv_heads, int head_size, int page_size,
    int64_t query_stride, int64_t out_stride, int64_t page_stride, int64_t entry_stride,
    float sm_scale, int causal, int64_t window_left, int64_t max_query_len, void* workspace,
    int64_t workspace_bytes, int dtype, void* stream) {
  return sarathi_paged_attention_fill(query, k_cache, v_cache, out, lse, qo_indptr, kv_indptr, kv_indices,
                                      kv_last_page_len, num_tokens, num_seqs, num_kv_indices, num_pages,
                                      num_heads, num_kv_heads, head_size, page_size, query_stride, out_stride,
                                      page_stride, entry_stride, sm_scale, causal, window_left, max_query_len,
                                      workspace, workspace_bytes, dtype, 0, stream);
}
