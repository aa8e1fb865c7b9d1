// Pieces shared by the kernels that attend over a paged KV cache (paged_attention.hip,
// paged_attention_tiles.hip).
//
// For a request with n new tokens whose sequence holds s tokens after the append, new token j sits
// at position x = s - n + j and sees the keys [lo, hi):
//   hi = x + 1 (causal) or s,   lo = max(0, x - window) with a window, else 0.
// With z_i = scale * <q, k_i> its state is
//   lse = log sum_i exp(z_i),   o = sum_i exp(z_i - lse) v_i      (no key: o = 0, lse = -inf).
// The query heads that share a key head are rows of the same product: a request's rows for one key
// head are its new tokens times the G = heads / kv_heads query heads, token by token.
//
// Work items.  A kernel takes a request's rows in tiles and may cut the keys of a tile into parts
// that different workgroups attend to; the parts' states are joined afterwards (the formula of
// merge_attention_states).  Nothing is planned ahead: every workgroup sums up the requests' lengths
// itself, arrives at the same part length and finds its own item, so a captured launch follows the
// lengths that it finds on the GPU.
#pragma once

#include <stdint.h>

#include "vec16.h"

namespace sarathi_hip {

constexpr int kAttnMaxHead = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedAttnArgs {
  const void* q;          // [T, heads, D], tokens q_stride elements apart
  const void* k_cache;
  const void* v_cache;
  void* out;              // [T, heads, D], tokens out_stride elements apart
  float* lse;             // [T, heads] or null
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* last_page_len;
  float* part_o;          // states of the parts, or null: nothing is cut
  float* part_ml;         // [.. , 2]: running maximum (in powers of two) and sum
  int32_t* part_map;      // [seqs + 1] first item, then [seqs] parts per tile
  int64_t q_stride, out_stride;           // elements
  int64_t page_stride, entry_stride;      // bytes
  uint32_t page_magic;    // ceil(2^page_shift / page_size): division of positions by page_size
  uint32_t page_shift;
  int32_t seqs, tokens, heads, kv_heads, group, head_size;
  int32_t page_size, num_pages, num_indices;
  int32_t causal, window;                 // window < 0: none
  float scale_log2;                       // softmax scale * log2(e)
  int32_t min_rows, max_rows;             // this kernel takes requests with rows in [min, max]
  int32_t target;                         // items per key head that cutting aims at; 0: do not cut
  int32_t min_part;                       // least keys of a part, a multiple of 64
};

// One request as the kernels see it; whatever the index vectors hold, nothing outside the
// tensors is reached.
struct AttnSeq {
  int32_t q0, n;    // first row of the query tensor, new tokens
  int32_t kv0, s;   // first entry of kv_indices, keys
};
SK_DEV int32_t clamp_i32(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }
SK_DEV AttnSeq attn_seq(const PagedAttnArgs& a, int32_t r) {
  AttnSeq x;
  x.q0 = clamp_i32(a.qo_indptr[r], 0, a.tokens);
  x.n = clamp_i32(a.qo_indptr[r + 1], x.q0, a.tokens) - x.q0;
  x.kv0 = clamp_i32(a.kv_indptr[r], 0, a.num_indices);
  const int32_t pages = clamp_i32(a.kv_indptr[r + 1], x.kv0, a.num_indices) - x.kv0;
  const int64_t s = pages > 0 ? (int64_t)(pages - 1) * a.page_size +
                                    clamp_i32(a.last_page_len[r], 0, a.page_size)
                              : 0;
  x.s = s < 0x3fffffffLL ? (int32_t)s : 0x3fffffff;
  return x;
}

// Keys [lo, hi) that new token j of the request sees.
SK_DEV void attn_span(const PagedAttnArgs& a, const AttnSeq& x, int32_t j, int32_t& lo, int32_t& hi) {
  const int32_t pos = x.s - x.n + j;
  hi = a.causal ? clamp_i32(pos + 1, 0, x.s) : x.s;
  lo = a.window >= 0 && pos > a.window ? pos - a.window : 0;
  if (lo > hi) lo = hi;
}

// Position -> index of its page in the request's part of kv_indices.
SK_DEV int32_t attn_page_of(const PagedAttnArgs& a, int32_t pos) {
  return (int32_t)(((uint64_t)(uint32_t)pos * (uint64_t)a.page_magic) >> a.page_shift);
}
// A page number outside the cache is never followed: the last page stands in for it.
SK_DEV int32_t attn_clip_page(const PagedAttnArgs& a, int32_t page) {
  return (uint32_t)page < (uint32_t)a.num_pages ? page : a.num_pages - 1;
}
// Byte offset of the entry that holds key `pos` (below x.s) of the request.
SK_DEV int64_t attn_entry(const PagedAttnArgs& a, const AttnSeq& x, int32_t pos) {
  const int32_t pg = attn_page_of(a, pos);
  const int32_t page = attn_clip_page(a, a.kv_indices[x.kv0 + pg]);
  return page * a.page_stride + (int64_t)(pos - pg * a.page_size) * a.entry_stride;
}

// ---- work items ------------------------------------------------------------------------------

struct AttnItem {
  int32_t r;       // request, -1: none
  int32_t tile;    // tile of its rows
  int32_t part, parts;
  int32_t index;   // item index over all requests: where the part's state goes
  int32_t part_len;
};

SK_DEV uint64_t wave_scan_u64(uint64_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t u = __shfl_up(v, d, 64);
    if (lane >= d) v += u;
  }
  return v;
}

// Most keys that a tile of the request spans with a window, counted from a multiple of 64.
SK_DEV int32_t attn_window_keys(const PagedAttnArgs& a, const AttnSeq& x) {
  const int64_t s = (int64_t)a.window + x.n + 63;
  return s < x.s ? (int32_t)s : x.s;
}

// Rows per tile ROWS, WAVES waves in the workgroup.  `want` counts the items of one key head in
// the order request, tile, part.  Two sums over the requests: keys times tiles, which fixes the
// part length (the same for all, at least min_part, a multiple of 64, so that about a.target
// items come out), and the number of items.  When nothing is cut the first is left out.  The
// workgroup with `map` set leaves the item counts for the kernel that joins the parts.
template <int ROWS, int WAVES>
SK_DEV AttnItem attn_find_item(const PagedAttnArgs& a, uint32_t want, bool map) {
  __shared__ uint64_t sums[WAVES];
  __shared__ AttnItem found;
  constexpr int NT = WAVES * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t run = (a.seqs + NT - 1) / NT;
  const int64_t first = (int64_t)tid * run;
  const int32_t r0 = first < a.seqs ? (int32_t)first : a.seqs;
  const int32_t r1 = first + run < a.seqs ? (int32_t)(first + run) : a.seqs;
  const bool narrow = a.seqs <= 64;  // all requests in the first wave's lanes: no exchange
  int32_t part_len = 0x7fffffff;
  auto tiles_of = [&](const AttnSeq& x) {
    const int64_t rows = (int64_t)x.n * a.group;
    return rows >= a.min_rows && rows <= a.max_rows ? (int32_t)((rows + ROWS - 1) / ROWS) : 0;
  };
  if (tid == 0) found.r = -1;
  if (a.target > 0) {
    uint64_t work = 0;
    for (int32_t r = r0; r < r1; ++r) {
      const AttnSeq x = attn_seq(a, r);
      int32_t s = x.s;  // keys that the tiles of this request walk, roughly
      if (a.window >= 0) s = attn_window_keys(a, x);
      work += (uint64_t)tiles_of(x) * (uint32_t)s;
    }
    work = wave_scan_u64(work, lane);
    if (lane == 63) sums[wave] = work;
    __syncthreads();
    work = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) work += sums[w];
    const uint64_t len = (work + (uint32_t)a.target - 1) / (uint32_t)a.target;
    const uint64_t up = (len + 63) & ~63ull;
    part_len = up > 0x3fffffc0ull ? 0x3fffffc0 : (int32_t)up;
    if (part_len < a.min_part) part_len = a.min_part;
    __syncthreads();  // sums[] is written again below
  }
  auto parts_of = [&](const AttnSeq& x) {
    const int32_t s = a.window >= 0 ? attn_window_keys(a, x) : x.s;
    return part_len == 0x7fffffff || s <= part_len ? 1 : (s - 1) / part_len + 1;
  };
  uint64_t mine = 0;
  for (int32_t r = r0; r < r1; ++r) {
    const AttnSeq x = attn_seq(a, r);
    mine += (uint64_t)tiles_of(x) * (uint32_t)parts_of(x);
  }
  const uint64_t incl = wave_scan_u64(mine, lane);
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  uint64_t at = incl - mine;
  if (!narrow)
    for (int w = 0; w < wave; ++w) at += sums[w];
  for (int32_t r = r0; r < r1; ++r) {
    const AttnSeq x = attn_seq(a, r);
    const int32_t parts = parts_of(x);
    const uint64_t cnt = (uint64_t)tiles_of(x) * (uint32_t)parts;
    if (map) {
      a.part_map[r] = (int32_t)at;
      a.part_map[a.seqs + r] = cnt ? parts : 0;
    }
    if (want >= at && want < at + cnt) {
      const int32_t in = (int32_t)(want - at);
      found = {r, in / parts, in % parts, parts, (int32_t)want, part_len};
    }
    at += cnt;
  }
  __syncthreads();
  AttnItem it = found;
  it.r = __builtin_amdgcn_readfirstlane(it.r);
  it.tile = __builtin_amdgcn_readfirstlane(it.tile);
  it.part = __builtin_amdgcn_readfirstlane(it.part);
  it.parts = __builtin_amdgcn_readfirstlane(it.parts);
  it.index = __builtin_amdgcn_readfirstlane(it.index);
  it.part_len = __builtin_amdgcn_readfirstlane(it.part_len);
  return it;
}

// ---- matrix cores --------------------------------------------------------------------------------

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 16 x 16 products: A has rows (lane & 15), B columns (lane & 15); lane group lane >> 4 holds k =
// 8 g .. 8 g + 7 (depth 32) or 4 g .. 4 g + 3 (depth 16); the result has column lane & 15 and rows
// 4 g .. 4 g + 3.
template <int DT> SK_DEV f32x4 mfma16x32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT> SK_DEV f32x4 mfma16x16(u32x2 a, u32x2 b, f32x4 c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                     __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                 __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) char lds_char;
// Transposing reads: 16 lanes read four rows of sixteen 16-bit values, lane i the i % 4-th 8 bytes of
// row i / 4, and receive column i: the values of the four rows.  N of them from byte addresses in
// LDS, with their wait in the same block (the compiler's own form of this read waits for every load
// into LDS that is in flight, also those of other buffers).
SK_DEV uint32_t lds_addr(const lds_char* p) { return (uint32_t)(uintptr_t)p; }
SK_DEV void lds_read_tr4(const uint32_t (&at)[4], u32x2 (&v)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %5\n\t"
      "ds_read_b64_tr_b16 %2, %6\n\tds_read_b64_tr_b16 %3, %7\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
      : "memory");
}
// One 16-byte (or 4-byte) piece per lane from global memory into LDS: lane l lands at base + 16 l
// (4 l), base uniform over the wave; lanes that are off write nothing.  Completion counts in the
// wave's vmcnt.
template <int BYTES> SK_DEV void dma_to_lds(const void* src, lds_char* base) {
  // (the builtin wants its size as a literal)
  if constexpr (BYTES == 16)
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)base, 16, 0, 0);
  else
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)base, 4, 0, 0);
}

// The same read for one address, its wait placed by the compiler; for kernels whose loads into LDS
// are the ones below, of which the compiler knows nothing.
SK_DEV u32x2 lds_read_tr_b64(const lds_char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)p));
}
// dma_to_lds() as instructions that the compiler does not look into: it places no waits for them, so
// every read of what they bring stands behind a counted wait_vmcnt() (and a barrier, where another
// wave loaded it).  No register is written but M0, which nothing else in those kernels uses.
// `to` is the LDS address of the first lane, less `plus` (a constant).
SK_DEV void dma_asm16(const void* src, uint32_t to, int plus) {
  asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(src), "n"(plus)
               : "memory", "scc");
}
SK_DEV void dma_asm16(const char* uniform_base, uint32_t off, uint32_t to, int plus) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off),
               "s"(uniform_base), "n"(plus)
               : "memory", "scc");
}
SK_DEV void dma_asm4(const void* src, lds_char* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_addr(base)), "v"(src)
               : "memory");
}
// Meets the other waves; only LDS reads of this wave have to be complete (they are: their results
// have been used).
SK_DEV void wave_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Maximum / sum over the lanes that differ in bits 4 and 5.
SK_DEV float group_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(as_u32(v), as_u32(v), false, false);
  v = fmaxf(as_f32(a[0]), as_f32(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
  return fmaxf(as_f32(b[0]), as_f32(b[1]));
}
SK_DEV float group_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(as_u32(v), as_u32(v), false, false);
  v = as_f32(a[0]) + as_f32(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
  return as_f32(b[0]) + as_f32(b[1]);
}

// lse of a state with maximum m (in powers of two) and sum l; -inf where nothing was seen
SK_DEV float attn_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

}  // namespace sarathi_hip
