// Pieces shared by the kernels that attend over a paged KV cache (paged_attention*.hip).
//
// For a request with n new tokens whose sequence holds s tokens after the append, new token j sits
// at position x = s - n + j and sees the keys [lo, hi):
//   hi = x + 1 (causal) or s,   lo = max(0, x - window) with a window, else 0.
// With z_i = scale * <q, k_i> its state is
//   lse = log sum_i exp(z_i),   o = sum_i exp(z_i - lse) v_i      (no key: o = 0, lse = -inf).
// The query heads that share a key head are rows of the same product: a request's rows for one key
// head are its new tokens times the G = heads / kv_heads query heads, token by token.
//
// Work items.  The kernels take a request's rows in tiles and may cut the keys of a tile into parts
// that different workgroups attend to; the parts' states are joined afterwards (the formula of
// merge_attention_states).  Nothing is planned ahead: every workgroup sums up the requests' lengths
// itself, arrives at the same part length and finds its own item, so a captured launch follows the
// lengths that it finds on the GPU.
#pragma once

#include <stdint.h>

#include "vec16.h"

namespace sarathi_hip {

constexpr int kAttnMaxHead = 256;
constexpr int kAttnWaves = 4;  // of a workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// How the requests of one class are cut into work items.
struct AttnClass {
  int32_t rows_log2;  // rows per tile; -1: the class is empty
  int32_t max_rows;   // few: requests with more rows belong to the other class
  int32_t target;     // items per key head that cutting stays below; 0: do not cut
  int32_t fill;       // items per key head that are taken to fill the GPU once
  int32_t min_part;   // least keys of a part, a multiple of 64
  int32_t most;       // few: items that sound index vectors stay within, cut or not
};

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
  float* part_ml;         // [.. , 2]: reference (in powers of two) and sum
  int32_t* part_map;      // [seqs] first state row, [seqs] parts per tile, and whether any is cut
  int32_t state_room;     // rows per key head that there is room for in the states
  uint32_t* plan;         // or null: what the planning kernel found, see attn_planned_item
  int64_t q_stride, out_stride;           // elements
  int64_t page_stride, entry_stride;      // bytes
  uint32_t page_magic;    // ceil(2^page_shift / page_size): division of positions by page_size
  uint32_t page_shift;
  int32_t seqs, tokens, heads, kv_heads, group, head_size;
  int32_t page_size, num_pages, num_indices;
  int32_t causal, window;                 // window < 0: none
  int32_t fill;           // rows of no request: 1: lse becomes -inf, 2: out becomes 0, 3: both
  uint32_t item_groups;   // workgroups of the items; those behind them fill
  float scale_log2;                       // softmax scale * log2(e)
  AttnClass few, tile;                    // requests of up to few.max_rows rows; those of more
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

// Rows in front of the first request and behind the last one.  A few workgroups of 256 threads behind
// those of the items, which find none, fill them; rows are 8-byte aligned here.  (Filled by the items'
// own workgroups they cost the chunks' loop 1 %; told apart before the search, short decodes 5 %.)
SK_DEV void attn_fill(const PagedAttnArgs& a) {
  if (blockIdx.x < a.item_groups) return;
  const int32_t lo = clamp_i32(a.qo_indptr[0], 0, a.tokens), hi = clamp_i32(a.qo_indptr[a.seqs], lo, a.tokens);
  const int32_t rows = lo + a.tokens - hi;
  for (int64_t i = blockIdx.x - a.item_groups; i < rows; i += gridDim.x - a.item_groups) {
    const int64_t tok = i < lo ? i : hi + (i - lo);
    if (a.fill & 2)
      for (int32_t d = threadIdx.x * 4; d < a.heads * a.head_size; d += 64 * kAttnWaves * 4)
        *reinterpret_cast<u32x2*>(reinterpret_cast<char*>(a.out) + (tok * a.out_stride + d) * 2) = u32x2{0, 0};
    if (a.fill & 1)
      for (int32_t h = threadIdx.x; h < a.heads; h += 64 * kAttnWaves) a.lse[tok * a.heads + h] = -INFINITY;
  }
}

// ---- work items ------------------------------------------------------------------------------

constexpr int kPartKeys = 1024;
constexpr int kCutKeys = 512;
constexpr int kBins = 4;
constexpr int kSortRounds = 10;

struct AttnItem {
  int32_t r;         // request, -1: none
  int32_t tiled;     // 1: a tile of a chunk, 0: a tile of few rows
  int32_t tile;      // tile of its rows
  int32_t part, parts, part_len;
  int32_t state_row; // first state row of this tile and part (key head 0), where parts > 1
  AttnSeq seq;
};

// Inclusive sum over the lanes up to one's own: sixteen lanes by row shifts, then the row totals are
// broadcast to the rows behind.
template <int CTRL, int ROWS> SK_DEV uint32_t dpp_scan_add(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
SK_DEV uint32_t wave_scan(uint32_t v) {
  v = dpp_scan_add<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = dpp_scan_add<0x112, 0xf>(v);
  v = dpp_scan_add<0x114, 0xf>(v);
  v = dpp_scan_add<0x118, 0xf>(v);
  v = dpp_scan_add<0x142, 0xa>(v);  // lane 15 of a row to the next: rows 1 and 3
  return dpp_scan_add<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
}

// Most keys that a tile of the request spans, counted from a multiple of 64 where a window cuts the
// front off.
SK_DEV int32_t attn_keys(const PagedAttnArgs& a, const AttnSeq& x) {
  const int64_t s = (int64_t)a.window + x.n + 63;
  return a.window >= 0 && s < x.s ? (int32_t)s : x.s;
}

SK_DEV AttnItem attn_uniform(const AttnItem& found) {  // the same in every lane: into scalar registers
  AttnItem it;
  it.r = __builtin_amdgcn_readfirstlane(found.r);
  it.tiled = __builtin_amdgcn_readfirstlane(found.tiled);
  it.tile = __builtin_amdgcn_readfirstlane(found.tile);
  it.part = __builtin_amdgcn_readfirstlane(found.part);
  it.parts = __builtin_amdgcn_readfirstlane(found.parts);
  it.part_len = __builtin_amdgcn_readfirstlane(found.part_len);
  it.state_row = __builtin_amdgcn_readfirstlane(found.state_row);
  it.seq.q0 = __builtin_amdgcn_readfirstlane(found.seq.q0);
  it.seq.n = __builtin_amdgcn_readfirstlane(found.seq.n);
  it.seq.kv0 = __builtin_amdgcn_readfirstlane(found.seq.kv0);
  it.seq.s = __builtin_amdgcn_readfirstlane(found.seq.s);
  return it;
}

// Tiles of request r, and the keys that one spans; its parts once they are known.
struct AttnLoad {
  int32_t tiles, keys;
  bool tiled;
  AttnSeq seq;
  int32_t parts;
};
SK_DEV AttnLoad attn_look(const PagedAttnArgs& a, int32_t r) {
  const AttnSeq x = attn_seq(a, r);
  const int64_t rows = (int64_t)x.n * a.group;
  AttnLoad v;
  v.tiled = a.few.rows_log2 < 0 || (a.tile.rows_log2 >= 0 && rows > a.few.max_rows);
  const int32_t lg = v.tiled ? a.tile.rows_log2 : a.few.rows_log2;
  v.tiles = (int32_t)((rows + ((int64_t)1 << lg) - 1) >> lg);
  v.keys = attn_keys(a, x);
  v.seq = x;
  v.parts = 0;
  return v;
}
SK_DEV int32_t attn_parts(int32_t keys, int32_t len) { return keys <= len ? 1 : (keys - 1) / len + 1; }
// States are kept of cut requests only, both classes' in one row: the rows per key head that a request
// needs for its states.
SK_DEV uint32_t attn_state_rows(const AttnClass& c, int32_t tiles, int32_t parts) {
  return parts > 1 ? ((uint32_t)tiles * (uint32_t)parts) << c.rows_log2 : 0;
}
// Index vectors that decrease can ask for more states than there are: such a request is left out.
SK_DEV bool attn_no_room(const PagedAttnArgs& a, const AttnClass& c, uint32_t before, int32_t tiles, int32_t parts) {
  return parts > 1 && before + (((uint64_t)tiles * (uint32_t)parts) << c.rows_log2) > (uint32_t)a.state_room;
}
SK_DEV int32_t attn_state_at(const PagedAttnArgs& a, const AttnClass& c, int32_t first, int32_t item) {
  return first + (int32_t)((uint32_t)(item * a.kv_heads) << c.rows_log2);
}

// Tiles of chunks (bound by the matrix cores) and of few rows (by memory) in turn, so that both
// are at work all the time; the last quarter of the few ones evens out the end.  A chunk of 2048
// tokens beside 256 decodes: 7 % faster than with all tiles first.
SK_DEV bool attn_turn(uint32_t want, uint32_t tile_items, uint32_t few_items, uint32_t& in_class) {
  const uint32_t mixed = tile_items + (uint32_t)((uint64_t)few_items * 3 / 4);
  uint32_t tiles_before = tile_items;
  bool tiled = false;
  if (want < mixed) {
    tiles_before = (uint32_t)(((uint64_t)want * tile_items + mixed - 1) / mixed);
    tiled = (uint32_t)(((uint64_t)(want + 1) * tile_items + mixed - 1) / mixed) > tiles_before;
  }
  in_class = tiled ? tiles_before : want - tiles_before;
  return tiled;
}

// Finds item `want` of a key head: tiles of the chunks, in the order request, tile, part, and in
// between those of few rows, sorted by length into kBins bins, the longest first, so that the end is
// even (256 requests: 5 % faster), unless they are short, all there at once, or so many (kSortRounds
// times what fills the GPU) that the short ones in a row cost more (1000 requests: 4 % slower).
//
// Two sums over the requests: keys times tiles of either class, which fix the classes' part lengths,
// and the numbers of items.  A part is as long as filling the GPU once allows but no longer than
// kPartKeys (below, its start and the way of its state to memory and back weigh in), unless that
// made more than `target` items; it is at least min_part keys and a multiple of 64.  Where no context
// is more than kCutKeys longer than that, nothing is cut: a workgroup takes about 5 us for 512 keys,
// and joining parts as long.  When nothing is cut the first sum is left out.  The workgroup with `map`
// set leaves the state rows for the kernel that joins the parts.  The work is summed in 32-bit floats
// (it only chooses a length, the same in every workgroup; rounded up by more than their error, so
// that the items stay within what the launch has workgroups for).
//
// PLAN: one workgroup writes down what it finds for all requests instead (unsorted).
template <int WAVES, bool PLAN>
SK_DEV AttnItem attn_find_item(const PagedAttnArgs& a, uint32_t want, bool map) {
  __shared__ float work_sums[2][2][WAVES];
  // of the waves: items of chunks, of few rows in bins 0 and 1, 2 and 3; rows of the states
  __shared__ alignas(16) uint32_t sums[4][WAVES];
  __shared__ AttnItem found;
  // Index vectors that decrease can overflow the packed counts below, and then more than one thread
  // takes an item for its own: one of them may write it down, never a mixture of two requests.
  __shared__ uint32_t taken;
  constexpr int NT = WAVES * 64, KEEP = 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t run = (a.seqs + NT - 1) / NT;
  const int64_t first = (int64_t)tid * run;
  const int32_t r0 = first < a.seqs ? (int32_t)first : a.seqs;
  const int32_t r1 = first + run < a.seqs ? (int32_t)(first + run) : a.seqs;
  typedef AttnLoad Load;
  auto look = [&](int32_t r) { return attn_look(a, r); };
  Load kept[KEEP];  // the first requests of this thread are looked at once
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    kept[i] = {0, 0, false, {0, 0, 0, 0}, 0};
    if (r0 + i < r1) kept[i] = look(r0 + i);
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (r0 + i < r1) f(r0 + i, kept[i]);
    for (int32_t r = r0 + KEEP; r < r1; ++r) {
      Load v = look(r);
      f(r, v);
    }
  };
  if (tid == 0) {
    found.r = -1;
    taken = 0;
  }
  int32_t few_len = 0x7fffffff, tile_len = 0x7fffffff;
  bool sorted = false;    // items of few rows, into bins
  float per_block = 0.f;  // bins per 64 keys
  if (a.few.target > 0 || a.tile.target > 0) {
    float few = 0.f, tile = 0.f, few_most = 0.f, tile_most = 0.f;  // keys times tiles; longest
    each([&](int32_t, const Load& v) {
      const float blocks = (float)((v.keys + 63) >> 6);
      (v.tiled ? tile : few) += (float)v.tiles * blocks;
      float& most = v.tiled ? tile_most : few_most;
      if (v.tiles > 0) most = fmaxf(most, blocks);
    });
    few = wave64_sum(few);
    tile = wave64_sum(tile);
    few_most = wave64_max(few_most);
    tile_most = wave64_max(tile_most);
    if (lane == 0) {
      work_sums[0][0][wave] = few;
      work_sums[0][1][wave] = few_most;
      work_sums[1][0][wave] = tile;
      work_sums[1][1][wave] = tile_most;
    }
    __syncthreads();
    auto length = [](const float (&sum)[2][WAVES], const AttnClass& c) {
      if (c.target <= 0) return 0x7fffffff;
      float work = 0.f, most = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        work += sum[0][w];
        most = fmaxf(most, sum[1][w]);
      }
      work *= 1.001f;
      const float len = fmaxf(fminf(work * __builtin_amdgcn_rcpf((float)c.fill), kPartKeys / 64),
                              work * __builtin_amdgcn_rcpf((float)c.target));
      if (most <= len + kCutKeys / 64) return 0x7fffffff;
      const int32_t keys = len > 1.6e7f ? 0x3fffffc0 : (int32_t)ceilf(len) * 64;
      return keys > c.min_part ? keys : c.min_part;
    };
    few_len = length(work_sums[0], a.few);
    tile_len = length(work_sums[1], a.tile);
    float work = 0.f, longest = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      work += work_sums[0][0][w];
      longest = fmaxf(longest, work_sums[0][1][w]);
    }
    const float len = fminf(longest, (float)(few_len >> 6));
    sorted = !PLAN && __builtin_amdgcn_readfirstlane(
        a.few.target > 0 && a.few.most <= 0xffff &&  // bins count in 16 bits
        longest > kPartKeys / 64 && work > len * (float)(a.few.fill - a.seqs) &&
        work <= len * (float)(kSortRounds * a.few.fill - a.seqs));
    per_block = kBins * __builtin_amdgcn_rcpf(len + 1.f);
  }
  auto bin_of = [&](int32_t keys) {
    const int32_t b = (int32_t)((float)((keys >> 6) + 1) * per_block);
    return b < kBins - 1 ? b : kBins - 1;
  };
  // items in bin b of packed counts (those that are not sorted are one number, in the first word)
  auto in_bin = [](uint32_t c01, uint32_t c23, int b) { return ((b < 2 ? c01 : c23) >> (16 * (b & 1))) & 0xffffu; };
  auto parts_of = [&](const Load& v) {
    return attn_parts(v.keys, v.tiled ? tile_len : few_len);
  };
  // the whole parts of a request of few rows, and the rest of each tile
  auto whole_bin = [&](int32_t parts) { return parts > 1 ? bin_of(few_len) : 0; };
  auto rest_bin = [&](const Load& v, int32_t parts) {
    return bin_of(parts > 1 ? v.keys - (parts - 1) * few_len : v.keys);
  };
  const bool cutting = (few_len & tile_len) != 0x7fffffff;
  uint32_t my_tile = 0, my01 = 0, my23 = 0, my_state = 0;
  auto add = [&](int32_t b, uint32_t n) { (b < 2 ? my01 : my23) += n << (16 * (b & 1)); };
  each([&](int32_t, Load& v) {
    v.parts = parts_of(v);
    my_state += attn_state_rows(v.tiled ? a.tile : a.few, v.tiles, v.parts);
    if (v.tiled) {
      my_tile += (uint32_t)(v.tiles * v.parts);
    } else if (sorted) {
      add(whole_bin(v.parts), (uint32_t)(v.tiles * (v.parts - 1)));
      add(rest_bin(v, v.parts), (uint32_t)v.tiles);
    } else {
      my01 += (uint32_t)(v.tiles * v.parts);
    }
  });
  uint32_t tile_at = wave_scan(my_tile), at01 = wave_scan(my01), at23 = 0, state_at = 0;
  if (sorted) at23 = wave_scan(my23);
  if (cutting) state_at = wave_scan(my_state);
  if (lane == 63) {
    sums[0][wave] = tile_at;
    sums[1][wave] = at01;
    sums[2][wave] = at23;
    sums[3][wave] = state_at;
  }
  tile_at -= my_tile;
  at01 -= my01;
  at23 -= my23;
  state_at -= my_state;
  __syncthreads();
  uint32_t tile_items = 0, all01 = 0, all23 = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) {
      tile_at += sums[0][w];
      at01 += sums[1][w];
      at23 += sums[2][w];
      state_at += sums[3][w];
    }
    tile_items += sums[0][w];
    all01 += sums[1][w];
    all23 += sums[2][w];
  }
  uint32_t few_items = all01, few_at = at01;
  if (sorted) {
    few_items = (all01 & 0xffffu) + (all01 >> 16) + (all23 & 0xffffu) + (all23 >> 16);
    few_at = (at01 & 0xffffu) + (at01 >> 16) + (at23 & 0xffffu) + (at23 >> 16);
  }
  uint32_t in_class;
  const bool tiled = attn_turn(want, tile_items, few_items, in_class);
  // few rows: the item's bin, the longest first, and this thread's place in it
  int32_t bin = -1;
  uint32_t at_bin = 0;
  if (sorted && !tiled) {
#pragma unroll
    for (int b = kBins - 1; b >= 0; --b) {
      const uint32_t all = in_bin(all01, all23, b);
      const bool here = bin < 0 && in_class < all;
      in_class -= bin < 0 && !here ? all : 0;
      at_bin = here ? in_bin(at01, at23, b) : at_bin;
      bin = here ? b : bin;
    }
  }
  int32_t cut = 0;
  each([&](int32_t r, const Load& v) {
    const int32_t all = v.parts > 0 ? v.parts : parts_of(v);
    int32_t parts = all;
    uint32_t cnt = (uint32_t)(v.tiles * parts);
    uint32_t& mine_at = v.tiled ? tile_at : few_at;
    const AttnClass& c = v.tiled ? a.tile : a.few;
    const int32_t state = (int32_t)(state_at * (uint32_t)a.kv_heads);
    if (attn_no_room(a, c, state_at, v.tiles, parts)) {
      mine_at += cnt;
      cnt = 0;
      parts = 1;
    }
    state_at += attn_state_rows(c, v.tiles, all);
    if constexpr (PLAN) {
      a.plan[4 + r] = few_at;
      a.plan[4 + a.seqs + r] = tile_at;
    }
    if (map) {
      a.part_map[r] = state;
      a.part_map[a.seqs + r] = parts;
      cut |= parts > 1;
    }
    int32_t tile = -1, part = 0;
    if (tiled || !sorted) {
      const uint32_t in = in_class - mine_at;
      if (v.tiled == tiled && in < cnt) {
        tile = (int32_t)(in / (uint32_t)parts);
        part = (int32_t)(in % (uint32_t)parts);
        if (tiled) tile = v.tiles - 1 - tile;  // a chunk's last tokens have the most keys: first
      }
    } else if (!v.tiled) {
      const uint32_t whole = whole_bin(all) == bin ? (uint32_t)(v.tiles * (all - 1)) : 0;
      const uint32_t rest = rest_bin(v, all) == bin ? (uint32_t)v.tiles : 0;
      const uint32_t in = in_class - at_bin;
      if (cnt > 0 && in < whole) {
        tile = (int32_t)(in / (uint32_t)(all - 1));
        part = (int32_t)(in % (uint32_t)(all - 1));
      } else if (cnt > 0 && in - whole < rest) {
        tile = (int32_t)(in - whole);
        part = all - 1;
      }
      at_bin += whole + rest;
    }
    if (!PLAN && tile >= 0 && atomicExch(&taken, 1u) == 0)
      found = {r, v.tiled, tile, part, parts, v.tiled ? tile_len : few_len,
               attn_state_at(a, c, state, tile * parts + part), v.seq};
    mine_at += cnt;
  });
  if (PLAN && tid == 0) {
    a.plan[0] = (uint32_t)few_len;
    a.plan[1] = (uint32_t)tile_len;
    a.plan[2] = few_items;
    a.plan[3] = tile_items;
  }
  if (map) {  // uniform over the workgroup
    cut = __syncthreads_or(cut);
    if (tid == 0) a.part_map[2 * a.seqs] = cut;
  }
  __syncthreads();
  return found;
}

// The same for batches of many requests, where looking at all of them in every workgroup would cost
// more than a launch (2048 decodes of up to 300 keys, 32 + 8 heads of 128: 0.90 ms, 0.34 this way): the
// planning kernel has left the part lengths, the numbers of items, for either class the items before
// every request, and the state rows.
SK_DEV AttnItem attn_planned_item(const PagedAttnArgs& a, uint32_t want) {
  const int lane = threadIdx.x & 63;
  AttnItem it = {};
  it.r = -1;
  uint32_t in_class;
  const uint32_t few_items = a.plan[2], tile_items = a.plan[3];
  const bool tiled = attn_turn(want, tile_items, few_items, in_class);
  if (in_class >= (tiled ? tile_items : few_items)) return it;
  const AttnClass& c = tiled ? a.tile : a.few;
  const int32_t len = (int32_t)a.plan[tiled ? 1 : 0];
  // the last request with no more items before it: 64 candidates at a time
  const uint32_t* const before = a.plan + 4 + (tiled ? a.seqs : 0);
  int32_t r = 0, width = a.seqs;
  while (true) {
    const int32_t step = (width + 63) / 64;
    const bool ok = lane * step < width && before[r + lane * step] <= in_class;
    const int cnt = __popcll(__builtin_amdgcn_ballot_w64(ok));
    if (cnt == 0) return it;
    r += (cnt - 1) * step;
    if (step == 1) break;
    width = width - (cnt - 1) * step < step ? width - (cnt - 1) * step : step;
  }
  r = __builtin_amdgcn_readfirstlane(r);
  const AttnLoad v = attn_look(a, r);
  const int32_t parts = attn_parts(v.keys, len);
  const uint32_t first = before[r], in = in_class - first;
  if (v.tiled != tiled || in >= (uint32_t)(v.tiles * parts)) return it;
  if (parts > 1 && a.part_map[a.seqs + r] != parts) return it;  // no room for its states
  it.r = r;
  it.tiled = tiled;
  it.tile = (int32_t)(in / (uint32_t)parts);
  it.part = (int32_t)(in % (uint32_t)parts);
  if (tiled) it.tile = v.tiles - 1 - it.tile;
  it.parts = parts;
  it.part_len = len;
  it.state_row = parts > 1 ? attn_state_at(a, c, a.part_map[r], it.tile * parts + it.part) : 0;
  it.seq = v.seq;
  return it;
}

SK_DEV AttnItem attn_item(const PagedAttnArgs& a, uint32_t want, bool first) {
  return attn_uniform(__builtin_expect(a.plan != nullptr, 0) ? attn_planned_item(a, want)
                             : attn_find_item<kAttnWaves, false>(a, want, first && a.part_map != nullptr));
}

// Keys [begin, end) of a part; keys are counted from a multiple of 64, so that sixteen of them lie
// in one page where pages are multiples of 16.
SK_DEV void attn_part(const AttnItem& it, int32_t span_lo, int32_t span_hi, int32_t& begin, int32_t& end) {
  begin = span_lo & ~63;
  end = span_hi;
  if (it.parts > 1) {
    const int64_t b = begin + (int64_t)it.part * it.part_len, e = b + it.part_len;
    begin = b < span_hi ? (int32_t)b : span_hi;
    end = e < span_hi ? (int32_t)e : span_hi;
  }
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
SK_DEV uint32_t lds_addr(const lds_char* p) { return (uint32_t)(uintptr_t)p; }
// Transposing read: 16 lanes read four rows of sixteen 16-bit values, lane i the i % 4-th 8 bytes of
// row i / 4, and receive column i: the values of the four rows.
SK_DEV u32x2 lds_read_tr_b64(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)(uintptr_t)at));
}
SK_DEV u32x4 lds_read_b128(uint32_t at) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)at;
}
// One 16-byte (or 4-byte) piece per lane from global memory into LDS: lane l lands at the base + 16 l
// (4 l), the base uniform over the wave; lanes that are off write nothing.  Completion counts in the
// wave's vmcnt.  Written as instructions that the compiler does not look into, because for its own
// form of them it has the next transposing read wait for every load in flight.  So it places no waits
// for them: every read of what they bring stands behind a counted wait_vmcnt() (and a barrier, where
// another wave loaded it).  No register is written but M0, which nothing else in these kernels uses.
// `to` is the LDS address of the first lane, less `plus` (a constant).  ONCE: data that no other
// workgroup reads (non-temporal: 7.1 instead of 6.3 TB/s where a kernel does nothing but read).
template <bool ONCE> SK_DEV void dma_asm16(const void* src, uint32_t to, int plus) {
  if constexpr (ONCE)
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(to), "v"(src),
                 "n"(plus) : "memory", "scc");
  else
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(src),
                 "n"(plus) : "memory", "scc");
}
template <bool ONCE>
SK_DEV void dma_asm16(const char* uniform_base, uint32_t off, uint32_t to, int plus) {
  if constexpr (ONCE)
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(to), "v"(off),
                 "s"(uniform_base), "n"(plus) : "memory", "scc");
  else
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off),
                 "s"(uniform_base), "n"(plus) : "memory", "scc");
}
SK_DEV void dma_asm4(const void* src, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(src) : "memory");
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

// ---- loads of sixteen keys or values ---------------------------------------------------------------
//
// A share is sixteen consecutive keys (or values), the first at a multiple of 16, brought from
// global memory straight into LDS by one wave: kDmas instructions of 1 KiB, whole rows of the head
// side by side, 16-byte chunks swizzled within their row.  Keys outside [first, end) are never read:
// the nearest one inside stands in (its score is masked).
template <int DP> struct HeadShape {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kChunks = DP / 8;            // 16-byte chunks of a row
  static constexpr int kRowsPerDma = 64 / kChunks;  // rows one load instruction moves
  static constexpr int kDmas = 16 / kRowsPerDma;
  static constexpr int kShareBytes = 16 * kRowBytes;
};

// PAD: the head is shorter than DP (chunks beyond it are not loaded).  PAGE16: pages of a multiple
// of 16 keys, so that a share lies in one page and its address is scalar; the page number is a
// scalar load that the caller issues ahead.  Otherwise page numbers, one per key, go through a small
// LDS ring, loaded IDS / 2 shares ahead.  ONCE: no other workgroup reads these keys.
template <int DP, bool PAD, bool PAGE16, int IDS, bool ONCE> struct ShareLoader {
  using H = HeadShape<DP>;
  const PagedAttnArgs& a;
  const AttnSeq& x;
  int32_t first, end;
  int lane;
  uint32_t ids;  // LDS address of this wave's page numbers, 64 bytes per share

  SK_DEV int row_of(int n) const { return n * H::kRowsPerDma + lane / H::kChunks; }
  // this lane's chunk of load n, with PAGE16 from the share's first entry on
  template <typename Swz> SK_DEV uint32_t chunk(int n, Swz swz) const {
    const uint32_t c = (uint32_t)((lane % H::kChunks) ^ swz(row_of(n))) * 16u;
    return PAGE16 ? c + (uint32_t)row_of(n) * (uint32_t)a.entry_stride : c;
  }
  SK_DEV bool inside_head(int n, uint32_t c) const {
    if constexpr (PAGE16) c -= (uint32_t)row_of(n) * (uint32_t)a.entry_stride;
    return c < (uint32_t)a.head_size * 2u;
  }
  SK_DEV int32_t clamp_key(int32_t t) const { return t < first ? first : t < end ? t : end - 1; }
  // the share at key t, or the nearest one that holds a key
  SK_DEV int32_t base(int32_t t) const { return clamp_i32(t, first & ~15, (end - 1) & ~15); }
  // its page number, through the scalar cache: as a vector load its wait would be one for every load
  // into LDS that is in flight (nothing writes page numbers while a kernel runs)
  SK_DEV int32_t page(int32_t t) const {
    if constexpr (!PAGE16) return 0;
    return ((const __attribute__((address_space(4))) int32_t*)a.kv_indices)[x.kv0 + attn_page_of(a, base(t))];
  }
  SK_DEV void load_ids(int32_t t, int32_t n) const {
    if constexpr (!PAGE16) {
      const int32_t* const from = a.kv_indices + x.kv0 + attn_page_of(a, clamp_key(t + (lane & 15)));
      if (lane < 16) dma_asm4(from, ids + (uint32_t)n % IDS * 64u);
    }
  }
  // share n at key t into LDS at to[r] for each of the R tensors src[r], chunks off[r][.]
  template <int R>
  SK_DEV void load(int32_t t, int32_t n, int32_t page, const char* const (&src)[R],
                   const uint32_t (&off)[R][H::kDmas], const uint32_t (&to)[R]) const {
    if constexpr (PAGE16) {
      const int32_t t0 = base(t);
      const int64_t e = attn_clip_page(a, page) * a.page_stride +
                        (int64_t)(t0 - attn_page_of(a, t0) * a.page_size) * a.entry_stride;
      const bool whole = t0 >= first && t0 + 16 <= end;  // uniform over the wave
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const char* const from = src[r] + e;
        if (whole) {
#pragma unroll
          for (int i = 0; i < H::kDmas; ++i)
            if (!PAD || inside_head(i, off[r][i])) dma_asm16<ONCE>(from, off[r][i], to[r], i * 1024);
        } else {
#pragma unroll
          for (int i = 0; i < H::kDmas; ++i) {
            const int32_t row = clamp_key(t0 + row_of(i)) - t0;
            if (!PAD || inside_head(i, off[r][i]))
              dma_asm16<ONCE>(from, off[r][i] + (uint32_t)(row - row_of(i)) * (uint32_t)a.entry_stride, to[r],
                        i * 1024);
          }
        }
      }
    } else {
      const int32_t key = clamp_key(t + (lane & 15));
      page = *(const __attribute__((address_space(3))) int32_t*)(uintptr_t)(
          ids + (uint32_t)n % IDS * 64u + (uint32_t)(lane & 15) * 4u);
      const int64_t e = attn_clip_page(a, page) * a.page_stride +
                        (int64_t)(key - attn_page_of(a, key) * a.page_size) * a.entry_stride;
      const int32_t e_lo = (int32_t)e, e_hi = (int32_t)(e >> 32);
#pragma unroll
      for (int i = 0; i < H::kDmas; ++i) {
        const int64_t s = (int64_t)(((uint64_t)(uint32_t)__shfl(e_hi, row_of(i), 64) << 32) |
                                    (uint32_t)__shfl(e_lo, row_of(i), 64));
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (!PAD || inside_head(i, off[r][i])) dma_asm16<ONCE>(src[r] + s + off[r][i], to[r], i * 1024);
      }
    }
  }
};

// The running maximum of a row is only a reference for its exponents, and it is raised only when a
// score passes the one it was set for by more than 2^8, so the output is almost never rescaled.  It is
// set kBelow under that score: probabilities stay below 2^8 in bfloat16 and, to use the range of
// float16 (which ends at 2^-24), below 2^15 there; the 32-bit sums mind neither.
constexpr float kRefStart = -3.0e38f;  // below every score; finite, so that no difference is undefined
template <int DT> constexpr float kBelow = DT == kF16 ? 7.f : 0.f;
template <int DT> constexpr float kRaise = 8.f + kBelow<DT>;

// lse of a state with reference m (in powers of two) and sum l; -inf where nothing was seen
SK_DEV float attn_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

}  // namespace sarathi_hip
