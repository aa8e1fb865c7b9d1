// Attention of a tile of few rows (decode steps): paged_attn.h has the formulas.
//
// Bound by the bytes of the keys and values.  The waves of a workgroup share one tile of 16 * RT rows
// and stream its keys 16 at a time, dealt to them in turn, each wave through a ring of its own in LDS
// (kStages shares of keys and of values), so that no wave waits for another before the end: there
// their states are joined through LDS.
//   scores  S^T = K Q^T: keys as rows, the tile's rows as columns, so a row's softmax stays inside
//           four lanes (lane & 15 names the row), and the probabilities come out of the product in
//           the very layout in which
//   output  O^T += V^T P^T takes them: no exchange between lanes, V is transposed by the LDS read.
// Chunks of 16 bytes are stored swizzled, K by XOR with the row so that sixteen rows' same chunk
// lie in different banks, V by XOR of chunk pairs so that eight rows' same sixteen elements do.
// Probabilities are rounded to the cache's type for the product (at most half a step each); maximum,
// sum and output stay in 32 bits.
//
// Measured, bfloat16, 32 + 8 heads of 128, pages of 16: 256 requests of up to 8191 tokens (4.3 GB) 0.68 ms,
// 6.35 TB/s, where a kernel that only reads the same way reaches 7.1; 64 such requests 0.20 ms, 5.5 TB/s;
// one of 4096 tokens 10 us and 4 us more for the join.  With 256 requests (0.715 ms then) two waves per
// workgroup took 0.73 ms, eight 0.78, twice the stages with one workgroup per compute unit 0.81.
#pragma once

#include "paged_attn.h"

namespace sarathi_hip {

template <int DP> struct FewShape : HeadShape<DP> {
  static constexpr int kStages = DP == 64 ? 4 : 2;
  static constexpr int kIdSlots = 2 * kStages;
  static constexpr int kWaveBytes = kStages * 2 * HeadShape<DP>::kShareBytes + kIdSlots * 64;
  SK_DEV static int swz_k(int row) { return DP == 64 ? (row >> 1) & 7 : row & 15; }
  SK_DEV static int swz_v(int row) { return DP == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1; }
};
// dynamic LDS: the rings, later the states that half of the waves hand over
template <int DP, int RT> constexpr int few_lds_bytes() {
  constexpr int ring = kAttnWaves * FewShape<DP>::kWaveBytes;
  constexpr int join = kAttnWaves / 2 * 64 * (2 + DP / 16 * 4) * RT * 4;
  return ring > join ? ring : join;
}

template <int DT, int DP, int RT, bool PAD, bool PAGE16>
SK_DEV void few_item(const PagedAttnArgs& a, const AttnItem& it, uint32_t h, lds_char* lds) {
  using Sh = FewShape<DP>;
  constexpr int WAVES = kAttnWaves, ROWS = 16 * RT, S = Sh::kStages, KSTEPS = DP / 32, DTILES = DP / 16;
  constexpr int kOps = 2 * Sh::kDmas + (PAGE16 ? 0 : 1);  // loads a wave issues per block
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnSeq x = it.seq;
  const int32_t rows_all = x.n * a.group, row0 = it.tile * ROWS;
  const int32_t rows = rows_all - row0 < ROWS ? rows_all - row0 : ROWS;

  // some row sees [span_lo, span_hi), every row [full_lo, full_hi)
  int32_t span_lo, span_hi, full_lo, full_hi, begin, end;
  attn_span(a, x, row0 / a.group, span_lo, full_hi);
  attn_span(a, x, (row0 + rows - 1) / a.group, full_lo, span_hi);
  span_lo = __builtin_amdgcn_readfirstlane(span_lo);
  span_hi = __builtin_amdgcn_readfirstlane(span_hi);
  full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  full_hi = __builtin_amdgcn_readfirstlane(full_hi);
  attn_part(it, span_lo, span_hi, begin, end);
  const int32_t first = begin > span_lo ? begin : span_lo;  // keys [first, end) are read
  // blocks of 16 keys are dealt to the waves in turn
  const int32_t blocks = end > begin ? (end - begin + 15) / 16 : 0;
  const int32_t nb = blocks > wave ? (blocks - wave - 1) / WAVES + 1 : 0;

  lds_char* const mine = lds + wave * Sh::kWaveBytes;
  const uint32_t ring = lds_addr(mine);
  ShareLoader<DP, PAD, PAGE16, Sh::kIdSlots, true> loader{a, x, first, end, lane,
                                                    ring + S * 2 * Sh::kShareBytes};
  const char* const src[2] = {reinterpret_cast<const char*>(a.k_cache) + (int64_t)h * a.head_size * 2,
                              reinterpret_cast<const char*>(a.v_cache) + (int64_t)h * a.head_size * 2};
  uint32_t off[2][Sh::kDmas];
#pragma unroll
  for (int n = 0; n < Sh::kDmas; ++n) {
    off[0][n] = loader.chunk(n, [](int row) { return Sh::swz_k(row); });
    off[1][n] = loader.chunk(n, [](int row) { return Sh::swz_v(row); });
  }
  auto key_at = [&](int32_t b) { return begin + (b * WAVES + wave) * 16; };
  auto load_block = [&](int32_t b, int32_t page) {
    const uint32_t to = ring + (uint32_t)b % S * (2 * Sh::kShareBytes);
    const uint32_t dst[2] = {to, to + Sh::kShareBytes};
    loader.load(key_at(b), b, page, src, off, dst);
  };
  if constexpr (PAD) {  // chunks beyond the head are never loaded: they stay zero
    for (int i = lane * 16; i < S * 2 * Sh::kShareBytes; i += 1024)
      *(__attribute__((address_space(3))) u32x4*)(mine + i) = u32x4{0, 0, 0, 0};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  // the first page numbers and this lane's rows (one per row tile) on their way together
  int32_t page[S + 1];
  if (nb > 0) {
#pragma unroll
    for (int i = 0; i < S; ++i) loader.load_ids(key_at(i), i);
#pragma unroll
    for (int i = 0; i <= S; ++i) page[i] = loader.page(key_at(i));
  }
  u32x4 q[RT][KSTEPS];
  int32_t row_tok[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int32_t i = rt * 16 + col;
    const int32_t p = row0 + (i < rows ? i : rows - 1);
    const int32_t j = p / a.group;
    row_tok[rt] = j;
    const int32_t head = (int32_t)h * a.group + (p - j * a.group);
    const char* from = reinterpret_cast<const char*>(a.q) +
                       ((int64_t)(x.q0 + j) * a.q_stride + (int64_t)head * a.head_size) * 2;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const int d = k * 32 + g * 8;
      q[rt][k] = !PAD || d < a.head_size ? *reinterpret_cast<const u32x4*>(from + d * 2)
                                         : u32x4{0, 0, 0, 0};
    }
  }
  // the compiler counts no load that this file writes out: its wait for q must not come later
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) asm volatile("" : "+v"(q[rt][k]));

  float ref[RT], l[RT];
  f32x4 o[RT][DTILES];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    ref[rt] = kRefStart;
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  uint32_t kread[KSTEPS], vread[DTILES];
#pragma unroll
  for (int k = 0; k < KSTEPS; ++k)
    kread[k] = ring + col * Sh::kRowBytes + ((k * 4 + g) ^ Sh::swz_k(col)) * 16;
  const int vrow = g * 4 + (col >> 2);
#pragma unroll
  for (int dt = 0; dt < DTILES; ++dt)
    vread[dt] = ring + Sh::kShareBytes + vrow * Sh::kRowBytes +
                ((dt * 2 + ((col >> 1) & 1)) ^ Sh::swz_v(vrow)) * 16 + (col & 1) * 8;

  if (nb > 0) {
    wait_vmcnt<0>();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      load_block(i, page[i]);
      loader.load_ids(key_at(S + i), S + i);
    }
  }
  int32_t next_page = nb > 0 ? page[S] : 0;
  for (int32_t b = 0; b < nb; ++b) {
    // everything up to this block's values (and the page numbers of block b + S)
    wait_vmcnt<(S - 1) * kOps>();
    const uint32_t at = (uint32_t)b % S * (2 * Sh::kShareBytes);
    const int32_t t0 = key_at(b);
    f32x4 s[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const u32x4 kk = lds_read_b128(kread[k] + at);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt] = mfma16x32<DT>(kk, q[rt][k], s[rt]);
    }
    if (!(t0 >= full_lo && t0 + 16 <= full_hi && t0 + 16 <= end)) {  // uniform over the wave
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        int32_t lo, hi;
        attn_span(a, x, row_tok[rt], lo, hi);
        const int32_t low = (lo > begin ? lo : begin) - t0 - g * 4, top = (hi < end ? hi : end) - t0 - g * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) s[rt][j] = j >= low && j < top ? s[rt][j] : -INFINITY;
      }
    }
    float z[RT];
    bool need = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      z[rt] = group_max(fmaxf(fmaxf(s[rt][0], s[rt][1]), fmaxf(s[rt][2], s[rt][3]))) * a.scale_log2;
      need |= z[rt] > ref[rt] + kRaise<DT>;
    }
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float next = fmaxf(ref[rt], z[rt] - kBelow<DT>);
        const float keep = __builtin_amdgcn_exp2f(ref[rt] - next);
        ref[rt] = next;
        l[rt] *= keep;
#pragma unroll
        for (int dt = 0; dt < DTILES; ++dt) o[rt][dt] *= keep;
      }
    }
    u32x2 p[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        e[j] = __builtin_amdgcn_exp2f(fmaf(s[rt][j], a.scale_log2, -ref[rt]));
      l[rt] += (e[0] + e[1]) + (e[2] + e[3]);
      p[rt] = u32x2{pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3])};
    }
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt) {
      const u32x2 vv = lds_read_tr_b64(vread[dt] + at);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma16x16<DT>(vv, p[rt], o[rt][dt]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the block is read: its place can be filled
    load_block(b + S, next_page);
    loader.load_ids(key_at(b + 2 * S), b + 2 * S);
    next_page = loader.page(key_at(b + S + 1));
  }
  wait_vmcnt<0>();  // nothing may land in LDS from here on
  __syncthreads();

  // join the waves' states: the upper half hands over to the lower, until one is left
  typedef __attribute__((address_space(3))) float lds_float;
  constexpr int kTile = 64 * (2 + DTILES * 4);  // floats per row tile
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) l[rt] = group_sum(l[rt]);
#pragma unroll
  for (int step = WAVES / 2; step > 0; step >>= 1) {
    lds_float* const box = (lds_float*)lds + (wave & (step - 1)) * (kTile * RT);
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        lds_float* const b = box + rt * kTile;
        b[lane] = ref[rt];
        b[64 + lane] = l[rt];
#pragma unroll
        for (int dt = 0; dt < DTILES; ++dt)
          *(__attribute__((address_space(3))) f32x4*)(b + 128 + dt * 256 + lane * 4) = o[rt][dt];
      }
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        lds_float* const b = box + rt * kTile;
        const float ref2 = b[lane], l2 = b[64 + lane];
        const float top = fmaxf(ref[rt], ref2);
        const float w1 = __builtin_amdgcn_exp2f(ref[rt] - top), w2 = __builtin_amdgcn_exp2f(ref2 - top);
        ref[rt] = top;
        l[rt] = l[rt] * w1 + l2 * w2;
#pragma unroll
        for (int dt = 0; dt < DTILES; ++dt)
          o[rt][dt] = o[rt][dt] * w1 +
                      *(__attribute__((address_space(3))) f32x4*)(b + 128 + dt * 256 + lane * 4) * w2;
      }
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int32_t i = rt * 16 + col;
    if (i >= rows) continue;
    if (it.parts > 1) {
      const int64_t row = (int64_t)it.state_row + h * ROWS + i;
      if (g == 0) {
        a.part_ml[row * 2] = ref[rt];
        a.part_ml[row * 2 + 1] = l[rt];
      }
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
        if (!PAD || dt * 16 + g * 4 < a.head_size)
          *reinterpret_cast<f32x4*>(a.part_o + row * a.head_size + dt * 16 + g * 4) = o[rt][dt];
    } else {
      const float inv = l[rt] == 0.f ? 0.f : 1.f / l[rt];
      const int64_t tok = x.q0 + row_tok[rt];
      const int32_t head = (int32_t)h * a.group + (row0 + i - row_tok[rt] * a.group);
      char* const dst = reinterpret_cast<char*>(a.out) + (tok * a.out_stride + (int64_t)head * a.head_size) * 2;
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
        if (!PAD || dt * 16 + g * 4 < a.head_size)
          *reinterpret_cast<u32x2*>(dst + (dt * 16 + g * 4) * 2) =
              u32x2{pack2<DT>(o[rt][dt][0] * inv, o[rt][dt][1] * inv),
                    pack2<DT>(o[rt][dt][2] * inv, o[rt][dt][3] * inv)};
      if (a.lse && g == 0) a.lse[tok * a.heads + head] = attn_lse(ref[rt], l[rt]);
    }
  }
}

}  // namespace sarathi_hip
