// Attention of a chunk of new tokens, in tiles of 128 rows: paged_attn.h has the formulas and the
// order of rows.
//
// Bound by the matrix cores (at the clock that their power leaves) and just below by the vector
// unit's exponentials, so the two have to run side by side.  Four waves, one per SIMD, own 32 rows each
// and walk the keys in steps of 64 that they share in LDS; two workgroups of a compute unit are not
// tied to each other, so that one's softmax runs beside the other's products.
//   scores  S^T = K Q^T (keys as rows, rows as columns: a row's softmax stays in two lanes), output
//           O^T += V^T P^T; the probabilities leave the first product in the layout in which the
//           second takes them, V is transposed by the LDS read.
//   overlap 32 keys' softmax is cut into pieces, each placed behind the products of one operand of
//           the NEXT 32 keys' scores; their row maximum is folded in behind the products with the
//           values.  sched_barrier keeps the pieces apart.
//   loads   keys and values go from global memory straight into LDS, two steps of each (66 KiB: two
//           workgroups per compute unit; 130 KiB and one with heads above 128), asked for as soon as
//           their place is read.  Four steps of each made short chunks no faster.
// Chunks of 16 bytes are stored swizzled so that operand reads meet no bank twice: K by XOR with the
// row, V by XOR of its 64-byte pieces with the row.  Built with the products' results in vector
// registers (build.py): as accumulators they cost a move per score.
// Measured with one chunk of 4096 tokens at 12288, 32 + 8 heads of 128, bfloat16: 0.89 - 0.95 ms by
// machine, 1.01 - 1.08 PFLOP/s, where a library product of 8192^3 reaches 1.2, once the clock has settled
// (the first launches after idling take up to 1.2 ms); with zeros for data, which leave the clock alone,
// it runs a quarter faster.  Eight waves sharing their keys (one workgroup per compute
// unit) were 2 % faster there, 3 % slower on four ragged chunks, 4 % on a hybrid batch and 25 % on 512
// tokens at 8192; four waves of 64 rows (half the LDS reads, one wave per SIMD) took 1.08 ms; the
// softmax spread evenly over both products, or a raised wave priority for the second, changed nothing.
// Heads of 256, 64 + 8 of them, 4096 tokens at 4096: 1.64 - 1.67 ms, 0.99 - 1.01 PFLOP/s (4.72 ms in tiles of 32 rows).
// A launch of few tiles is bound by the chain of a wave alone on its SIMD: 1.4 us per 64 keys and tile.
#pragma once

#include <type_traits>

#include "paged_attn.h"

namespace sarathi_hip {

template <int DT> SK_DEV f32x16 mfma32x16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DP> struct TileShape : HeadShape<DP> {
  static constexpr int kRows = 32 * kAttnWaves;
  static constexpr int kSteps = 2;  // of keys, and of values, in LDS at a time
  static constexpr int kStepBytes = 64 * HeadShape<DP>::kRowBytes;
  static constexpr int kIdSlots = 8;
  static constexpr int kRingBytes = 2 * kSteps * kStepBytes;
  static constexpr int kBytes = kRingBytes + kAttnWaves * kIdSlots * 64;
  SK_DEV static int swz_k(int row) { return DP == 64 ? (row >> 1) & 7 : row & 15; }
  SK_DEV static int swz_v(int row) { return DP == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
};

SK_DEV void fence_order() { __builtin_amdgcn_sched_barrier(0); }

template <int DT, int DP, bool PAD, bool PAGE16>
SK_DEV void tile_item(const PagedAttnArgs& a, const AttnItem& it, uint32_t h, lds_char* lds) {
  using Sh = TileShape<DP>;
  constexpr int ROWS = Sh::kRows, KSTEPS = DP / 16, DTILES = DP / 32;
  constexpr int kOps = Sh::kDmas + (PAGE16 ? 0 : 1);  // loads a wave issues at a time
  constexpr int AHEAD = 3;                   // operands read from LDS before their products
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnSeq x = it.seq;
  const int32_t rows_all = x.n * a.group;
  const int32_t row0 = it.tile * ROWS;
  const int32_t rows = rows_all - row0 < ROWS ? rows_all - row0 : ROWS;

  // this lane's row, and its token counted from the request's first new one
  const int32_t row = wave * 32 + col, row_in = row0 + (row < rows ? row : rows - 1);
  const int32_t row_tok = row_in / a.group;
  const int32_t head = (int32_t)h * a.group + (row_in - row_tok * a.group);
  u32x4 q[KSTEPS];
  {
    const char* const from = reinterpret_cast<const char*>(a.q) +
                             ((int64_t)(x.q0 + row_tok) * a.q_stride + (int64_t)head * a.head_size) * 2;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const int d = k * 16 + half * 8;
      q[k] = !PAD || d < a.head_size ? *reinterpret_cast<const u32x4*>(from + d * 2) : u32x4{0, 0, 0, 0};
    }
  }
  // some row of the tile sees [span_lo, span_hi), every row of this wave [full_lo, full_hi)
  int32_t span_lo, span_hi, full_lo, full_hi, begin, end, skip;
  attn_span(a, x, row0 / a.group, span_lo, skip);
  attn_span(a, x, (row0 + rows - 1) / a.group, skip, span_hi);
  const int32_t w0 = wave * 32, w1 = w0 + 31;
  attn_span(a, x, (row0 + (w0 < rows ? w0 : rows - 1)) / a.group, skip, full_hi);
  attn_span(a, x, (row0 + (w1 < rows ? w1 : rows - 1)) / a.group, full_lo, skip);
  span_lo = __builtin_amdgcn_readfirstlane(span_lo);
  span_hi = __builtin_amdgcn_readfirstlane(span_hi);
  full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  full_hi = __builtin_amdgcn_readfirstlane(full_hi);
  attn_part(it, span_lo, span_hi, begin, end);
  const int32_t first = begin > span_lo ? begin : span_lo;  // keys [first, end) are read
  const int32_t steps = end > begin ? (end - begin + 63) / 64 : 0;

  f32x16 o[DTILES];
  float ref = kRefStart, l = 0.f;
#pragma unroll
  for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;

  const uint32_t klds = lds_addr(lds), vlds = klds + Sh::kSteps * Sh::kStepBytes;
  if constexpr (PAD) {  // chunks beyond the head are never loaded: they stay zero
    for (int i = tid * 16; i < Sh::kRingBytes; i += kAttnWaves * 1024)
      *(__attribute__((address_space(3))) u32x4*)(lds + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }

  // ---- loads: each of the four waves brings one share of the keys and one of the values of a step
  ShareLoader<DP, PAD, PAGE16, Sh::kIdSlots, false> loader{
      a, x, first, end, lane, klds + Sh::kRingBytes + (uint32_t)wave * (Sh::kIdSlots * 64)};
  const char* const src[2] = {reinterpret_cast<const char*>(a.k_cache) + (int64_t)h * a.head_size * 2,
                              reinterpret_cast<const char*>(a.v_cache) + (int64_t)h * a.head_size * 2};
  const uint32_t dst[2] = {klds + (uint32_t)wave * Sh::kShareBytes, vlds + (uint32_t)wave * Sh::kShareBytes};
  uint32_t off[2][1][Sh::kDmas];
#pragma unroll
  for (int n = 0; n < Sh::kDmas; ++n) {
    off[0][0][n] = loader.chunk(n, [](int row) { return Sh::swz_k(row); });
    off[1][0][n] = loader.chunk(n, [](int row) { return Sh::swz_v(row); });
  }
  auto share_at = [&](int32_t j) { return begin + j * 64 + wave * 16; };
  auto load_ids = [&](int32_t j) { loader.load_ids(share_at(j), j); };
  auto share_page = [&](int32_t j) { return loader.page(share_at(j)); };
  auto load = [&](int r, int32_t j, int32_t page) {  // r: 0 keys, 1 values
    const char* const from[1] = {src[r]};
    const uint32_t to[1] = {dst[r] + (uint32_t)j % Sh::kSteps * Sh::kStepBytes};
    loader.load(share_at(j), j, page, from, off[r], to);
  };

  // ---- operand reads
  uint32_t kread[KSTEPS], vread[DTILES];
#pragma unroll
  for (int k = 0; k < KSTEPS; ++k)
    kread[k] = klds + col * Sh::kRowBytes + ((k * 2 + half) ^ Sh::swz_k(col)) * 16;
  const int vlane = lane & 15, vrow = half * 4 + (vlane >> 2);
#pragma unroll
  for (int dt = 0; dt < DTILES; ++dt) {
    const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((vlane >> 1) & 1);
    vread[dt] = vlds + vrow * Sh::kRowBytes + (chunk ^ Sh::swz_v(vrow)) * 16 + (vlane & 1) * 8;
  }
  auto read_k = [&](uint32_t step_at, int sub, int k) {
    return lds_read_b128(kread[k] + step_at + sub * (32 * Sh::kRowBytes));
  };
  auto read_v = [&](uint32_t step_at, int sub, int ks, int dt) {  // ks: 16 of the 32 keys
    const uint32_t at = vread[dt] + step_at + (sub * 32 + ks * 16) * Sh::kRowBytes;
    const u32x2 x0 = lds_read_tr_b64(at), x1 = lds_read_tr_b64(at + 8 * Sh::kRowBytes);
    return u32x4{x0[0], x0[1], x1[0], x1[1]};
  };

  // ---- 32 keys u at a time: keys 32 * (u & 1) of step u / 2
  auto mask = [&](int32_t u, f32x16& s) {
    const int32_t t0 = begin + u * 32;
    if (t0 >= full_lo && t0 + 32 <= full_hi && t0 + 32 <= end) return;  // uniform over the wave
    int32_t lo, hi;
    attn_span(a, x, row_tok, lo, hi);
    const int32_t low = (lo > begin ? lo : begin) - t0 - 4 * half, top = (hi < end ? hi : end) - t0 - 4 * half;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int32_t t = 8 * (i / 4) + i % 4;
      s[i] = t >= low && t < top ? s[i] : -INFINITY;
    }
  };
  // raises the reference of rows whose new maximum (of raw scores) passes it by more than kRaise
  auto raise = [&](float top) {
    auto w = __builtin_amdgcn_permlane32_swap(as_u32(top), as_u32(top), false, false);
    const float z = fmaxf(as_f32(w[0]), as_f32(w[1])) * a.scale_log2;
    if (__builtin_amdgcn_ballot_w64(z > ref + kRaise<DT>) == 0) return;
    const float next = fmaxf(ref, z - kBelow<DT>);
    const float keep = __builtin_amdgcn_exp2f(ref - next);
    ref = next;
    l *= keep;
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt) o[dt] *= keep;
  };
  // The scores of keys u become probabilities and meet the values, while (MORE) those of keys u + 1
  // are formed and their maximum is taken.  SUB = u & 1.
  auto body = [&](int32_t u, auto sub, f32x16& cur, f32x16& next, auto more) {
    constexpr bool MORE = decltype(more)::value;
    constexpr int SUB = decltype(sub)::value;
    constexpr int PV = 2 * DTILES;       // operands of the output's products
    // pairs of probabilities are made behind the operands of the next scores, and pairs of scores
    // enter the maximum behind those of the output: as many of the eight by the n-th of `all`
    auto pairs_by = [](int n, int all) { return n * 8 / all; };
    const uint32_t v_at = (uint32_t)u / 2 % Sh::kSteps * Sh::kStepBytes;
    const uint32_t k_at = ((uint32_t)u + 1) / 2 % Sh::kSteps * Sh::kStepBytes;
    u32x4 p[2], kf[AHEAD + 1], vf[AHEAD + 1];
    if constexpr (MORE) {
#pragma unroll
      for (int i = 0; i < 16; ++i) next[i] = 0.f;
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) kf[n] = read_k(k_at, SUB ^ 1, n);
    }
#pragma unroll
    for (int n = 0; n < KSTEPS; ++n) {
      if constexpr (MORE) {
        if (n + AHEAD < KSTEPS) kf[(n + AHEAD) % (AHEAD + 1)] = read_k(k_at, SUB ^ 1, n + AHEAD);
        next = mfma32x16<DT>(kf[n % (AHEAD + 1)], q[n], next);
      }
      if (n >= KSTEPS - AHEAD) {
        const int i = n - (KSTEPS - AHEAD);
        vf[i] = read_v(v_at, SUB, i / DTILES, i % DTILES);
      }
#pragma unroll
      for (int i = 2 * pairs_by(n, KSTEPS); i < 2 * pairs_by(n + 1, KSTEPS); i += 2) {
        const float z0 = __builtin_amdgcn_exp2f(fmaf(cur[i], a.scale_log2, -ref));
        const float z1 = __builtin_amdgcn_exp2f(fmaf(cur[i + 1], a.scale_log2, -ref));
        l += z0 + z1;
        uint32_t w = pack2<DT>(z0, z1);
        asm volatile("" : "+v"(w), "+v"(l));  // made here, not where they are used
        p[i / 8][i / 2 % 4] = w;
      }
      fence_order();
    }
    if constexpr (MORE) mask(u + 1, next);
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < PV; ++n) {
      if (n + AHEAD < PV)
        vf[(n + AHEAD) % (AHEAD + 1)] = read_v(v_at, SUB, (n + AHEAD) / DTILES, (n + AHEAD) % DTILES);
      o[n % DTILES] = mfma32x16<DT>(vf[n % (AHEAD + 1)], p[n / DTILES], o[n % DTILES]);
      if constexpr (MORE) {
#pragma unroll
        for (int i = 2 * pairs_by(n, PV); i < 2 * pairs_by(n + 1, PV); i += 2) top = fmaxf(fmaxf(top, next[i]), next[i + 1]);
      }
      fence_order();
    }
    if constexpr (MORE) raise(top);
  };

  if (steps > 0) {
    if constexpr (!PAGE16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_ids(i);
      wait_vmcnt<0>();
    }
    // pages of the steps whose values, resp. keys, are asked for next
    int32_t page_v = share_page(1), page_k = share_page(2);
    {
      const int32_t page = share_page(0);
      load(0, 0, page);
      load(1, 0, page);
    }
    load(0, 1, page_v);
    load_ids(4);
    wait_vmcnt<Sh::kDmas + kOps>();  // keys 0
    wave_barrier();
    f32x16 s0, s1;
    {
#pragma unroll
      for (int i = 0; i < 16; ++i) s0[i] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) s0 = mfma32x16<DT>(read_k(0, 0, k), q[k], s0);
      mask(0, s0);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s0[i]);
      raise(top);
    }
    const std::integral_constant<int, 0> sub0{};
    const std::integral_constant<int, 1> sub1{};
    // Values j + 1 are asked for when values j - 1 are used up, at the start of step j, and keys j + 2
    // when keys j are, in its middle.  Both have a step's time to land, and what is waited for is all
    // but the last thing asked for.
    int32_t j = 0;
    wait_vmcnt<kOps>();
    while (j + 1 < steps) {
      wave_barrier();
      load(1, j + 1, page_v);
      body(2 * j, sub0, s0, s1, std::true_type{});
      wait_vmcnt<Sh::kDmas>();
      wave_barrier();
      load(0, j + 2, page_k);
      load_ids(j + 5);
      page_v = page_k;
      page_k = share_page(j + 3);
      body(2 * j + 1, sub1, s1, s0, std::true_type{});
      wait_vmcnt<kOps>();
      ++j;
    }
    wave_barrier();
    body(2 * j, sub0, s0, s1, std::true_type{});
    body(2 * j + 1, sub1, s1, s0, std::false_type{});
    wait_vmcnt<0>();  // nothing may land in LDS after this workgroup has left it
  }

  auto w = __builtin_amdgcn_permlane32_swap(as_u32(l), as_u32(l), false, false);
  l = as_f32(w[0]) + as_f32(w[1]);
  if (row >= rows) return;
  if (it.parts > 1) {
    const int64_t at = (int64_t)it.state_row + h * ROWS + row;
    if (half == 0) {
      a.part_ml[at * 2] = ref;
      a.part_ml[at * 2 + 1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int d = dt * 32 + b * 8 + half * 4;
        if (!PAD || d < a.head_size)
          *reinterpret_cast<f32x4*>(a.part_o + at * a.head_size + d) =
              f32x4{o[dt][b * 4], o[dt][b * 4 + 1], o[dt][b * 4 + 2], o[dt][b * 4 + 3]};
      }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t tok = x.q0 + row_tok;
  char* const to = reinterpret_cast<char*>(a.out) + (tok * a.out_stride + (int64_t)head * a.head_size) * 2;
#pragma unroll
  for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int d = dt * 32 + b * 8 + half * 4;
      if (!PAD || d < a.head_size)
        *reinterpret_cast<u32x2*>(to + d * 2) =
            u32x2{pack2<DT>(o[dt][b * 4] * inv, o[dt][b * 4 + 1] * inv),
                  pack2<DT>(o[dt][b * 4 + 2] * inv, o[dt][b * 4 + 3] * inv)};
    }
  if (a.lse && half == 0) a.lse[tok * a.heads + head] = attn_lse(ref, l);
}

}  // namespace sarathi_hip
