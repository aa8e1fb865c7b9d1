// Attention of chunks of new tokens over the paged cache: tiles of 128 or 256 rows on the matrix
// cores (paged_attn.h has the formulas and the order of rows).
//
// Bound by the matrix cores and, just below, by the vector unit's exponentials: per 64 keys a wave
// of 64 rows spends 2048 cycles in products and some 1500 in the softmax, so the two have to run
// side by side.  Four waves, one per SIMD with the whole register file, own 32 * QT rows each
// (QT = 2: every operand read from LDS feeds two products, half the LDS bandwidth; with 32 rows per
// wave the reads alone would fill it) and walk the keys in steps of 64 that they share in LDS.
//
//   scores  S^T = K Q^T (keys as rows, rows as columns: a row's softmax stays in two lanes), output
//           O^T += V^T P^T; the probabilities leave the first product in the layout in which the
//           second takes them, V is transposed by the LDS read.
//   overlap a step's softmax is cut into sixteen pieces, each placed behind the products of one
//           operand of the NEXT step's scores; the next step's row maximum is folded in behind the
//           products with the values.  sched_barrier keeps the pieces apart.
//   maximum the running maximum is only raised when a row's new one exceeds it by more than 2^8:
//           probabilities then stay below 2^8, which neither 16-bit type nor the 32-bit sums mind,
//           and the output is almost never rescaled.
//   loads   keys and values go from global memory straight into LDS, three steps of each, two of
//           them in flight; one barrier per step.  Where the sixteen keys of a wave's share lie in
//           one page and none is past an end their address is scalar.
// Chunks of 16 bytes are stored swizzled so that operand reads meet no bank twice: K by XOR with the
// row, V by XOR of its 64-byte pieces with the row.
#include <type_traits>

#include "launch.h"
#include "paged_attn.h"
#include "paged_attn_tiles.h"

namespace sarathi_hip {

template <int DT> SK_DEV f32x16 mfma32x16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DP> struct TileShape {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kChunks = DP / 8;
  static constexpr int kRowsPerDma = 64 / kChunks;
  static constexpr int kDmas = 16 / kRowsPerDma;  // a wave's 16 keys (or values) of a step
  static constexpr int kSteps = 4;                // of keys, and of values, in LDS at a time
  static constexpr int kStepBytes = 64 * kRowBytes;
  static constexpr int kIdSlots = 8;
  static constexpr int kRingBytes = 2 * kSteps * kStepBytes;
  static constexpr int kBytes = kRingBytes + 8 * kIdSlots * 64;
  SK_DEV static int swz_k(int row) { return DP == 64 ? (row >> 1) & 7 : row & 15; }
  SK_DEV static int swz_v(int row) { return DP == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
};

constexpr float kRefStart = -3.0e38f;  // below every score; finite, so that no difference is undefined
constexpr float kRaise = 8.f;          // see "maximum" above

SK_DEV void fence_order() { __builtin_amdgcn_sched_barrier(0); }

// PAGE16: pages of a multiple of 16 keys, so that a wave's share of a step lies in one page.
template <int DT, int DP, int WAVES, int QT, bool PAD, bool PAGE16>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(WAVES / 4, WAVES / 4)))
void paged_attn_tile_kernel(PagedAttnArgs a) {
  using Sh = TileShape<DP>;
  constexpr int ROWS = WAVES * 32 * QT, KSTEPS = DP / 16, DTILES = DP / 32;
  constexpr int ROLES = WAVES == 8 ? 1 : 2;  // 8 waves: half of them bring keys, half values
  constexpr int kOps = ROLES * Sh::kDmas + (PAGE16 ? 0 : 1);  // loads a wave issues per step
  constexpr int AHEAD = 3;                   // operands read from LDS before their products
  extern __shared__ u32x4 tile_lds[];
  const uint32_t h = blockIdx.x % (uint32_t)a.kv_heads;
  const AttnItem it = attn_find_item<ROWS, WAVES>(a, blockIdx.x / (uint32_t)a.kv_heads,
                                              a.part_map != nullptr && blockIdx.x == 0);
  if (it.r < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int share = wave & 3;
  const AttnSeq x = attn_seq(a, it.r);
  const int32_t rows_all = x.n * a.group;
  const int32_t tiles = (rows_all + ROWS - 1) / ROWS;
  const int32_t tile = tiles - 1 - it.tile;  // the last tokens have the most keys: first
  const int32_t row0 = tile * ROWS;
  const int32_t rows = rows_all - row0 < ROWS ? rows_all - row0 : ROWS;

  u32x4 q[QT][KSTEPS];
  int32_t row_tok[QT];  // token of this lane's row, counted from the request's first new one
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int32_t i = (wave * QT + qt) * 32 + col;
    const int32_t p = row0 + (i < rows ? i : rows - 1);
    const int32_t j = p / a.group;
    row_tok[qt] = j;
    const int32_t head = (int32_t)h * a.group + (p - j * a.group);
    const char* src = reinterpret_cast<const char*>(a.q) +
                      ((int64_t)(x.q0 + j) * a.q_stride + (int64_t)head * a.head_size) * 2;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const int d = k * 16 + half * 8;
      q[qt][k] = !PAD || d < a.head_size ? *reinterpret_cast<const u32x4*>(src + d * 2)
                                         : u32x4{0, 0, 0, 0};
    }
  }
  // some row of the tile sees [span_lo, span_hi), every row of this wave [full_lo, full_hi)
  int32_t span_lo, span_hi, full_lo, full_hi, skip;
  attn_span(a, x, row0 / a.group, span_lo, skip);
  attn_span(a, x, (row0 + rows - 1) / a.group, skip, span_hi);
  {
    const int32_t i0 = wave * QT * 32, i1 = i0 + QT * 32 - 1;
    attn_span(a, x, (row0 + (i0 < rows ? i0 : rows - 1)) / a.group, skip, full_hi);
    attn_span(a, x, (row0 + (i1 < rows ? i1 : rows - 1)) / a.group, full_lo, skip);
  }
  span_lo = __builtin_amdgcn_readfirstlane(span_lo);
  span_hi = __builtin_amdgcn_readfirstlane(span_hi);
  full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  full_hi = __builtin_amdgcn_readfirstlane(full_hi);
  // steps of 64 keys, counted from a multiple of 64
  int32_t begin = span_lo & ~63, end = span_hi;
  if (it.parts > 1) {
    const int64_t b = begin + (int64_t)it.part * it.part_len;
    begin = b < span_hi ? (int32_t)b : span_hi;
    const int64_t e = b + it.part_len;
    end = e < span_hi ? (int32_t)e : span_hi;
  }
  const int32_t first = begin > span_lo ? begin : span_lo;  // keys [first, end) are loaded
  const int32_t steps = end > begin ? (end - begin + 63) / 64 : 0;

  f32x16 o[DTILES][QT];
  float ref[QT], l[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    ref[qt] = kRefStart;
    l[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][qt][i] = 0.f;
  }

  lds_char* const lds = (lds_char*)tile_lds;
  lds_char* const klds = lds;
  lds_char* const vlds = lds + Sh::kSteps * Sh::kStepBytes;
  lds_char* const ids = lds + Sh::kRingBytes + wave * (Sh::kIdSlots * 64);
  if constexpr (PAD) {  // chunks beyond the head are never loaded: they stay zero
    for (int i = tid * 16; i < Sh::kRingBytes; i += WAVES * 1024)
      *(__attribute__((address_space(3))) u32x4*)(lds + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }

  // ---- loads.  A share is sixteen keys or values of a step; a wave brings one share of each, or
  // (8 waves) waves 0-3 bring keys and waves 4-7 values.
  const char* src[ROLES];
  lds_char* dst[ROLES];
  uint32_t off[ROLES][Sh::kDmas];  // this lane's chunk of each load, from the share's first entry
  const int row_l = lane / Sh::kChunks, pos_l = lane % Sh::kChunks;
#pragma unroll
  for (int r = 0; r < ROLES; ++r) {
    const bool keys = ROLES == 2 ? r == 0 : wave < 4;
    src[r] = reinterpret_cast<const char*>(keys ? a.k_cache : a.v_cache) + (int64_t)h * a.head_size * 2;
    dst[r] = (keys ? klds : vlds) + share * (16 * Sh::kRowBytes);
#pragma unroll
    for (int n = 0; n < Sh::kDmas; ++n) {
      const int row = n * Sh::kRowsPerDma + row_l;
      off[r][n] = (uint32_t)(pos_l ^ (keys ? Sh::swz_k(row) : Sh::swz_v(row))) * 16u;
      if constexpr (PAGE16) off[r][n] += (uint32_t)row * (uint32_t)a.entry_stride;
    }
  }
  // chunk of off[r][n] inside the head's row
  auto chunk_of = [&](int r, int n) {
    return PAGE16 ? off[r][n] - (uint32_t)(n * Sh::kRowsPerDma + row_l) * (uint32_t)a.entry_stride
                  : off[r][n];
  };
  auto share_at = [&](int32_t j) { return begin + j * 64 + share * 16; };
  auto clamp_key = [&](int32_t t) { return t < first ? first : t < end ? t : end - 1; };
  auto load_ids = [&](int32_t j) {
    if constexpr (!PAGE16) {
      const int32_t* const from = a.kv_indices + x.kv0 + attn_page_of(a, clamp_key(share_at(j) + (lane & 15)));
      if (lane < 16) dma_asm4(from, ids + (j % Sh::kIdSlots) * 64);
    }
  };
  // PAGE16: the share of step j, or the nearest one that holds one of the keys [first, end), and its
  // page number (a scalar load, used one step later)
  const int32_t share_lo = first & ~15, share_hi = (end - 1) & ~15;
  auto share_base = [&](int32_t j) { return clamp_i32(share_at(j), share_lo, share_hi); };
  auto share_page = [&](int32_t j) {
    return PAGE16 ? a.kv_indices[x.kv0 + attn_page_of(a, share_base(j))] : 0;
  };
  auto load_step = [&](int32_t j, int32_t page) {
    const uint32_t slot = (uint32_t)j % Sh::kSteps * Sh::kStepBytes;
    if constexpr (PAGE16) {
      const int32_t t0 = share_base(j);
      const int64_t e = attn_clip_page(a, page) * a.page_stride +
                        (int64_t)(t0 - attn_page_of(a, t0) * a.page_size) * a.entry_stride;
      const bool inside = t0 >= first && t0 + 16 <= end;  // uniform over the wave
#pragma unroll
      for (int r = 0; r < ROLES; ++r) {
        const char* const base = src[r] + e;
        const uint32_t to = lds_addr(dst[r]) + slot;
        if (inside) {
#pragma unroll
          for (int n = 0; n < Sh::kDmas; ++n)
            if (!PAD || chunk_of(r, n) < (uint32_t)a.head_size * 2u) dma_asm16(base, off[r][n], to, n * 1024);
        } else {
#pragma unroll
          for (int n = 0; n < Sh::kDmas; ++n) {
            const int32_t row = clamp_key(t0 + n * Sh::kRowsPerDma + row_l) - t0;
            const uint32_t c = chunk_of(r, n);
            if (!PAD || c < (uint32_t)a.head_size * 2u)
              dma_asm16(base, (uint32_t)row * (uint32_t)a.entry_stride + c, to, n * 1024);
          }
        }
      }
    } else {
      const int32_t t = clamp_key(share_at(j) + (lane & 15));
      page = *(const __attribute__((address_space(3))) int32_t*)(
          ids + (j % Sh::kIdSlots) * 64 + (lane & 15) * 4);
      const int64_t e = attn_clip_page(a, page) * a.page_stride +
                        (int64_t)(t - attn_page_of(a, t) * a.page_size) * a.entry_stride;
      const int32_t e_lo = (int32_t)e, e_hi = (int32_t)(e >> 32);
#pragma unroll
      for (int n = 0; n < Sh::kDmas; ++n) {
        const int row = n * Sh::kRowsPerDma + row_l;
        const int64_t s = (int64_t)(((uint64_t)(uint32_t)__shfl(e_hi, row, 64) << 32) |
                                    (uint32_t)__shfl(e_lo, row, 64));
#pragma unroll
        for (int r = 0; r < ROLES; ++r)
          if (!PAD || off[r][n] < (uint32_t)a.head_size * 2u)
            dma_asm16(src[r] + s + off[r][n], lds_addr(dst[r]) + slot, n * 1024);
      }
    }
  };

  // ---- operand reads
  uint32_t kread[KSTEPS], vread[DTILES];
#pragma unroll
  for (int k = 0; k < KSTEPS; ++k)
    kread[k] = lds_addr(klds) + col * Sh::kRowBytes + (((k * 2 + half) ^ Sh::swz_k(col)) * 16);
  const int vlane = lane & 15, vrow = half * 4 + (vlane >> 2);
#pragma unroll
  for (int dt = 0; dt < DTILES; ++dt) {
    const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((vlane >> 1) & 1);
    vread[dt] = lds_addr(vlds) + vrow * Sh::kRowBytes + (chunk ^ Sh::swz_v(vrow)) * 16 + (vlane & 1) * 8;
  }
  auto read_k = [&](uint32_t step_at, int sub, int k) {
    return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(
        kread[k] + step_at + sub * (32 * Sh::kRowBytes));
  };
  auto read_v = [&](uint32_t step_at, int sub, int ks, int dt) {  // ks: 16 of the 32 keys
    const lds_char* const p = (const lds_char*)(uintptr_t)(vread[dt] + step_at) +
                              (sub * 32 + ks * 16) * Sh::kRowBytes;
    const u32x2 x0 = lds_read_tr_b64(p), x1 = lds_read_tr_b64(p + 8 * Sh::kRowBytes);
    return u32x4{x0[0], x0[1], x1[0], x1[1]};
  };

  // ---- 32 keys u at a time: keys 32 * (u & 1) of step u / 2
  struct Scores { f32x16 s[QT]; };
  auto mask = [&](int32_t u, Scores& sc) {
    const int32_t t0 = begin + u * 32;
    if (t0 >= full_lo && t0 + 32 <= full_hi && t0 + 32 <= end) return;  // uniform over the wave
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      int32_t lo, hi;
      attn_span(a, x, row_tok[qt], lo, hi);
      const int32_t top = (hi < end ? hi : end) - t0 - 4 * half, low = lo - t0 - 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int32_t t = 8 * (i / 4) + i % 4;
        sc.s[qt][i] = t >= low && t < top ? sc.s[qt][i] : -INFINITY;
      }
    }
  };
  // raises the reference of rows whose new maximum (of raw scores) passes it by more than kRaise
  auto raise = [&](float (&top)[QT]) {
    bool need = false;
    float z[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      auto w = __builtin_amdgcn_permlane32_swap(as_u32(top[qt]), as_u32(top[qt]), false, false);
      z[qt] = fmaxf(as_f32(w[0]), as_f32(w[1])) * a.scale_log2;
      need |= z[qt] > ref[qt] + kRaise;
    }
    if (__builtin_amdgcn_ballot_w64(need) == 0) return;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float next = fmaxf(ref[qt], z[qt]);
      const float keep = __builtin_amdgcn_exp2f(ref[qt] - next);
      ref[qt] = next;
      l[qt] *= keep;
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt) o[dt][qt] *= keep;
    }
  };
  // The scores of keys u become probabilities and meet the values, while (MORE) those of keys u + 1
  // are formed and their maximum is taken.
  auto body = [&](int32_t u, auto sub, Scores& cur, Scores& next, auto more) {
    constexpr bool MORE = decltype(more)::value;
    constexpr int SUB = decltype(sub)::value;  // u & 1
    const uint32_t v_at = (uint32_t)u / 2 % Sh::kSteps * Sh::kStepBytes;
    const uint32_t k_at = ((uint32_t)u + 1) / 2 % Sh::kSteps * Sh::kStepBytes;
    constexpr int PV = 2 * DTILES;      // operands of the output's products
    constexpr int PER = QT * 16 / KSTEPS;  // probabilities per operand of the next scores
    constexpr int PERM = QT * 16 / PV;  // scores that enter the maximum per operand
    u32x4 p[QT][2], kf[AHEAD + 1], vf[AHEAD + 1];
    if constexpr (MORE) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int i = 0; i < 16; ++i) next.s[qt][i] = 0.f;
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) kf[n] = read_k(k_at, SUB ^ 1, n);
    }
#pragma unroll
    for (int n = 0; n < KSTEPS; ++n) {
      if constexpr (MORE) {
        if (n + AHEAD < KSTEPS) kf[(n + AHEAD) % (AHEAD + 1)] = read_k(k_at, SUB ^ 1, n + AHEAD);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          next.s[qt] = mfma32x16<DT>(kf[n % (AHEAD + 1)], q[qt][n], next.s[qt]);
      }
      if (n >= KSTEPS - AHEAD) {
        const int i = n - (KSTEPS - AHEAD);
        vf[i] = read_v(v_at, SUB, i / DTILES, i % DTILES);
      }
#pragma unroll
      for (int e = n * PER; e < (n + 1) * PER; e += 2) {
        const int qt = e / 16, i = e % 16;
        const float z0 = __builtin_amdgcn_exp2f(fmaf(cur.s[qt][i], a.scale_log2, -ref[qt]));
        const float z1 = __builtin_amdgcn_exp2f(fmaf(cur.s[qt][i + 1], a.scale_log2, -ref[qt]));
        l[qt] += z0 + z1;
        uint32_t w = pack2<DT>(z0, z1);
        asm volatile("" : "+v"(w), "+v"(l[qt]));  // made here, not where they are used
        p[qt][i / 8][i / 2 % 4] = w;
      }
      fence_order();
    }
    if constexpr (MORE) mask(u + 1, next);
    float top[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) top[qt] = -INFINITY;
#pragma unroll
    for (int n = 0; n < PV; ++n) {
      if (n + AHEAD < PV)
        vf[(n + AHEAD) % (AHEAD + 1)] = read_v(v_at, SUB, (n + AHEAD) / DTILES, (n + AHEAD) % DTILES);
      const int ks = n / DTILES, dt = n % DTILES;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) o[dt][qt] = mfma32x16<DT>(vf[n % (AHEAD + 1)], p[qt][ks], o[dt][qt]);
      if constexpr (MORE) {
#pragma unroll
        for (int e = n * PERM; e < (n + 1) * PERM; e += 2) {
          const int qt = e / 16, i = e % 16;
          top[qt] = fmaxf(fmaxf(top[qt], next.s[qt][i]), next.s[qt][i + 1]);
        }
      }
      fence_order();
    }
    if constexpr (MORE) raise(top);
  };

  if (steps > 0) {
    if constexpr (!PAGE16) {
#pragma unroll
      for (int i = 0; i < 6; ++i) load_ids(i);
      wait_vmcnt<0>();
    }
    int32_t page = share_page(3);  // of the step that is asked for next
    load_step(0, share_page(0));
    load_step(1, share_page(1));
    load_step(2, share_page(2));
    wait_vmcnt<2 * ROLES * Sh::kDmas>();  // step 0
    wave_barrier();
    Scores s0, s1;
    {
      float top[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s0.s[qt][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        const u32x4 kk = read_k(0, 0, k);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s0.s[qt] = mfma32x16<DT>(kk, q[qt][k], s0.s[qt]);
      }
      mask(0, s0);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        top[qt] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) top[qt] = fmaxf(top[qt], s0.s[qt][i]);
      }
      raise(top);
    }
    // Step j needs keys up to j + 1 and values j: all but what step j - 1 has asked for (before the
    // first: step 2).
    int32_t j = 0;
    wait_vmcnt<ROLES * Sh::kDmas>();
    while (j + 1 < steps) {
      wave_barrier();
      load_step(j + 3, page);
      load_ids(j + 6);
      page = share_page(j + 4);
      body(2 * j, std::integral_constant<int, 0>{}, s0, s1, std::true_type{});
      body(2 * j + 1, std::integral_constant<int, 1>{}, s1, s0, std::true_type{});
      wait_vmcnt<kOps>();
      ++j;
    }
    wave_barrier();
    body(2 * j, std::integral_constant<int, 0>{}, s0, s1, std::true_type{});
    body(2 * j + 1, std::integral_constant<int, 1>{}, s1, s0, std::false_type{});
    wait_vmcnt<0>();  // nothing may land in LDS after this workgroup has left it
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    auto w = __builtin_amdgcn_permlane32_swap(as_u32(l[qt]), as_u32(l[qt]), false, false);
    l[qt] = as_f32(w[0]) + as_f32(w[1]);
    const int32_t i = (wave * QT + qt) * 32 + col;
    if (i >= rows) continue;
    if (it.parts > 1) {
      // items are counted in launch order, the join counts tiles from the first row on
      const int64_t item = (int64_t)it.index - it.part - (int64_t)it.tile * it.parts +
                           (int64_t)tile * it.parts + it.part;
      const int64_t slot = (item * a.kv_heads + h) * ROWS + i;
      if (half == 0) {
        a.part_ml[slot * 2] = ref[qt];
        a.part_ml[slot * 2 + 1] = l[qt];
      }
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int d = dt * 32 + b * 8 + half * 4;
          if (!PAD || d < a.head_size)
            *reinterpret_cast<f32x4*>(a.part_o + slot * a.head_size + d) =
                f32x4{o[dt][qt][b * 4], o[dt][qt][b * 4 + 1], o[dt][qt][b * 4 + 2], o[dt][qt][b * 4 + 3]};
        }
    } else {
      const float inv = l[qt] == 0.f ? 0.f : 1.f / l[qt];
      const int64_t tok = x.q0 + row_tok[qt];
      const int32_t head = (int32_t)h * a.group + (row0 + i - row_tok[qt] * a.group);
      char* const dst = reinterpret_cast<char*>(a.out) +
                        (tok * a.out_stride + (int64_t)head * a.head_size) * 2;
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int d = dt * 32 + b * 8 + half * 4;
          if (!PAD || d < a.head_size)
            *reinterpret_cast<u32x2*>(dst + d * 2) =
                u32x2{pack2<DT>(o[dt][qt][b * 4] * inv, o[dt][qt][b * 4 + 1] * inv),
                      pack2<DT>(o[dt][qt][b * 4 + 2] * inv, o[dt][qt][b * 4 + 3] * inv)};
        }
      if (a.lse && half == 0)
        a.lse[tok * a.heads + head] = attn_lse(ref[qt], l[qt]);
    }
  }
}

template <int DT, int DP, int WAVES, int QT, bool PAD, bool PAGE16>
static int launch_tile_pages(const PagedAttnArgs& a, int64_t groups, hipStream_t st) {
  constexpr int bytes = TileShape<DP>::kBytes;
  if (!allow_lds<paged_attn_tile_kernel<DT, DP, WAVES, QT, PAD, PAGE16>>(bytes)) return SARATHI_ERR_LAUNCH;
  hipLaunchKernelGGL((paged_attn_tile_kernel<DT, DP, WAVES, QT, PAD, PAGE16>), dim3((unsigned)groups),
                     dim3(WAVES * 64), bytes, st, a);
  return launch_status();
}
template <int DT, int DP, int WAVES, int QT>
static int launch_tile(const PagedAttnArgs& a, int64_t groups, hipStream_t st) {
  // offsets inside a share are 32-bit
  const bool page16 = a.page_size % 16 == 0 && a.entry_stride < (1 << 26);
  if (a.head_size == DP)
    return page16 ? launch_tile_pages<DT, DP, WAVES, QT, false, true>(a, groups, st)
                  : launch_tile_pages<DT, DP, WAVES, QT, false, false>(a, groups, st);
  return page16 ? launch_tile_pages<DT, DP, WAVES, QT, true, true>(a, groups, st)
                : launch_tile_pages<DT, DP, WAVES, QT, true, false>(a, groups, st);
}
template <int DT>
static int launch_tile_heads(const PagedAttnArgs& a, int rows, int64_t groups, hipStream_t st) {
  if (a.head_size <= 64)
    return rows == 256 ? launch_tile<DT, 64, 8, 1>(a, groups, st) : launch_tile<DT, 64, 4, 1>(a, groups, st);
  return rows == 256 ? launch_tile<DT, 128, 8, 1>(a, groups, st) : launch_tile<DT, 128, 4, 1>(a, groups, st);
}

int launch_attn_tiles(const PagedAttnArgs& a, int dtype, int rows, int64_t groups, hipStream_t st) {
  return dtype == kBF16 ? launch_tile_heads<kBF16>(a, rows, groups, st)
                        : launch_tile_heads<kF16>(a, rows, groups, st);
}

}  // namespace sarathi_hip
