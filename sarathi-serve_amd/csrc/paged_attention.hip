// Attention of the new tokens of a hybrid batch over their requests' pages (paged_attn.h has the
// formulas).  Stands for the two flashinfer wrappers that the reference plans and runs per batch
// (sarathi/model_executor/attention/flashinfer_attention_wrapper.py:169-209, 262-304): one entry
// for chunks of new tokens and for single decode tokens alike.
//
// This file holds the kernel for few rows (decode steps), the plain kernel for any head size and
// alignment, the kernel that joins the parts of a cut context, and the entry point that chooses.
#include "launch.h"
#include "paged_attn.h"
#include "paged_attn_tiles.h"

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
  if (tok >= clamp_i32(a.qo_indptr[a.seqs], 0, a.tokens) || tok < a.qo_indptr[0]) return;
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

// ---- few rows: decode steps --------------------------------------------------------------------
//
// Bound by the bytes of the keys and values.  A workgroup is four waves that share one tile of
// 16 * RT rows and stream its keys 16 at a time, each wave through a ring in LDS of its own
// (kFewStages blocks of 16 keys and values, filled by loads that write LDS directly), so that no
// wave waits for another before the end: there the four states are joined through LDS.
//   scores  S^T = K Q^T: keys as rows, the tile's rows as columns, so a row's softmax stays inside
//           four lanes (lane & 15 names the row), and the probabilities come out of the product in
//           the very layout in which
//   output  O^T += V^T P^T takes them: no exchange between lanes, V is transposed by the LDS read.
// Chunks of 16 bytes are stored swizzled, K by XOR with the row so that sixteen rows' same chunk
// lie in different banks, V by XOR of chunk pairs so that eight rows' same sixteen elements do.
// Probabilities are rounded to the cache's type for the product (at most half a step each, of
// values up to 1); maximum, sum and output stay in 32 bits.
template <int DP> struct FewShape {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kChunks = DP / 8;            // 16-byte chunks of a row
  static constexpr int kRowsPerDma = 64 / kChunks;  // rows one load instruction moves
  static constexpr int kDmas = 16 / kRowsPerDma;    // per block of 16 keys (and as many for values)
  static constexpr int kStages = DP >= 256 ? 2 : DP == 128 ? 2 : 4;
  static constexpr int kBlockBytes = 16 * kRowBytes;
  static constexpr int kIdSlots = 2 * kStages;
  static constexpr int kWaveBytes = kStages * 2 * kBlockBytes + kIdSlots * 256;
  SK_DEV static int swz_k(int row) { return DP == 64 ? (row >> 1) & 7 : row & 15; }
  SK_DEV static int swz_v(int row) { return DP == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1; }
};

template <int DT, int DP, int RT, bool PAD>
__global__ __launch_bounds__(256) void paged_attn_few_kernel(PagedAttnArgs a) {
  using Sh = FewShape<DP>;
  constexpr int ROWS = 16 * RT, S = Sh::kStages, KSTEPS = DP / 32, DTILES = DP / 16;
  constexpr int kOps = 2 * Sh::kDmas + 1;  // loads a block takes: keys, values, page numbers
  extern __shared__ u32x4 few_lds[];
  const uint32_t h = blockIdx.x % (uint32_t)a.kv_heads;
  const AttnItem it = attn_find_item<ROWS, 4>(a, blockIdx.x / (uint32_t)a.kv_heads,
                                              a.part_map != nullptr && blockIdx.x == 0);
  if (it.r < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AttnSeq x = attn_seq(a, it.r);
  const int32_t rows_all = x.n * a.group, row0 = it.tile * ROWS;
  const int32_t rows = rows_all - row0 < ROWS ? rows_all - row0 : ROWS;

  // this lane's rows (one per row tile): query operand, span of keys
  u32x4 q[RT][KSTEPS];
  int32_t lo[RT], hi[RT], tok[RT], head[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int32_t i = rt * 16 + col;
    const int32_t p = row0 + (i < rows ? i : rows - 1);
    const int32_t j = p / a.group;
    tok[rt] = x.q0 + j;
    head[rt] = (int32_t)h * a.group + (p - j * a.group);
    attn_span(a, x, j, lo[rt], hi[rt]);
    const char* src = reinterpret_cast<const char*>(a.q) +
                      ((int64_t)tok[rt] * a.q_stride + (int64_t)head[rt] * a.head_size) * 2;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const int d = k * 32 + g * 8;
      q[rt][k] = d < a.head_size ? *reinterpret_cast<const u32x4*>(src + d * 2) : u32x4{0, 0, 0, 0};
    }
  }
  // some row sees [span_lo, span_hi), every row [full_lo, full_hi)
  int32_t span_lo, span_hi, full_lo, full_hi;
  attn_span(a, x, row0 / a.group, span_lo, full_hi);
  attn_span(a, x, (row0 + rows - 1) / a.group, full_lo, span_hi);
  full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  full_hi = __builtin_amdgcn_readfirstlane(full_hi);
  const int32_t begin = __builtin_amdgcn_readfirstlane(
      it.parts > 1 ? (int32_t)min((int64_t)span_hi, span_lo + (int64_t)it.part * it.part_len) : span_lo);
  const int32_t end = __builtin_amdgcn_readfirstlane(
      it.parts > 1 ? (int32_t)min((int64_t)span_hi, (int64_t)begin + it.part_len) : span_hi);

  float m[RT], l[RT];
  f32x4 o[RT][DTILES];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  lds_char* const base = (lds_char*)few_lds + wave * Sh::kWaveBytes;
  lds_char* const ids = base + S * 2 * Sh::kBlockBytes;
  if constexpr (PAD) {  // chunks beyond the head are never loaded: they stay zero
    for (int i = lane * 16; i < S * 2 * Sh::kBlockBytes; i += 1024)
      *(__attribute__((address_space(3))) u32x4*)(base + i) = u32x4{0, 0, 0, 0};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // blocks of 16 keys are dealt to the waves in turn
  const int32_t total = end - begin;
  const int32_t nb = total > wave * 16 ? (total - wave * 16 + 63) / 64 : 0;
  auto key_of = [&](int32_t b, int row) {  // past the end: the last key again
    const int32_t t = begin + (b * 4 + wave) * 16 + row;
    return t < end ? t : end - 1;
  };
  auto load_ids = [&](int32_t b) {
    const int32_t* src = a.kv_indices + x.kv0 + attn_page_of(a, key_of(b, col));
    dma_to_lds<4>(src, ids + (b % Sh::kIdSlots) * 256);  // four copies, no lane off
  };
  const char* const kc = reinterpret_cast<const char*>(a.k_cache) + (int64_t)h * a.head_size * 2;
  const char* const vc = reinterpret_cast<const char*>(a.v_cache) + (int64_t)h * a.head_size * 2;
  auto load_block = [&](int32_t b) {
    const int32_t t = key_of(b, col);
    const int32_t pg = attn_page_of(a, t);
    const int32_t page = attn_clip_page(
        a, *(const __attribute__((address_space(3))) int32_t*)(ids + (b % Sh::kIdSlots) * 256 + col * 4));
    const int64_t off = page * a.page_stride + (int64_t)(t - pg * a.page_size) * a.entry_stride;
    const int32_t off_lo = (int32_t)off, off_hi = (int32_t)(off >> 32);
    lds_char* const dst = base + (b % S) * 2 * Sh::kBlockBytes;
#pragma unroll
    for (int n = 0; n < Sh::kDmas; ++n) {
      const int row = n * Sh::kRowsPerDma + lane / Sh::kChunks, pos = lane % Sh::kChunks;
      const int64_t e = (int64_t)(((uint64_t)(uint32_t)__shfl(off_hi, row, 64) << 32) |
                                  (uint32_t)__shfl(off_lo, row, 64));
      const int ck = pos ^ Sh::swz_k(row), cv = pos ^ Sh::swz_v(row);
      if (!PAD || ck * 8 < a.head_size) dma_to_lds<16>(kc + e + ck * 16, dst + n * 1024);
      if (!PAD || cv * 8 < a.head_size)
        dma_to_lds<16>(vc + e + cv * 16, dst + Sh::kBlockBytes + n * 1024);
    }
  };

  if (nb > 0) {
#pragma unroll
    for (int i = 0; i < S; ++i) load_ids(i);
    wait_vmcnt<0>();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      load_block(i);
      load_ids(S + i);
    }
  }
  for (int32_t b = 0; b < nb; ++b) {
    // everything up to this block's values and the page numbers of block b + S
    wait_vmcnt<(S - 1) * kOps>();
    const lds_char* const kb = base + (b % S) * 2 * Sh::kBlockBytes;
    const lds_char* const vb = kb + Sh::kBlockBytes;
    const int32_t t0 = begin + (b * 4 + wave) * 16;
    f32x4 s[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const u32x4 kk = *(const __attribute__((address_space(3))) u32x4*)(
          kb + col * Sh::kRowBytes + (((k * 4 + g) ^ Sh::swz_k(col)) * 16));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt] = mfma16x32<DT>(kk, q[rt][k], s[rt]);
    }
    const bool whole = t0 >= full_lo && t0 + 16 <= full_hi && t0 + 16 <= end;
    u32x2 p[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float z[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = s[rt][j] * a.scale_log2;
      if (!whole) {
        const int32_t top = hi[rt] < end ? hi[rt] : end;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int32_t t = t0 + g * 4 + j;
          z[j] = t >= lo[rt] && t < top ? z[j] : -INFINITY;
        }
      }
      const float top = fmaxf(m[rt], group_max(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]))));
      const float ref = top == -INFINITY ? 0.f : top;
      const float keep = __builtin_amdgcn_exp2f(m[rt] - ref);
      m[rt] = top;
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = __builtin_amdgcn_exp2f(z[j] - ref);
      l[rt] = l[rt] * keep + ((z[0] + z[1]) + (z[2] + z[3]));
      p[rt] = u32x2{pack2<DT>(z[0], z[1]), pack2<DT>(z[2], z[3])};
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt) o[rt][dt] *= keep;
    }
    const int vrow = g * 4 + (col >> 2);
    const uint32_t vaddr = lds_addr(vb + vrow * Sh::kRowBytes + (col & 1) * 8);
#pragma unroll
    for (int d0 = 0; d0 < DTILES; d0 += 4) {
      uint32_t at[4];
      u32x2 vv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        at[i] = vaddr + ((((d0 + i) * 2 + ((col >> 1) & 1)) ^ Sh::swz_v(vrow)) * 16);
      lds_read_tr4(at, vv);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][d0 + i] = mfma16x16<DT>(vv[i], p[rt], o[rt][d0 + i]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the block is read: its place can be filled
    load_block(b + S);
    load_ids(b + 2 * S);
  }
  wait_vmcnt<0>();
  __syncthreads();

  // join the four waves: 2 and 3 hand over to 0 and 1, then 1 to 0
  typedef __attribute__((address_space(3))) float lds_float;
  constexpr int kState = 64 * (2 + DTILES * 4) * RT;  // floats a wave hands over
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) l[rt] = group_sum(l[rt]);
#pragma unroll
  for (int step = 2; step > 0; step >>= 1) {
    lds_float* const box = (lds_float*)few_lds + (wave & (step - 1)) * kState;
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        lds_float* const b = box + rt * 64 * (2 + DTILES * 4);
        b[lane] = m[rt];
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
        lds_float* const b = box + rt * 64 * (2 + DTILES * 4);
        const float m2 = b[lane], l2 = b[64 + lane];
        const float top = fmaxf(m[rt], m2), ref = top == -INFINITY ? 0.f : top;
        const float w1 = __builtin_amdgcn_exp2f(m[rt] - ref), w2 = __builtin_amdgcn_exp2f(m2 - ref);
        m[rt] = top;
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
    if (rt * 16 + col >= rows) continue;
    if (it.parts > 1) {
      const int64_t slot = ((int64_t)it.index * a.kv_heads + h) * ROWS + rt * 16 + col;
      if (g == 0) {
        a.part_ml[slot * 2] = m[rt];
        a.part_ml[slot * 2 + 1] = l[rt];
      }
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
        if (dt * 16 + g * 4 < a.head_size)
          *reinterpret_cast<f32x4*>(a.part_o + slot * a.head_size + dt * 16 + g * 4) = o[rt][dt];
    } else {
      const float inv = l[rt] == 0.f ? 0.f : 1.f / l[rt];
      char* const dst = reinterpret_cast<char*>(a.out) +
                        ((int64_t)tok[rt] * a.out_stride + (int64_t)head[rt] * a.head_size) * 2;
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
        if (dt * 16 + g * 4 < a.head_size)
          *reinterpret_cast<u32x2*>(dst + (dt * 16 + g * 4) * 2) =
              u32x2{pack2<DT>(o[rt][dt][0] * inv, o[rt][dt][1] * inv),
                    pack2<DT>(o[rt][dt][2] * inv, o[rt][dt][3] * inv)};
      if (a.lse && g == 0) a.lse[(int64_t)tok[rt] * a.heads + head[rt]] = attn_lse(m[rt], l[rt]);
    }
  }
}

// ---- joins the parts of cut contexts -------------------------------------------------------------
//
// One wave per token and query head; parts whose sum is zero have no output.  Parts are added in
// their order, so results do not depend on which workgroup ran when.
template <int DT, int VALS>  // VALS elements of the head per lane
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttnArgs a, int32_t rows_per_tile) {
  const int lane = threadIdx.x & 63;
  const int32_t head = (int32_t)blockIdx.y * 4 + (threadIdx.x >> 6);
  const int32_t tok = (int32_t)blockIdx.x;
  if (head >= a.heads) return;
  if (tok >= clamp_i32(a.qo_indptr[a.seqs], 0, a.tokens) || tok < a.qo_indptr[0]) return;
  int32_t r = 0, hi_r = a.seqs;
  while (hi_r - r > 1) {
    const int32_t mid = (r + hi_r) >> 1;
    if (a.qo_indptr[mid] <= tok) r = mid; else hi_r = mid;
  }
  const int32_t parts = a.part_map[a.seqs + r];
  if (parts <= 1) return;
  const AttnSeq x = attn_seq(a, r);
  if (tok < x.q0 || tok >= x.q0 + x.n) return;
  const int32_t h = head / a.group;
  const int32_t row = (tok - x.q0) * a.group + (head - h * a.group);
  const int32_t tile = row / rows_per_tile, in_tile = row - tile * rows_per_tile;
  const int64_t item0 = (int64_t)a.part_map[r] + (int64_t)tile * parts;
  auto slot_of = [&](int32_t p) {
    return ((item0 + p) * a.kv_heads + h) * rows_per_tile + in_tile;
  };
  float m = -INFINITY;
  for (int32_t p = lane; p < parts; p += 64) {
    const int64_t s = slot_of(p);
    if (a.part_ml[s * 2 + 1] != 0.f) m = fmaxf(m, a.part_ml[s * 2]);
  }
  m = wave64_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[VALS] = {};
  const int d0 = lane * VALS;
  const bool on = d0 < a.head_size;
#pragma unroll 4
  for (int32_t p = 0; p < parts; ++p) {
    const int64_t s = slot_of(p);
    const float pl = a.part_ml[s * 2 + 1];
    const float w = pl != 0.f ? __builtin_amdgcn_exp2f(a.part_ml[s * 2] - ref) : 0.f;
    l += pl * w;
    if (on && pl != 0.f) {
#pragma unroll
      for (int i = 0; i < VALS; ++i) o[i] = fmaf(a.part_o[s * a.head_size + d0 + i], w, o[i]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (on) {
    const int64_t base = (int64_t)tok * a.out_stride + (int64_t)head * a.head_size + d0;
#pragma unroll
    for (int i = 0; i < VALS; ++i) store_elem<DT>(a.out, base + i, o[i] * inv);
  }
  if (a.lse && lane == 0) a.lse[(int64_t)tok * a.heads + head] = attn_lse(m, l);
}

template <int DT, int DP, int RT>
static int launch_few(const PagedAttnArgs& a, int64_t groups, hipStream_t st) {
  constexpr int ring = 4 * FewShape<DP>::kWaveBytes;
  constexpr int join = 2 * 64 * (2 + DP / 16 * 4) * RT * 4;
  constexpr int bytes = ring > join ? ring : join;
  const dim3 grid((unsigned)groups), block(256);
  if (a.head_size == DP) {
    if (!allow_lds<paged_attn_few_kernel<DT, DP, RT, false>>(bytes)) return SARATHI_ERR_LAUNCH;
    hipLaunchKernelGGL((paged_attn_few_kernel<DT, DP, RT, false>), grid, block, bytes, st, a);
  } else {
    if (!allow_lds<paged_attn_few_kernel<DT, DP, RT, true>>(bytes)) return SARATHI_ERR_LAUNCH;
    hipLaunchKernelGGL((paged_attn_few_kernel<DT, DP, RT, true>), grid, block, bytes, st, a);
  }
  return launch_status();
}
template <int DT, int DP>
static int launch_few_rows(const PagedAttnArgs& a, int row_tiles, int64_t groups, hipStream_t st) {
  if (row_tiles == 1) return launch_few<DT, DP, 1>(a, groups, st);
  if constexpr (DP <= 128)
    if (row_tiles == 4) return launch_few<DT, DP, 4>(a, groups, st);
  return launch_few<DT, DP, 2>(a, groups, st);
}
template <int DT>
static int launch_few_heads(const PagedAttnArgs& a, int row_tiles, int64_t groups, hipStream_t st) {
  if (a.head_size <= 64) return launch_few_rows<DT, 64>(a, row_tiles, groups, st);
  if (a.head_size <= 128) return launch_few_rows<DT, 128>(a, row_tiles, groups, st);
  return launch_few_rows<DT, 256>(a, row_tiles, groups, st);
}

template <int DT>
static int launch_join(const PagedAttnArgs& a, int rows_per_tile, hipStream_t st) {
  const dim3 grid((unsigned)a.tokens, (unsigned)((a.heads + 3) / 4));
  if (a.head_size <= 64)
    hipLaunchKernelGGL((paged_attn_join_kernel<DT, 1>), grid, dim3(256), 0, st, a, rows_per_tile);
  else if (a.head_size <= 128)
    hipLaunchKernelGGL((paged_attn_join_kernel<DT, 2>), grid, dim3(256), 0, st, a, rows_per_tile);
  else
    hipLaunchKernelGGL((paged_attn_join_kernel<DT, 4>), grid, dim3(256), 0, st, a, rows_per_tile);
  return launch_status();
}

// ---- what a call launches ------------------------------------------------------------------------

// The requests of a batch fall into two classes by their rows (new tokens times query heads per key
// head): few rows, and chunks, which take the tile kernel.  All sizes here are known on the host.
struct AttnClass {
  int rows;            // rows per tile, 0: the class is empty
  int32_t min_rows, max_rows;
  int64_t tiles;       // at most so many tiles per key head
  int32_t target, min_part;
  int64_t items;       // at most so many items per key head
  int64_t map_bytes, ml_bytes, o_bytes;  // of the workspace
  int64_t bytes() const { return map_bytes + ml_bytes + o_bytes; }
};
struct AttnPlan {
  AttnClass few, tile;
};
static int64_t round256(int64_t v) { return (v + 255) & ~(int64_t)255; }

// Aims at `items` work items per key head, of at least min_part keys each.
static void plan_parts(AttnClass& c, int64_t items, int32_t min_part, int64_t seqs,
                       int64_t capacity, int kv_heads, int head_size) {
  const int64_t most = c.tiles * (capacity / min_part);  // no sequence is longer than all pages
  c.min_part = min_part;
  c.target = (int32_t)(items < most ? items : most);
  c.items = c.tiles + c.target;
  if (c.target <= 0) return;
  c.map_bytes = round256((2 * seqs + 1) * 4);
  c.ml_bytes = round256(c.items * kv_heads * c.rows * 8);
  c.o_bytes = round256(c.items * kv_heads * c.rows * head_size * 4);
}

static AttnPlan plan_attention(int64_t tokens, int64_t seqs, int64_t indices, int heads,
                               int kv_heads, int head_size, int page_size, int64_t max_query_len) {
  AttnPlan p{};
  const int group = heads / kv_heads;
  const int64_t longest = max_query_len > 0 && max_query_len < tokens ? max_query_len : tokens;
  const int64_t most_rows = longest * group, all_rows = tokens * group;
  const int64_t capacity = indices * page_size;
  const int units = compute_units();
  const int few_limit = head_size > 128 ? 32 : 64;
  AttnClass& f = p.few;
  AttnClass& t = p.tile;
  f.min_rows = 1;
  if (most_rows <= few_limit || head_size > 128) {
    // all requests in tiles of few rows (max_query_len may be wrong: any number of tiles each)
    f.rows = most_rows <= 16 ? 16 : most_rows <= 32 ? 32 : few_limit;
    f.max_rows = 0x7fffffff;
    f.tiles = all_rows / f.rows + seqs;
  } else {
    // single tokens in one tile each, longer requests in large tiles
    f.rows = group <= 16 ? 16 : group <= 32 ? 32 : few_limit;
    f.max_rows = f.rows;
    f.tiles = seqs;
    t.min_rows = f.rows + 1;
    t.max_rows = 0x7fffffff;
    t.rows = all_rows / 256 * kv_heads >= units ? 256 : 128;
    const int64_t chunks = seqs < all_rows / t.min_rows ? seqs : all_rows / t.min_rows;
    t.tiles = all_rows / t.rows + chunks;
    const int64_t fill = 2 * (int64_t)units / kv_heads;
    plan_parts(t, t.tiles < fill ? (fill > 0 ? fill : 1) : 0, 512, seqs, capacity, kv_heads, head_size);
  }
  if (f.tiles > all_rows) f.tiles = all_rows;
  const int64_t fill = 2 * (int64_t)units / kv_heads;
  plan_parts(f, fill > 0 ? fill : 1, 128, seqs, capacity, kv_heads, head_size);
  return p;
}

// Launches one class; `ws` is its part of the workspace or null.
template <typename Launch>
static int run_class(PagedAttnArgs a, const AttnClass& c, char* ws, int dtype, hipStream_t st,
                     Launch launch) {
  if (c.rows == 0) return SARATHI_OK;
  a.min_rows = c.min_rows;
  a.max_rows = c.max_rows;
  const bool cut = c.target > 0 && ws;
  if (cut) {
    a.part_map = reinterpret_cast<int32_t*>(ws);
    a.part_ml = reinterpret_cast<float*>(ws + c.map_bytes);
    a.part_o = reinterpret_cast<float*>(ws + c.map_bytes + c.ml_bytes);
    a.target = c.target;
    a.min_part = c.min_part;
  }
  const int64_t groups = (cut ? c.items : c.tiles) * a.kv_heads;
  if (groups > 0x7fffffffLL) return SARATHI_ERR_UNSUPPORTED;
  if (groups == 0) return SARATHI_OK;
  const int rc = launch(a, groups);
  if (rc != SARATHI_OK || !cut) return rc;
  return dtype == kBF16 ? launch_join<kBF16>(a, c.rows, st) : launch_join<kF16>(a, c.rows, st);
}

}  // namespace sarathi_hip

using namespace sarathi_hip;

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
  return p.few.bytes() + p.tile.bytes();
}

extern "C" int sarathi_paged_attention(
    const void* query, const void* k_cache, const void* v_cache, void* out, float* lse,
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t num_tokens, int64_t num_seqs, int64_t num_kv_indices,
    int64_t num_pages, int num_heads, int num_kv_heads, int head_size, int page_size,
    int64_t query_stride, int64_t out_stride, int64_t page_stride, int64_t entry_stride,
    float sm_scale, int causal, int64_t window_left, int64_t max_query_len, void* workspace,
    int64_t workspace_bytes, int dtype, void* stream) {
  if (!attn_sizes_ok(num_tokens, num_seqs, num_kv_indices, num_heads, num_kv_heads, head_size,
                     page_size) || num_pages < 0)
    return SARATHI_ERR_INVALID_ARG;
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
  if (num_tokens == 0 || num_seqs == 0) return SARATHI_OK;
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
  a.scale_log2 = sm_scale * kLog2e;
  hipStream_t st = (hipStream_t)stream;
  const bool vec = head_size % 8 == 0 && aligned16(query) && aligned16(k_cache) &&
                   aligned16(v_cache) && aligned16(out) && query_stride % 8 == 0 &&
                   out_stride % 4 == 0 && page_stride % 8 == 0 && entry_stride % 8 == 0;
  if (!vec) {
    const dim3 grid((unsigned)num_tokens, (unsigned)num_heads);
    if (dtype == kBF16)
      hipLaunchKernelGGL((paged_attn_plain_kernel<kBF16>), grid, dim3(64), 0, st, a);
    else
      hipLaunchKernelGGL((paged_attn_plain_kernel<kF16>), grid, dim3(64), 0, st, a);
    return launch_status();
  }
  // a workspace that is missing or too small means no cutting, not an error
  char* ws = workspace && aligned16(workspace) && workspace_bytes >= p.few.bytes() + p.tile.bytes()
                 ? reinterpret_cast<char*>(workspace)
                 : nullptr;
  int rc = run_class(a, p.tile, ws, dtype, st, [&](const PagedAttnArgs& x, int64_t groups) {
    return launch_attn_tiles(x, dtype, p.tile.rows, groups, st);
  });
  if (rc != SARATHI_OK) return rc;
  return run_class(a, p.few, ws ? ws + p.tile.bytes() : nullptr, dtype, st,
                   [&](const PagedAttnArgs& x, int64_t groups) {
                     return dtype == kBF16 ? launch_few_heads<kBF16>(x, p.few.rows / 16, groups, st)
                                           : launch_few_heads<kF16>(x, p.few.rows / 16, groups, st);
                   });
}
