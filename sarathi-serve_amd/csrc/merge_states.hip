// Joins attention states computed over disjoint parts of a context, e.g. a shared prefix and each
// request's own suffix:
//   z = log sum_s exp(lse_s),   out = sum_s exp(lse_s - z) v_s.
// Streaming: every state's output is read once and the joined one written once, so HBM bandwidth
// bounds it.  A lane takes one 16-byte vector of a (token, head) row, issues the loads of all
// states together and folds them with weights relative to the largest lse; sums in 32 bits, one
// rounding.  A state whose lse is -inf has no output: its values are not used, whatever they are.
// Without any state that has one, out = 0 and z = -inf.
//
// Measured: two states of 16 tokens, 32 heads of 128, 3 us; four of 2304 tokens, 64 heads of 128 (192 MB),
// bfloat16, 28 us back to back, 34 us with inputs not seen before (5.6 TB/s).
#include "launch.h"
#include "paged_attn.h"

namespace sarathi_hip {

struct MergeArgs {
  const void* v;
  const float* lse;
  void* out;
  float* out_lse;                    // or null
  int64_t v_state, v_token;          // elements
  int64_t lse_state, lse_token;
  int64_t out_token, out_lse_token;
  int32_t states, heads, head_size;
  uint32_t blocks_per_token;
};

// N states known at compile time (their loads go out together), 0: a loop over any number.
template <int DT, int N>
__global__ __launch_bounds__(256) void merge_states_kernel(MergeArgs a) {
  constexpr int E = VecElems<DT>::value;
  const int64_t tok = blockIdx.x / a.blocks_per_token;
  const uint32_t vec = (blockIdx.x - (uint32_t)tok * a.blocks_per_token) * 256u + threadIdx.x;
  const uint32_t per_head = (uint32_t)a.head_size / E;
  const uint32_t head = vec / per_head;
  if (head >= (uint32_t)a.heads) return;
  const float* lse = a.lse + tok * a.lse_token + head;
  // rows of a token: the same for the workgroup, so scalar buffer resources
  const char* v = reinterpret_cast<const char*>(a.v) + tok * a.v_token * ElemBytes<DT>::value;
  const int64_t step = a.v_state * ElemBytes<DT>::value;
  const uint32_t row_bytes = (uint32_t)a.heads * (uint32_t)a.head_size * ElemBytes<DT>::value;
  float top = -INFINITY, l = 0.f;
  Vec<DT> acc;
#pragma unroll
  for (int i = 0; i < E; ++i) acc.f[i] = 0.f;
  if constexpr (N > 0) {
    u32x4 raw[N];
    float z[N];
#pragma unroll
    for (int s = 0; s < N; ++s) z[s] = lse[s * a.lse_state];
#pragma unroll
    for (int s = 0; s < N; ++s) raw[s] = buf_load16<kStreamLoad>(make_rsrc(v + s * step, row_bytes), vec * 16u);
    __builtin_amdgcn_sched_barrier(0);  // every load is issued before anything waits
#pragma unroll
    for (int s = 0; s < N; ++s) top = fmaxf(top, z[s]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      const float w = __builtin_amdgcn_exp2f((z[s] - ref) * kLog2e);
      l += w;
      Vec<DT> x;
      x.unpack(raw[s]);
#pragma unroll
      for (int i = 0; i < E; ++i) acc.f[i] = fmaf(z[s] == -INFINITY ? 0.f : x.f[i], w, acc.f[i]);
    }
  } else {
    for (int s = 0; s < a.states; ++s) top = fmaxf(top, lse[s * a.lse_state]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
    for (int s = 0; s < a.states; ++s) {
      const float z = lse[s * a.lse_state];
      const float w = __builtin_amdgcn_exp2f((z - ref) * kLog2e);
      l += w;
      Vec<DT> x;
      x.unpack(buf_load16<kStreamLoad>(make_rsrc(v + s * step, row_bytes), vec * 16u));
#pragma unroll
      for (int i = 0; i < E; ++i) acc.f[i] = fmaf(z == -INFINITY ? 0.f : x.f[i], w, acc.f[i]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) acc.f[i] *= inv;
  buf_store16<kStreamStore>(
      make_rsrc(reinterpret_cast<char*>(a.out) + tok * a.out_token * ElemBytes<DT>::value, row_bytes),
      vec * 16u, acc.pack());
  if (a.out_lse && vec == head * per_head)
    a.out_lse[tok * a.out_lse_token + head] = l == 0.f ? -INFINITY : top + logf(l);
}

// Any alignment and head size: one thread per element.
template <int DT>
__global__ __launch_bounds__(256) void merge_states_plain_kernel(MergeArgs a) {
  const int64_t tok = blockIdx.x / a.blocks_per_token;
  const uint32_t at = (blockIdx.x - (uint32_t)tok * a.blocks_per_token) * 256u + threadIdx.x;
  const uint32_t head = at / (uint32_t)a.head_size;
  if (head >= (uint32_t)a.heads) return;
  const float* lse = a.lse + tok * a.lse_token + head;
  float top = -INFINITY, l = 0.f, acc = 0.f;
  for (int s = 0; s < a.states; ++s) top = fmaxf(top, lse[s * a.lse_state]);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int s = 0; s < a.states; ++s) {
    const float z = lse[s * a.lse_state];
    const float w = __builtin_amdgcn_exp2f((z - ref) * kLog2e);
    l += w;
    if (z != -INFINITY) acc = fmaf(load_elem<DT>(a.v, s * a.v_state + tok * a.v_token + at), w, acc);
  }
  store_elem<DT>(a.out, tok * a.out_token + at, l == 0.f ? 0.f : acc / l);
  if (a.out_lse && at == head * (uint32_t)a.head_size)
    a.out_lse[tok * a.out_lse_token + head] = l == 0.f ? -INFINITY : top + logf(l);
}

template <int DT> static int launch_merge(MergeArgs a, int64_t tokens, bool vec, hipStream_t st) {
  const int per = vec ? VecElems<DT>::value : 1;
  const int64_t width = (int64_t)a.heads * a.head_size / per;
  a.blocks_per_token = (uint32_t)((width + 255) / 256);
  const int64_t groups = tokens * a.blocks_per_token;
  if (groups > 0x7fffffffLL) return SARATHI_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)groups), block(256);
  if (!vec) hipLaunchKernelGGL((merge_states_plain_kernel<DT>), grid, block, 0, st, a);
  else if (a.states == 2) hipLaunchKernelGGL((merge_states_kernel<DT, 2>), grid, block, 0, st, a);
  else if (a.states == 3) hipLaunchKernelGGL((merge_states_kernel<DT, 3>), grid, block, 0, st, a);
  else if (a.states == 4) hipLaunchKernelGGL((merge_states_kernel<DT, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((merge_states_kernel<DT, 0>), grid, block, 0, st, a);
  return launch_status();
}

}  // namespace sarathi_hip

using namespace sarathi_hip;

extern "C" int sarathi_merge_attention_states(const void* v, const float* lse, void* out,
                                              float* out_lse, int64_t num_states,
                                              int64_t num_tokens, int num_heads, int head_size,
                                              int64_t v_state_stride, int64_t v_token_stride,
                                              int64_t lse_state_stride, int64_t lse_token_stride,
                                              int64_t out_token_stride,
                                              int64_t out_lse_token_stride, int dtype,
                                              void* stream) {
  if (num_states < 1 || num_tokens < 0 || num_heads <= 0 || head_size <= 0 || v_state_stride < 0 ||
      lse_state_stride < 0)
    return SARATHI_ERR_INVALID_ARG;
  const int64_t row = (int64_t)num_heads * head_size;
  if (num_tokens > 1 && (v_token_stride < row || out_token_stride < row || lse_token_stride < num_heads ||
                         (out_lse && out_lse_token_stride < num_heads)))
    return SARATHI_ERR_INVALID_ARG;
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16) return SARATHI_ERR_UNSUPPORTED;
  if (num_states > 0x7fffffffLL || row > 0x1fffffffLL) return SARATHI_ERR_UNSUPPORTED;
  if (num_tokens == 0) return SARATHI_OK;
  if (!v || !lse || !out) return SARATHI_ERR_INVALID_ARG;
  MergeArgs a{v, lse, out, out_lse, v_state_stride, v_token_stride, lse_state_stride,
              lse_token_stride, out_token_stride, out_lse_token_stride, (int32_t)num_states,
              num_heads, head_size, 0};
  const int e = dtype == kF32 ? 4 : 8;
  const bool vec = head_size % e == 0 && v_state_stride % e == 0 && v_token_stride % e == 0 &&
                   out_token_stride % e == 0 && aligned16(v) && aligned16(out);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32) return launch_merge<kF32>(a, num_tokens, vec, st);
  if (dtype == kF16) return launch_merge<kF16>(a, num_tokens, vec, st);
  return launch_merge<kBF16>(a, num_tokens, vec, st);
}
