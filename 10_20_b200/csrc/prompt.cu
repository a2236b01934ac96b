// Latent attention, expanded form: see v1x_prompt_attention in v1x.h.
//
// One warp per (query, head), one key per step: the query, the running maximum
// and sum of the softmax (in powers of two) and the output row in registers.
#include "attention.cuh"

namespace v1x {
namespace {

using namespace attn;

struct PromptArgs {
  const void *q, *k, *k_rope, *v;
  int64_t qs0, qs1, ks0, ks1, krs0, vs0, vs1;
  const int32_t *offsets, *kv_offsets;
  int64_t requests, tokens, keys, heads;
  int dr;
  float scale_log2;
  void* out;
  float* lse;
};

template <typename T>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const __grid_constant__ PromptArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t i = blockIdx.x, h = static_cast<int64_t>(blockIdx.y) * 4 + (threadIdx.x >> 5);
  if (h >= a.heads) return;
  // the last request whose first query is at or before i
  int64_t lo = 0, hi = a.requests;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (a.offsets[mid] <= i) lo = mid;
    else hi = mid;
  }
  const int64_t q0 = max(a.offsets[lo], 0), q1 = min(static_cast<int64_t>(a.offsets[lo + 1]), a.tokens);
  if (i < q0 || i >= q1) return;
  const int64_t k0 = max(a.kv_offsets[lo], 0), k1 = min(static_cast<int64_t>(a.kv_offsets[lo + 1]), a.keys);
  const int64_t end = min(k1, k0 + (i - q0) + 1 + (k1 - k0) - (q1 - q0));
  const T* q = static_cast<const T*>(a.q) + i * a.qs0 + h * a.qs1;
  float2 qv[3];
#pragma unroll
  for (int c = 0; c < 3; ++c)
    qv[c] = c < 2 || a.dr ? to_float2<T>(*reinterpret_cast<const uint32_t*>(q + 64 * c + 2 * lane)) : make_float2(0, 0);
  float2 acc[2] = {make_float2(0, 0), make_float2(0, 0)};
  float m = -CUDART_INF_F, l = 0.0f;
  for (int64_t j = k0; j < end; ++j) {
    const T* k = static_cast<const T*>(a.k) + j * a.ks0 + h * a.ks1 + 2 * lane;
    const T* v = static_cast<const T*>(a.v) + j * a.vs0 + h * a.vs1 + 2 * lane;
    float dot = 0.0f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float2 x = to_float2<T>(*reinterpret_cast<const uint32_t*>(k + 64 * c));
      dot = fmaf(qv[c].x, x.x, fmaf(qv[c].y, x.y, dot));
    }
    if (a.dr) {
      const float2 x = to_float2<T>(*reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.k_rope) + j * a.krs0 + 2 * lane));
      dot = fmaf(qv[2].x, x.x, fmaf(qv[2].y, x.y, dot));
    }
    const float x = warp_sum(dot) * a.scale_log2, top = fmaxf(m, x);
    const float shrink = exp2f(m - top), p = exp2f(x - top);
    l = l * shrink + p;
    m = top;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float2 y = to_float2<T>(*reinterpret_cast<const uint32_t*>(v + 64 * c));
      acc[c].x = fmaf(p, y.x, acc[c].x * shrink);
      acc[c].y = fmaf(p, y.y, acc[c].y * shrink);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  T* out = static_cast<T*>(a.out) + (i * a.heads + h) * 128 + 2 * lane;
#pragma unroll
  for (int c = 0; c < 2; ++c) *reinterpret_cast<uint32_t*>(out + 64 * c) = pack2<T>(acc[c].x * inv, acc[c].y * inv);
  if (lane == 0) a.lse[i * a.heads + h] = l > 0.0f ? (m + log2f(l)) * kLn2 : -CUDART_INF_F;
}

}  // namespace
}  // namespace v1x

extern "C" int v1x_prompt_attention(const void* q, int64_t qs0, int64_t qs1, const void* k, int64_t ks0, int64_t ks1,
                                    const void* k_rope, int64_t krs0, const void* v, int64_t vs0, int64_t vs1,
                                    const int32_t* offsets, const int32_t* kv_offsets, int64_t requests,
                                    int64_t tokens, int64_t keys, int64_t heads, int64_t dr, float scale, int dtype,
                                    void* out, float* lse, int32_t* status, void* stream) {
  using namespace v1x;
  using namespace v1x::attn;
  clear_error();
  V1X_CHECK_ARG(dtype == 1 || dtype == 2, "prompt_attention: dtype must be 1 (bf16) or 2 (f16)");
  V1X_CHECK_ARG(tokens >= 0 && tokens < (int64_t(1) << 31) && keys >= 0 && keys < (int64_t(1) << 31) && requests >= 0 &&
                    heads >= 1 && heads <= 1024,
                "prompt_attention: bad geometry");
  V1X_CHECK_ARG((dr == 0 && !k_rope) || (dr == 64 && (k_rope || keys == 0)), "prompt_attention: dr must be 0 without k_rope, 64 with it");
  V1X_CHECK_ARG(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_rope) |
                  reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                    (qs0 | qs1 | ks0 | ks1 | krs0 | vs0 | vs1) % 8 == 0,
                "prompt_attention: q, k, k_rope, v and out rows must be 16-byte aligned");
  if (tokens == 0 || requests == 0) return V1X_OK;
  V1X_CHECK_ARG(q && out && lse && offsets && kv_offsets && ((k && v) || keys == 0), "prompt_attention: NULL argument");
  PromptArgs a{q,   k,   k_rope, v,   qs0, qs1, ks0, ks1, krs0, vs0, vs1, offsets, kv_offsets, requests, tokens,
               keys, heads, static_cast<int>(dr), scale * kLog2e, out, lse};
  const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>((heads + 3) / 4));
  if (dtype == 1)
    launch_kernel_prio(LaunchPriority::kDefault, prompt_rows_kernel<__nv_bfloat16>, grid, dim3(128), 0, as_stream(stream), a);
  else
    launch_kernel_prio(LaunchPriority::kDefault, prompt_rows_kernel<__half>, grid, dim3(128), 0, as_stream(stream), a);
  return launch_status("v1x_prompt_attention");
}
