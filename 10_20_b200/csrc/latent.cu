// Latent attention, absorbed form: see v1x_latent_attention in v1x.h.
//
// One warp per (row, head): the query in registers, one token per step, the
// running maximum and sum of the softmax (in powers of two) and the output row
// in registers; one pass over the tokens.
#include "attention.cuh"

namespace v1x {
namespace {

using namespace attn;

struct LatentArgs {
  const void* q;
  int64_t qs0, qs1;
  const void* pool;
  int64_t slots, pool_stride;
  const int32_t* req;
  int64_t req_len;
  const int32_t* index;
  int64_t index_stride, count;
  const int32_t* lens;
  int64_t rows, heads;
  int dim, latent;
  float scale_log2;
  void* out;
  float* lse;
};

// The pool slot of token j of row r, or -1 if there is none.
__device__ __forceinline__ int64_t slot_of(const LatentArgs& a, const int32_t* index, int64_t j, int64_t n) {
  if (j >= n) return -1;
  int64_t s;
  if (a.lens) {
    s = static_cast<int64_t>(index[j >> 6]) * 64 + (j & 63);
  } else {
    s = index[j];
    if (a.req) s = s >= 0 && s < a.req_len ? a.req[s] : -1;
  }
  return s >= 0 && s < a.slots ? s : -1;
}

constexpr int kMaxPairs = 9;  // 576 = 32 lanes * 9 pairs

template <typename T>
__global__ void __launch_bounds__(128) latent_rows_kernel(const __grid_constant__ LatentArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t h = static_cast<int64_t>(blockIdx.y) * 4 + (threadIdx.x >> 5), r = blockIdx.x;
  if (h >= a.heads) return;
  const T* q = static_cast<const T*>(a.q) + r * a.qs0 + h * a.qs1;
  const int32_t* index = a.index + r * a.index_stride;
  const int64_t n = a.lens ? min(static_cast<int64_t>(max(a.lens[r], 0)), a.count) : a.count;
  float2 qv[kMaxPairs], acc[kMaxPairs];
#pragma unroll
  for (int i = 0; i < kMaxPairs; ++i) {
    const int d = 2 * (lane + 32 * i);
    qv[i] = d < a.dim ? to_float2<T>(*reinterpret_cast<const uint32_t*>(q + d)) : make_float2(0.0f, 0.0f);
    acc[i] = make_float2(0.0f, 0.0f);
  }
  float m = -CUDART_INF_F, l = 0.0f;
  for (int64_t j = 0; j < n; ++j) {
    const int64_t s = slot_of(a, index, j, n);
    if (s < 0) continue;
    const T* row = static_cast<const T*>(a.pool) + s * a.pool_stride;
    float2 kv[kMaxPairs];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
      const int d = 2 * (lane + 32 * i);
      kv[i] = d < a.dim ? to_float2<T>(*reinterpret_cast<const uint32_t*>(row + d)) : make_float2(0.0f, 0.0f);
      dot = fmaf(qv[i].x, kv[i].x, fmaf(qv[i].y, kv[i].y, dot));
    }
    const float x = warp_sum(dot) * a.scale_log2, top = fmaxf(m, x);
    const float shrink = exp2f(m - top), p = exp2f(x - top);
    l = l * shrink + p;
    m = top;
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
      acc[i].x = fmaf(p, kv[i].x, acc[i].x * shrink);
      acc[i].y = fmaf(p, kv[i].y, acc[i].y * shrink);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  T* out = static_cast<T*>(a.out) + (r * a.heads + h) * a.latent;
#pragma unroll
  for (int i = 0; i < kMaxPairs; ++i) {
    const int d = 2 * (lane + 32 * i);
    if (d < a.latent) *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(acc[i].x * inv, acc[i].y * inv);
  }
  if (lane == 0) a.lse[r * a.heads + h] = l > 0.0f ? (m + log2f(l)) * kLn2 : -CUDART_INF_F;
}

}  // namespace
}  // namespace v1x

extern "C" int64_t v1x_latent_attention_workspace(int64_t rows, int64_t heads, int64_t count, int64_t latent) {
  return 0;
}

extern "C" int v1x_latent_attention(const void* q, int64_t qs0, int64_t qs1, const void* pool, int64_t slots,
                                    int64_t pool_stride, const int32_t* req, int64_t req_len, const int32_t* index,
                                    int64_t index_stride, int64_t count, const int32_t* lens, int64_t rows,
                                    int64_t heads, int64_t dim, int64_t latent, float scale, int dtype, void* out,
                                    float* lse, void* workspace, int64_t workspace_bytes, int32_t* status,
                                    void* stream) {
  using namespace v1x;
  using namespace v1x::attn;
  clear_error();
  V1X_CHECK_ARG(dtype == 1 || dtype == 2, "latent_attention: dtype must be 1 (bf16) or 2 (f16)");
  V1X_CHECK_ARG(rows >= 0 && rows < (int64_t(1) << 31) && heads >= 1 && heads <= 1024 && count >= 0 && slots >= 0,
                "latent_attention: bad geometry");
  V1X_CHECK_ARG(latent >= 128 && latent <= 512 && latent % 128 == 0 && (dim == latent || dim == latent + 64),
                "latent_attention: latent must be 128, 256, 384 or 512 and dim - latent 0 or 64");
  V1X_CHECK_ARG(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pool) |
                  reinterpret_cast<uintptr_t>(out)) & 15) == 0 && qs0 % 8 == 0 && qs1 % 8 == 0 && pool_stride % 8 == 0,
                "latent_attention: q, pool and out rows must be 16-byte aligned");
  V1X_CHECK_ARG(!lens || (count % 64 == 0 && !req), "latent_attention: a page table takes whole pages and no slot map");
  if (rows == 0) return V1X_OK;
  V1X_CHECK_ARG(q && out && lse && (index || count == 0) && (pool || slots == 0), "latent_attention: NULL argument");
  LatentArgs a{q,    qs0,  qs1,  pool,  slots, pool_stride, req, req_len, index, index_stride, count,
               lens, rows, heads, static_cast<int>(dim), static_cast<int>(latent), scale * kLog2e, out, lse};
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>((heads + 3) / 4));
  if (dtype == 1)
    launch_kernel_prio(LaunchPriority::kDefault, latent_rows_kernel<__nv_bfloat16>, grid, dim3(128), 0, as_stream(stream), a);
  else
    launch_kernel_prio(LaunchPriority::kDefault, latent_rows_kernel<__half>, grid, dim3(128), 0, as_stream(stream), a);
  return launch_status("v1x_latent_attention");
}
