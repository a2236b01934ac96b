// The paged 8-bit K/V cache: v1x_kv8_store and v1x_kv8_attend of v1x.h.
#include <cuda_fp8.h>

#include "attention.cuh"

namespace v1x {
namespace {

using namespace attn;

// ---- store -------------------------------------------------------------------
// One CTA per (touched page, head, K or V): the page's new tokens (four threads
// a token, 32 values a thread, in registers), the largest magnitude over the CTA,
// the scale, then the codes; the earlier tokens' codes are read only where the
// scale rises.  Pure traffic: bytes of the new tokens in, half of them out.
//
// The pages a request touches are found without a pass over the requests:
// request r gets the units from base(r) = offsets[r] / 64 + 2 r on, at least as
// many as the pages that its tokens can touch, and unit u looks up its request by
// a search over offsets, 32 candidates a step.
struct StoreArgs {
  uint8_t* cache[2];
  float* scale[2];
  const void* x[2];
  int64_t s0[2], s1[2];
  int64_t pages, heads, tokens;
  const int32_t* table;
  int64_t table_stride, table_pages;
  const int32_t *prefix, *offsets;
  int64_t requests;
};

__device__ __forceinline__ int64_t clamped(const int32_t* offsets, int64_t i, int64_t tokens) {
  return min(static_cast<int64_t>(max(offsets[i], 0)), tokens);
}

// smallest 2^e, -40 <= e <= 40, with 448 * 2^e >= most (448 = 0.875 * 2^9)
__device__ __forceinline__ float scale_for(float most) {
  if (!(most > 0.0f)) return exp2f(-40.0f);
  if (most > 4.0e14f) return exp2f(40.0f);   // 448 * 2^39 = 2.5e14 < 4.0e14 < 448 * 2^40
  int x;
  const float m = frexpf(most, &x);
  return ldexpf(1.0f, min(max(m <= 0.875f ? x - 9 : x - 8, -40), 40));
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

__device__ __forceinline__ float2 values2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
  return __half22float2(__half2(h));
}

template <typename T>
__global__ void __launch_bounds__(256) kv8_store_kernel(const __grid_constant__ StoreArgs a) {
  __shared__ int64_t found;
  __shared__ float part[8];
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t u = blockIdx.x, h = blockIdx.y, z = blockIdx.z;
  if (tid < 32) {
    // the last request r with base(r) <= u; base is strictly increasing
    int64_t lo = 0, n = a.requests;
    while (n > 1) {
      const int64_t step = (n + 31) / 32, c = lo + lane * step;
      const bool at = lane * step < n && clamped(a.offsets, c, a.tokens) / 64 + 2 * c <= u;
      const int64_t k = max(__popc(__ballot_sync(0xffffffffu, at)) - 1, 0);
      lo += k * step;
      n = min(step, n - k * step);
    }
    if (lane == 0) found = lo;
  }
  __syncthreads();
  const int64_t r = found;
  const int64_t t0 = clamped(a.offsets, r, a.tokens), t1 = clamped(a.offsets, r + 1, a.tokens);
  const int64_t first = max(a.prefix[r], 0), end = first + (t1 - t0);
  const int64_t n = u - (t0 / 64 + 2 * r);   // which of the request's pages (below 0: before the first request)
  const int64_t i = first / 64 + n;          // the page's place in the table
  if (t1 <= t0 || n < 0 || i * 64 >= end || i >= a.table_pages) return;
  const int64_t page = a.table[r * a.table_stride + i];
  if (page < 0 || page >= a.pages) return;

  const int64_t pos = i * 64 + (tid >> 2);
  const bool fresh = pos >= first && pos < end;
  const int d0 = (tid & 3) * 8;   // 16-byte chunks (tid & 3), + 4, + 8, + 12 of the row
  uint4 raw[4];
  float most = 0.0f;
  if (fresh) {
    const T* x = static_cast<const T*>(a.x[z]) + (t0 + pos - first) * a.s0[z] + h * a.s1[z];
#pragma unroll
    for (int c = 0; c < 4; ++c) raw[c] = *reinterpret_cast<const uint4*>(x + d0 + 32 * c);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = to_float2<T>(w[e]);
        most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));   // a NaN counts for nothing
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (lane == 0) part[tid >> 5] = most;
  __syncthreads();
  most = part[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) most = fmaxf(most, part[w]);
  float* const sp = a.scale[z] + page * a.heads + h;
  float now = scale_for(most);
  const bool begun = first > i * 64;
  const float old = begun ? *sp : now;
  now = begun ? fmaxf(now, old) : now;
  __syncthreads();   // everyone has the former scale
  if (tid == 0) *sp = now;

  uint8_t* const row = a.cache[z] + ((page * a.heads + h) * 64 + (tid >> 2)) * 128;
  if (fresh) {
    const float inv = 1.0f / now;   // a power of two
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float2 f0 = to_float2<T>(raw[c].x), f1 = to_float2<T>(raw[c].y);
      const float2 f2 = to_float2<T>(raw[c].z), f3 = to_float2<T>(raw[c].w);
      *reinterpret_cast<uint2*>(row + d0 + 32 * c) =
          make_uint2(codes4(f0.x * inv, f0.y * inv, f1.x * inv, f1.y * inv),
                     codes4(f2.x * inv, f2.y * inv, f3.x * inv, f3.y * inv));
    }
  } else if (pos < first && now != old) {
    const float ratio = old / now;
    uint4* const p = reinterpret_cast<uint4*>(row + (tid & 3) * 32);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint4 v = p[c];
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 lo = values2(w[e]), hi = values2(w[e] >> 16);
        w[e] = codes4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
      }
      p[c] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ---- attend ------------------------------------------------------------------
struct AttendArgs {
  const void* q;
  int64_t qs0, qs1;
  const uint8_t *k, *v;
  const float *ks, *vs;
  int64_t pages, kv_heads;
  const int32_t* table;
  int64_t table_stride, table_pages;
  const int32_t* lens;
  int64_t rows, heads;
  float scale_log2;
  void* out;
  float* lse;
};

// One warp per (row, query head), one token per step.
template <typename T>
__global__ void __launch_bounds__(128) kv8_rows_kernel(const __grid_constant__ AttendArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t r = blockIdx.x, h = static_cast<int64_t>(blockIdx.y) * 4 + (threadIdx.x >> 5);
  if (h >= a.heads) return;
  const int64_t g = h / (a.heads / a.kv_heads);
  const int64_t n = min(static_cast<int64_t>(max(a.lens[r], 0)), a.table_pages * 64);
  const uint2 qr = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.q) + r * a.qs0 + h * a.qs1 + 4 * lane);
  const float2 q0 = to_float2<T>(qr.x), q1 = to_float2<T>(qr.y);
  float4 acc = make_float4(0, 0, 0, 0);
  float m = -CUDART_INF_F, l = 0.0f;
  for (int64_t j = 0; j < n; ++j) {
    const int64_t page = a.table[r * a.table_stride + (j >> 6)];
    if (page < 0 || page >= a.pages) continue;
    const int64_t block = page * a.kv_heads + g, at = (block * 64 + (j & 63)) * 128 + 4 * lane;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(a.k + at), vw = *reinterpret_cast<const uint32_t*>(a.v + at);
    const float2 k0 = values2(kw), k1 = values2(kw >> 16), v0 = values2(vw), v1 = values2(vw >> 16);
    const float dot = fmaf(q0.x, k0.x, fmaf(q0.y, k0.y, fmaf(q1.x, k1.x, q1.y * k1.y)));
    const float x = warp_sum(dot) * a.ks[block] * a.scale_log2, top = fmaxf(m, x);
    const float shrink = exp2f(m - top), p = exp2f(x - top), pv = p * a.vs[block];
    l = l * shrink + p;
    m = top;
    acc = make_float4(fmaf(pv, v0.x, acc.x * shrink), fmaf(pv, v0.y, acc.y * shrink), fmaf(pv, v1.x, acc.z * shrink),
                      fmaf(pv, v1.y, acc.w * shrink));
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (r * a.heads + h) * 128 + 4 * lane) =
      make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
  if (lane == 0) a.lse[r * a.heads + h] = l > 0.0f ? (m + log2f(l)) * kLn2 : -CUDART_INF_F;
}

}  // namespace
}  // namespace v1x

extern "C" int v1x_kv8_store(uint8_t* k_cache, float* k_scale, uint8_t* v_cache, float* v_scale, int64_t pages,
                             int64_t heads, const void* k, int64_t ks0, int64_t ks1, const void* v, int64_t vs0,
                             int64_t vs1, int dtype, int64_t tokens, const int32_t* table, int64_t table_stride,
                             int64_t table_pages, const int32_t* prefix, const int32_t* offsets, int64_t requests,
                             void* stream) {
  using namespace v1x;
  clear_error();
  V1X_CHECK_ARG(dtype == 1 || dtype == 2, "kv8_store: dtype must be 1 (bf16) or 2 (f16)");
  V1X_CHECK_ARG(pages >= 0 && heads >= 1 && heads <= 65535 && tokens >= 0 && tokens < (int64_t(1) << 31) &&
                    requests >= 0 && requests < (int64_t(1) << 29) && table_pages >= 0,
                "kv8_store: bad geometry");
  V1X_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                  reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                    (ks0 | ks1 | vs0 | vs1) % 8 == 0,
                "kv8_store: the caches and the rows of k and v must be 16-byte aligned");
  if (tokens == 0 || requests == 0 || pages == 0 || table_pages == 0) return V1X_OK;
  V1X_CHECK_ARG(k_cache && k_scale && v_cache && v_scale && k && v && table && prefix && offsets, "kv8_store: NULL argument");
  StoreArgs a{{k_cache, v_cache}, {k_scale, v_scale}, {k, v}, {ks0, vs0}, {ks1, vs1}, pages, heads, tokens,
              table, table_stride, table_pages, prefix, offsets, requests};
  const dim3 grid(static_cast<unsigned>(tokens / 64 + 2 * requests), static_cast<unsigned>(heads), 2);
  if (dtype == 1)
    launch_kernel_prio(LaunchPriority::kDefault, kv8_store_kernel<__nv_bfloat16>, grid, dim3(256), 0, as_stream(stream), a);
  else
    launch_kernel_prio(LaunchPriority::kDefault, kv8_store_kernel<__half>, grid, dim3(256), 0, as_stream(stream), a);
  return launch_status("v1x_kv8_store");
}

extern "C" int64_t v1x_kv8_attend_workspace(int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_pages) {
  return 0;
}

extern "C" int v1x_kv8_attend(const void* q, int64_t qs0, int64_t qs1, const uint8_t* k_cache, const float* k_scale,
                              const uint8_t* v_cache, const float* v_scale, int64_t pages, int64_t kv_heads,
                              const int32_t* table, int64_t table_stride, int64_t table_pages, const int32_t* lens,
                              int64_t rows, int64_t heads, float scale, int dtype, void* out, float* lse,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace v1x;
  using namespace v1x::attn;
  clear_error();
  V1X_CHECK_ARG(dtype == 1 || dtype == 2, "kv8_attend: dtype must be 1 (bf16) or 2 (f16)");
  V1X_CHECK_ARG(rows >= 0 && rows < (int64_t(1) << 31) && pages >= 0 && table_pages >= 0 && kv_heads >= 1 && heads >= 1 &&
                    heads <= 1024 && heads % kv_heads == 0,
                "kv8_attend: bad geometry (heads must be a multiple of kv_heads, at most 1024)");
  V1X_CHECK_ARG(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
                  reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                    (qs0 | qs1) % 8 == 0,
                "kv8_attend: the caches and the rows of q and out must be 16-byte aligned");
  if (rows == 0) return V1X_OK;
  V1X_CHECK_ARG(q && out && lse && lens && (table || table_pages == 0) &&
                    ((k_cache && k_scale && v_cache && v_scale) || pages == 0),
                "kv8_attend: NULL argument");
  AttendArgs a{q, qs0, qs1, k_cache, v_cache, k_scale, v_scale, pages, kv_heads, table, table_stride, table_pages,
               lens, rows, heads, scale * kLog2e, out, lse};
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>((heads + 3) / 4));
  if (dtype == 1)
    launch_kernel_prio(LaunchPriority::kDefault, kv8_rows_kernel<__nv_bfloat16>, grid, dim3(128), 0, as_stream(stream), a);
  else
    launch_kernel_prio(LaunchPriority::kDefault, kv8_rows_kernel<__half>, grid, dim3(128), 0, as_stream(stream), a);
  return launch_status("v1x_kv8_attend");
}
