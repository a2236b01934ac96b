// The paged 8-bit K/V cache: v1x_kv8_store and v1x_kv8_attend of v1x.h.
#include <cuda_fp8.h>

#include <type_traits>

#include "attention.cuh"
#include "ranges.cuh"
#include "ring.cuh"
#include "sm100.cuh"

namespace v1x {
namespace {

using namespace attn;
using namespace sm100;

// ---- store -------------------------------------------------------------------
// One warp per (touched page, head, K or V): the page's new tokens (eight lanes a
// token, 16 values a lane, the whole page in registers), the largest magnitude by
// shuffles, the scale, then the codes; the earlier tokens' codes are read only
// where the scale rises.  Pure traffic, bytes of the new tokens in and half of them
// out, behind a chain of five dependent loads (request, its bounds, its page), which
// is what a decode step's single tokens cost: so no barriers, many warps (128 requests,
// 8 heads: 7.2 us; a CTA for each page and head 11.5).  Prompts of 16384 tokens: 23.6 us,
// 4.3 TB/s.
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

// The larger magnitudes of two pairs; of a NaN and a number the number.
template <typename T>
__device__ __forceinline__ uint32_t max_magnitudes(uint32_t a, uint32_t b) {
  using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const Pair m = __hmax2(__habs2(*reinterpret_cast<Pair*>(&a)), __habs2(*reinterpret_cast<Pair*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&m);
}

template <typename T>
__global__ void __launch_bounds__(128) kv8_store_kernel(const __grid_constant__ StoreArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t u = blockIdx.x, hz = static_cast<int64_t>(blockIdx.y) * 4 + (threadIdx.x >> 5);
  if (hz >= 2 * a.heads) return;
  const int64_t h = hz >> 1;
  const int z = static_cast<int>(hz & 1);
  // the last request r with base(r) <= u; base is strictly increasing
  int64_t r = 0;
  for (int64_t n = a.requests; n > 1;) {
    const int64_t step = (n + 31) / 32, c = r + lane * step;
    const bool at = lane * step < n && clamped(a.offsets, c, a.tokens) / 64 + 2 * c <= u;
    const int64_t k = max(__popc(__ballot_sync(0xffffffffu, at)) - 1, 0);
    r += k * step;
    n = min(step, n - k * step);
  }
  const int64_t t0 = clamped(a.offsets, r, a.tokens), t1 = clamped(a.offsets, r + 1, a.tokens);
  const int64_t first = max(a.prefix[r], 0), end = first + (t1 - t0);
  const int64_t nth = u - (t0 / 64 + 2 * r);   // which of the request's pages (below 0: before the first request)
  const int64_t i = first / 64 + nth;          // the page's place in the table
  if (t1 <= t0 || nth < 0 || i * 64 >= end || i >= a.table_pages) return;
  const int64_t page = a.table[r * a.table_stride + i];
  if (page < 0 || page >= a.pages) return;

  // the page's tokens [lo, hi) are new, those before lo earlier ones
  const int lo = static_cast<int>(max(first - i * 64, int64_t(0))), hi = static_cast<int>(min(end - i * 64, int64_t(64)));
  const int sub = lane >> 3, d0 = (lane & 7) * 16;   // of token 4 k + sub: values d0 .. d0 + 15
  const T* x = static_cast<const T*>(a.x[z]) + (t0 + i * 64 - first + sub) * a.s0[z] + h * a.s1[z] + d0;
  const int64_t four = 4 * a.s0[z];
  float* const sp = a.scale[z] + page * a.heads + h;
  const float former = *sp;
  uint4 raw[16][2];
  const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int t = 4 * k + sub;
    const bool fresh = t >= lo && t < hi;
    raw[k][0] = raw[k][1] = none;
    if (fresh) {
      raw[k][0] = *reinterpret_cast<const uint4*>(x);
      raw[k][1] = *reinterpret_cast<const uint4*>(x + 8);
    }
    x += four;
  }
  uint32_t tops[2] = {0, 0};     // pairs; a NaN counts for nothing
#pragma unroll
  for (int k = 0; k < 16; ++k)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      tops[c] = max_magnitudes<T>(tops[c], max_magnitudes<T>(raw[k][c].x, raw[k][c].y));
      tops[c] = max_magnitudes<T>(tops[c], max_magnitudes<T>(raw[k][c].z, raw[k][c].w));
    }
  const float2 top = to_float2<T>(max_magnitudes<T>(tops[0], tops[1]));
  float most = fmaxf(top.x, top.y);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  float now = scale_for(most);
  const float old = lo > 0 ? former : now;
  now = lo > 0 ? fmaxf(now, old) : now;
  if (lane == 0) *sp = now;

  uint8_t* const rows = a.cache[z] + (page * a.heads + h) * 64 * 128 + d0, * const own = rows + sub * 128;
  const float inv = 1.0f / now;   // a power of two
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int t = 4 * k + sub;
    if (t < lo || t >= hi) continue;
    uint32_t w[4];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float2 f0 = to_float2<T>(raw[k][c].x), f1 = to_float2<T>(raw[k][c].y);
      const float2 f2 = to_float2<T>(raw[k][c].z), f3 = to_float2<T>(raw[k][c].w);
      w[2 * c] = codes4(f0.x * inv, f0.y * inv, f1.x * inv, f1.y * inv);
      w[2 * c + 1] = codes4(f2.x * inv, f2.y * inv, f3.x * inv, f3.y * inv);
    }
    *reinterpret_cast<uint4*>(own + k * 512) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (now != old) {               // the same in all lanes
    const float ratio = old / now;
    for (int t = sub; t < lo; t += 4) {
      uint4* const p = reinterpret_cast<uint4*>(rows + t * 128);
      const uint4 v = *p;
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = values2(w[e]), g = values2(w[e] >> 16);
        w[e] = codes4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
      }
      *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ---- attend ------------------------------------------------------------------
// Bound by the cache's bytes: 16 KB a page and K/V head, about 2 flops a byte and
// query head.  Codes have to become 16-bit values on the way (e4m3 is exact in
// f16), so the products are warp-level f16 MMAs fed from registers, tokens and
// value columns as the 16-row operand, up to 8 query heads as the 8-column one:
//
//   S^T[16 tokens x 8 heads] = K . Q^T,   O^T[16 columns x 8 heads] += V^T . P^T
//
// A warp works alone: it brings a page's keys and values by TMA into a ring of
// three 8 KB buffers of its own (two in flight, 128 KB a CTA of eight warps), keeps
// the softmax of its heads and their output in registers, and takes its own equal
// range of the line of all pages (rows x K/V heads x pages); a row and head that
// lies in several ranges leaves unnormalised parts in the workspace, joined by
// kv8_join_kernel in the order of the ranges.
//   * element order inside a contraction is free, so a lane's bytes are contiguous:
//     of a key's 128 dims lane tig takes 32 tig .. 32 tig + 31, of the values' columns
//     lane g takes 16 g .. 16 g + 15; with the buffers' 128-byte swizzle every 16-byte
//     read is free of conflicts;
// 64 rows of 1-16 K tokens, 32 heads over 4: 103 us, 5.5 TB/s (the join about 8 of them);
// 64 heads over 4 157 us, where the two-tile kernel fills 255 registers and spills; one
// row of 4097 tokens 13 us.
//   * the query is held in f16 under a power of two per head that puts its largest
//     value in [1, 2); the weights, up to 2^15, are rounded to f16 once, sums stay in 32 bits; a
//     page's output is added under its value scale in 32 bits, so scales of any size
//     meet the f16 products unchanged.
struct AttendArgs {
  const void* q;
  int64_t qs0, qs1;
  const float *ks, *vs;
  int64_t pages, kv_heads;
  const int32_t* table;
  int64_t table_stride, table_pages;
  const int32_t* lens;
  int64_t rows, heads;
  int per_kv, groups, segments, ranges;   // query heads of a K/V head, groups of 8 kTiles of them, K/V heads x groups
  float scale_log2;
  void* out;
  float* lse;
  float* part;      // [ranges][2][8 kTiles][128], then [..][2] maxima and sums
  float* part_ml;
  int64_t* where;   // [ranges + 1][4]: the ranges' records; tiles are pages, place: row * segments + segment
  int32_t* status;
};

constexpr int kWarps = 8, kRing = 3, kMaxRanges = 148 * kWarps;
constexpr int kPageBytes8 = 64 * 128;
constexpr uint64_t kWaitNs = 2000000000ull;

struct AttendShared {
  uint64_t full[kWarps][kRing];
  int64_t prefix[kWarps * 32];
  int64_t scan[kWarps + 1];
  int abort, zero;
};

__device__ __forceinline__ int64_t row_pages(const AttendArgs& a, int64_t r) {
  const int64_t n = min(static_cast<int64_t>(max(a.lens[r], 0)), a.table_pages * 64);
  return (n + 63) / 64;
}

__device__ __forceinline__ uint32_t half2_of(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(two));
  return h;
}
__device__ __forceinline__ uint32_t half2_of_high(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(h) : "r"(two));
  return h;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// 8 kTiles query heads at a time
template <typename T, int kTiles>
__global__ void __launch_bounds__(kWarps * 32, 1)
    kv8_attend_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const __grid_constant__ AttendArgs a) {
  constexpr int kHeads = 8 * kTiles, kPasses = kTiles;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  AttendShared& sh = *reinterpret_cast<AttendShared*>(base + kWarps * kRing * kPageBytes8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
  if (tid == 0) {
    sh.abort = 0;
    sh.zero = 0;
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kRing; ++s) mbar_init(&sh.full[w][s], 1);
    fence_mbar_init();
    if (a.pages > 0) {
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
  }
  // ---- this warp's range of the line: pages of row 0's segments, row 1's, ... --------
  const int64_t chunk = (a.rows + kWarps * 32 - 1) / (kWarps * 32);
  const int64_t beg = min(tid * chunk, a.rows), end = min(beg + chunk, a.rows);
  int64_t own = 0, all;
  for (int64_t r = beg; r < end; ++r) own += row_pages(a, r) * a.segments;
  sh.prefix[tid] = block_exclusive_scan(own, sh.scan, &all);
  __syncthreads();
  // neighbouring ranges on different SMs
  const int64_t x = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
  const int64_t per = all >> 31 ? all / a.ranges : static_cast<uint32_t>(all) / static_cast<uint32_t>(a.ranges);
  const int64_t extra = all - per * a.ranges;
  const int64_t t0 = x * per + min(x, extra), pages_mine = x < a.ranges ? per + (x < extra ? 1 : 0) : 0;
  int64_t row = 0, page = 0, segment = 0;
  RangeBegin range = no_row(t0);               // an empty one stays so
  if (t0 < all && x < a.ranges) {
    int lo = 0;   // the last thread whose rows begin at or before t0 (those behind it with the same prefix are empty)
    for (int step = kWarps * 16; step > 0; step >>= 1)
      if (lo + step < kWarps * 32 && sh.prefix[lo + step] <= t0) lo += step;
    range = find_begin(t0, lo * chunk, a.rows, sh.prefix[lo], [&](int64_t r) { return row_pages(a, r) * a.segments; });
    row = range.place;
    const int64_t p = row_pages(a, row);
    segment = (t0 - range.first) / p;
    page = t0 - range.first - segment * p;
    range = RangeBegin{row * a.segments + segment, t0 - page, p, t0};
  }
  if (a.where && lane == 0 && x < a.ranges) {
    put_record(a.where, x, range);
    if (x == a.ranges - 1) a.where[4 * x + 7] = all;
  }

  // ---- the walk ---------------------------------------------------------------------
  const int n = static_cast<int>(pages_mine);
  struct Place {
    int row, segment, page, pages;
  };
  auto next = [&](Place& p) {
    if (++p.page < p.pages) return;
    p.page = 0;
    if (++p.segment < a.segments) return;
    p.segment = 0;
    do {
      ++p.row;
      p.pages = p.row < a.rows ? static_cast<int>(row_pages(a, p.row)) : 1;
    } while (p.pages == 0);
  };
  // a page of the cache and its scales; block < 0: none
  struct Block {
    int at;
    float ks, vs;
  };
  auto block_of = [&](const Place& p) {
    Block b{-1, 0.0f, 0.0f};
    const int id = a.table[p.row * a.table_stride + p.page];
    if (id >= 0 && id < a.pages) {             // pages * kv_heads < 2^25
      b.at = id * static_cast<int>(a.kv_heads) + p.segment / a.groups;
      b.ks = a.ks[b.at];
      b.vs = a.vs[b.at];
    }
    return b;
  };
  const uint32_t ring = smem_u32(base + warp * kRing * kPageBytes8);
  uint64_t* const full = sh.full[warp];
  // After a wait that gave up the warp ends its page, whose result is of no use, and its
  // walk; `state` keeps it from sending boxes.  (Leaving the page at once made 16 heads a
  // K/V head 168 us instead of 158: other spills.)
  RingState state;
  auto load = [&](const CUtensorMap* map, int slot, int at) {
    if (at < 0 || !state.start(slot)) return;
    if (lane == 0) {
      mbar_arrive_expect_tx(&full[slot], kPageBytes8);
      tma_load_2d(base + (warp * kRing + slot) * kPageBytes8, map, &full[slot], 0, at * 64);
    }
  };
  auto arrived = [&](int slot) {
    const bool done = __all_sync(0xffffffffu, mbar_wait(&full[slot], state.phase(slot), &sh.abort, kWaitNs));
    if (!done) {
      *reinterpret_cast<volatile int*>(&sh.abort) = 1;
      if (a.status) atomicExch(a.status, V1X_STATUS_TIMEOUT);
    }
    state.waited(slot, done);
  };

  Place now{static_cast<int>(row), static_cast<int>(segment), static_cast<int>(page), static_cast<int>(range.tiles)}, ahead = now;   // ahead: the page whose block was looked up last
  Block cur{-1, 0, 0}, nxt{-1, 0, 0};
  if (n > 0) {
    cur = block_of(ahead);
    load(&k_map, 0, cur.at);
    load(&v_map, 1, cur.at);
    if (n > 1) {
      next(ahead);
      nxt = block_of(ahead);
      load(&k_map, 2, nxt.at);
    }
  }
  uint32_t q[kTiles][8][2];
  float qscale[kTiles][2];                     // of the two heads of this lane's columns, scale and base 2 included
  float o[kTiles][8][4], m[kTiles][2], l[kTiles][2];
  bool fresh = true;
  int parts = 0;
  int slot = 0;                                // of the page's keys; its values follow
  for (int it = 0; it < n && state.ok; ++it) {
    const int kv = now.segment / a.groups, group = now.segment % a.groups;
    const int heads = min(kHeads, a.per_kv - group * kHeads);
    const int head0 = kv * a.per_kv + group * kHeads;
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        // lane (g, tig) holds head 8 t + g, dims 32 tig .. 32 tig + 31
        const int hh = 8 * t + g;
        uint4 raw[4];
        float most = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          raw[c] = make_uint4(0, 0, 0, 0);
          if (hh < heads)
            raw[c] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + now.row * a.qs0 + static_cast<int64_t>(head0 + hh) * a.qs1 +
                                                     32 * tig + 8 * c);
          const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = to_float2<T>(w[e]);
            most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // 2^e <= most < 2^(e+1), as two factors that stay in range
        const int e = most > 0.0f && most <= 3.0e38f ? min(max(ilogbf(most), -125), 126) : 0;
        const float down = ldexpf(1.0f, -e);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const uint4 v = raw[s >> 1];
          const float2 f0 = to_float2<T>(s & 1 ? v.z : v.x), f1 = to_float2<T>(s & 1 ? v.w : v.y);
          q[t][s][0] = pack2<__half>(f0.x * down, f0.y * down);
          q[t][s][1] = pack2<__half>(f1.x * down, f1.y * down);
        }
        const float up = ldexpf(1.0f, e);
        qscale[t][0] = __shfl_sync(0xffffffffu, up, 8 * tig) * a.scale_log2;        // head 2 tig: a lane with g = 2 tig
        qscale[t][1] = __shfl_sync(0xffffffffu, up, 8 * tig + 4) * a.scale_log2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m[t][i] = -CUDART_INF_F;
          l[t][i] = 0.0f;
        }
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][d][i] = 0.0f;
      }
    }
    // the block after the next one is looked up early, its loads are issued as buffers come free
    Block far{-1, 0, 0};
    if (it + 2 < n) {
      next(ahead);
      far = block_of(ahead);
    }
    const int left = min(a.lens[now.row] - now.page * 64, 64);   // page < pages: no overflow
    const int vslot = slot + 1 == kRing ? 0 : slot + 1;
    uint32_t p[kTiles][8];                     // weights as the second product's operand
    if (cur.at >= 0) {
      float s[kTiles][4][4];
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][j][i] = 0.0f;
      arrived(slot);
      const uint32_t k = ring + slot * kPageBytes8;
      // token tiles j innermost: their sums are independent, one's next step waits 20 cycles
      const uint32_t r0 = k + g * 128;         // tokens 16 j + g, + 8: the same row & 7
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t at = r0 + static_cast<uint32_t>(((2 * tig + c) ^ g) << 4);
        uint4 u[4], v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u[j] = lds128(at + j * 2048);
          v[j] = lds128(at + j * 2048 + 1024);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t uw = w == 0 ? u[j].x : w == 1 ? u[j].y : w == 2 ? u[j].z : u[j].w;
            const uint32_t vw = w == 0 ? v[j].x : w == 1 ? v[j].y : w == 2 ? v[j].z : v[j].w;
            const uint32_t a0 = half2_of(uw), a1 = half2_of(vw), a2 = half2_of_high(uw), a3 = half2_of_high(vw);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) mma16816(s[t][j], a0, a1, a2, a3, q[t][4 * c + w][0], q[t][4 * c + w][1]);
          }
      }
      __syncwarp();
      load(&v_map, slot, nxt.at);              // the keys' buffer is free: the next page's values
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float f = qscale[t][i] * cur.ks;
          float top = -CUDART_INF_F;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float& e = s[t][j][2 * y + i];
              e = 16 * j + 8 * y + g < left ? e * f : -CUDART_INF_F;
              top = fmaxf(top, e);
            }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          top = fmaxf(top - lift<__half>(0.0f), m[t][i]);   // m: the weights' reference
          const float ref = top == -CUDART_INF_F ? 0.0f : top;
          alpha[i] = exp2_fast(m[t][i] - ref);
          m[t][i] = top;
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float& e = s[t][j][2 * y + i];
              e = exp2_fast(e - ref);
              sum += e;
            }
          l[t][i] = fmaf(l[t][i], alpha[i], sum);
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
          for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][d][i] *= alpha[i & 1];
        }
        // 8 x 8 blocks [token][head] -> [head][token]
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;"
                         : "=r"(p[t][2 * j + y])
                         : "r"(pack2<__half>(s[t][j][2 * y], s[t][j][2 * y + 1])));
      }
      arrived(vslot);
      const uint32_t v = ring + vslot * kPageBytes8;
      // a lane's 16 columns in kPasses parts: two tiles' sums of all 16 would not fit the
      // registers beside the rest
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
        float acc[kTiles][8 / kPasses][4];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int d = 0; d < 8 / kPasses; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][d][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // tokens 16 j + 2 tig, + 1, + 8, + 9; columns 16 g .. 16 g + 15
          uint32_t x4[4][4 / kPasses];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int token = 16 * j + 2 * tig + (i & 1) + 8 * (i >> 1);
            const uint32_t at = v + token * 128 + ((g ^ ((2 * tig + (i & 1)) & 7)) << 4);
            // places behind the last token may hold NaN codes
            if constexpr (kPasses == 1) {
              uint4 u = lds128(at);
              if (token >= left) u = make_uint4(0, 0, 0, 0);
              x4[i][0] = u.x;
              x4[i][1] = u.y;
              x4[i][2] = u.z;
              x4[i][3] = u.w;
            } else {
              uint2 u = lds64(at + 8 * pass);
              if (token >= left) u = make_uint2(0, 0);
              x4[i][0] = u.x;
              x4[i][1] = u.y;
            }
          }
#pragma unroll
          for (int w = 0; w < 4 / kPasses; ++w)
#pragma unroll
            for (int y = 0; y < 2; ++y) {      // columns 4 w + 2 y, + 1 of the part: rows g and g + 8 of block 2 w + y
              const uint32_t lo = __byte_perm(x4[0][w], x4[1][w], y ? 0x7362 : 0x5140);
              const uint32_t hi = __byte_perm(x4[2][w], x4[3][w], y ? 0x7362 : 0x5140);
              const uint32_t a0 = half2_of(lo), a1 = half2_of_high(lo), a2 = half2_of(hi), a3 = half2_of_high(hi);
#pragma unroll
              for (int t = 0; t < kTiles; ++t) mma16816(acc[t][2 * w + y], a0, a1, a2, a3, p[t][2 * j], p[t][2 * j + 1]);
            }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int d = 0; d < 8 / kPasses; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float& e = o[t][pass * (8 / kPasses) + d][i];
              e = fmaf(acc[t][d][i], cur.vs, e);
            }
      }
      __syncwarp();
    } else {
      load(&v_map, slot, nxt.at);
    }
    load(&k_map, vslot, far.at);               // the values' buffer is free: the keys after the next ones

    // ---- the end of a segment ---------------------------------------------------------
    if (now.page == now.pages - 1 || it == n - 1) {
      const bool whole = now.page == now.pages - 1 && it >= now.page;   // the segment began in this range
      const int64_t slot_of_part = 2 * x + (parts > 0 ? 1 : 0);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float sum = l[t][i];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          const int hh = 8 * t + 2 * tig + i;
          if (hh >= heads) continue;
          const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
          if (whole) {
            T* const out = static_cast<T*>(a.out) + (static_cast<int64_t>(now.row) * a.heads + head0 + hh) * 128 + 16 * g;
            uint32_t w[8];
#pragma unroll
            for (int d = 0; d < 8; ++d) w[d] = pack2<T>(o[t][d][i] * inv, o[t][d][2 + i] * inv);
            *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(out + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            if (g == 0)
              a.lse[static_cast<int64_t>(now.row) * a.heads + head0 + hh] =
                  sum > 0.0f ? (m[t][i] + log2f(sum)) * kLn2 : (sum == 0.0f ? -CUDART_INF_F : sum);
          } else {
            float* const part = a.part + (slot_of_part * kHeads + hh) * 128 + 16 * g;
#pragma unroll
            for (int d = 0; d < 8; d += 2)
              *reinterpret_cast<float4*>(part + 2 * d) = make_float4(o[t][d][i], o[t][d][2 + i], o[t][d + 1][i], o[t][d + 1][2 + i]);
            if (g == 0) {
              a.part_ml[2 * (slot_of_part * kHeads + hh)] = m[t][i];
              a.part_ml[2 * (slot_of_part * kHeads + hh) + 1] = sum;
            }
          }
        }
      ++parts;
      fresh = true;
    }
    next(now);
    cur = nxt;
    nxt = far;
    slot = vslot + 1 == kRing ? 0 : vslot + 1;
  }
  if (!state.ok)   // what is under way lands before the CTA ends
    for (int i = 0; i < kRing; ++i)
      if (state.under_way(i)) mbar_wait(&full[i], state.phase(i), &sh.zero, kWaitNs);
  // ---- rows that have no page ----------------------------------------------------------
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    if (row_pages(a, r) > 0) continue;
    uint4* const out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + r * a.heads * 128);
    for (int64_t i = tid; i < a.heads * 16; i += kWarps * 32) out[i] = make_uint4(0, 0, 0, 0);
    for (int64_t i = tid; i < a.heads; i += kWarps * 32) a.lse[r * a.heads + i] = -CUDART_INF_F;
  }
}

// Joins the parts of the segments that lie in several ranges, in the order of the
// ranges.  Range y's part is its first (slot 0) unless the range begins in an earlier
// segment (then its last, slot 1); a range may be empty.  kShare warps share the parts
// of one head.  Grid x: with kShare = 1 the segment in which range x + 1 begins, if
// that is the first range to begin inside it (many segments of a few parts); else
// the segment x (a few of many parts).
template <typename T, int kTiles, int kShare>
__global__ void __launch_bounds__(kShare == 1 ? 128 : 32 * kShare) kv8_join_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int kHeads = 8 * kTiles;
  __shared__ float4 sums[kShare][32];
  __shared__ float ls[kShare];
  wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int x = blockIdx.x + 1;
  if constexpr (kShare > 1) {
    __shared__ int found;
    if (threadIdx.x == 0) found = kMaxRanges;
    __syncthreads();
    for (int i = threadIdx.x + 1; i < a.ranges; i += 32 * kShare)
      if (a.where[4 * i] == blockIdx.x && begins_inside(record_of(a.where, i))) atomicMin(&found, i);
    __syncthreads();
    x = found;
    if (x == kMaxRanges) return;
  }
  const RangeBegin cut = record_of(a.where, x);
  const int64_t before = begin_of(a.where, x - 1);
  if (!cuts_first(cut, before)) return;
  const int64_t place = cut.place, end = cut.first + cut.tiles;
  const int64_t row = place / a.segments, segment = place - row * a.segments;
  const int group = static_cast<int>(segment % a.groups), hg = kShare == 1 ? blockIdx.y * 4 + warp : blockIdx.y;
  if (hg >= min(kHeads, a.per_kv - group * kHeads)) return;   // kShare > 1: the whole block
  const int64_t h = segment / a.groups * a.per_kv + group * kHeads + hg;
  const int64_t shift = before < cut.first ? kHeads : 0;
  auto part = [&](int i) { return static_cast<int64_t>(x - 1 + i) * 2 * kHeads + hg + (i == 0 ? shift : 0); };
  float m = -CUDART_INF_F, l = 0.0f;
  int parts = 0;
  for (int i = lane; i <= a.ranges - x; i += 32) {
    const int64_t t0 = begin_of(a.where, x - 1 + i), t1 = begin_of(a.where, x + i);
    if (t0 >= end) break;
    parts = i + 1;
    if (t1 > t0) m = fmaxf(m, a.part_ml[2 * part(i)]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    parts = max(parts, __shfl_xor_sync(0xffffffffu, parts, o));
  }
  const float ref = m == -CUDART_INF_F ? 0.0f : m;
  float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 8
  for (int i = kShare == 1 ? 0 : warp; i < parts; i += kShare) {
    if (begin_of(a.where, x + i) == begin_of(a.where, x - 1 + i)) continue;
    const float w = exp2f(a.part_ml[2 * part(i)] - ref);
    l += a.part_ml[2 * part(i) + 1] * w;
    const float4 v = *reinterpret_cast<const float4*>(a.part + part(i) * 128 + 4 * lane);
    o = make_float4(fmaf(v.x, w, o.x), fmaf(v.y, w, o.y), fmaf(v.z, w, o.z), fmaf(v.w, w, o.w));
  }
  if constexpr (kShare > 1) {
    sums[warp][lane] = o;
    if (lane == 0) ls[warp] = l;
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < kShare; ++w) {
      const float4 v = sums[w][lane];
      o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
      l += ls[w];
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (row * a.heads + h) * 128 + 4 * lane) =
      make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
  if (lane == 0) a.lse[row * a.heads + h] = l > 0.0f ? (m + log2f(l)) * kLn2 : (l == 0.0f ? -CUDART_INF_F : l);
}

struct Plan {
  int64_t tiles, groups, segments, ranges;
};
Plan plan_for(int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_pages) {
  Plan p;
  const int64_t per = heads / kv_heads;
  // one 8-column operand where it holds all the heads, else two (64 rows of 1-16 K
  // tokens: 8 heads a K/V head 103 us with one, 169 with two; 16 heads 184 and 157)
  p.tiles = per <= 8 ? 1 : 2;
  p.groups = (per + 8 * p.tiles - 1) / (8 * p.tiles);
  p.segments = kv_heads * p.groups;
  const int64_t pages = rows * p.segments * table_pages;
  p.ranges = pages < kMaxRanges ? (pages > 0 ? pages : 1) : kMaxRanges;
  return p;
}

template <typename T, int kTiles>
void launch_attend(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendArgs& a, cudaStream_t s) {
  constexpr int kSmem = 1024 + kWarps * kRing * kPageBytes8 + static_cast<int>(sizeof(AttendShared));
  static_assert(kSmem <= 232448, "shared memory");
  static DeviceOnce once;
  once.run([] { cudaFuncSetAttribute(kv8_attend_kernel<T, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem); });
  const unsigned ctas = static_cast<unsigned>(a.ranges < 148 ? a.ranges : 148);
  launch_kernel_prio(LaunchPriority::kDefault, kv8_attend_kernel<T, kTiles>, dim3(ctas), dim3(kWarps * 32), kSmem, s, k_map,
                     v_map, a);
  if (a.ranges == 1) return;
  const unsigned cuts = static_cast<unsigned>(a.ranges - 1), heads = 8 * kTiles;
  // many parts a segment, or few segments: one row of 4097 tokens 13 us so, 37 with one
  // warp a head, of 512 tokens 9.9 and 11.3, 18 rows of 4097 29.3 and 31.4; else 24 rows
  // 37.8 and 35.3, 64 rows 74 and 58
  if (a.ranges >= 16 * a.rows * a.segments || a.rows * a.segments <= 8)
    launch_join(kv8_join_kernel<T, kTiles, 16>, dim3(static_cast<unsigned>(a.rows * a.segments), heads), dim3(512), s, a);
  else
    launch_join(kv8_join_kernel<T, kTiles, 1>, dim3(cuts, heads / 4), dim3(128), s, a);
}

// Rows of 128 codes, 64 (a page and head) a box, 128-byte swizzle.
int encode_cache(CUtensorMap* map, const uint8_t* cache, int64_t blocks) {
  const PFN_cuTensorMapEncodeTiled_v12000 fn = map_encoder();
  if (!fn) {
    set_error("kv8_attend: cuTensorMapEncodeTiled unavailable");
    return V1X_ERR_CUDA;
  }
  const cuuint64_t dims[2] = {128, static_cast<cuuint64_t>(blocks * 64)}, strides[1] = {128};
  const cuuint32_t box[2] = {128, 64}, steps[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(cache), dims, strides, box, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("kv8_attend: tensor map encode failed (%d)", static_cast<int>(r));
    return V1X_ERR_CUDA;
  }
  return V1X_OK;
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
  const dim3 grid(static_cast<unsigned>(tokens / 64 + 2 * requests), static_cast<unsigned>((2 * heads + 3) / 4));
  if (dtype == 1)
    launch_kernel_prio(LaunchPriority::kDefault, kv8_store_kernel<__nv_bfloat16>, grid, dim3(128), 0, as_stream(stream), a);
  else
    launch_kernel_prio(LaunchPriority::kDefault, kv8_store_kernel<__half>, grid, dim3(128), 0, as_stream(stream), a);
  return launch_status("v1x_kv8_store");
}

extern "C" int64_t v1x_kv8_attend_workspace(int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_pages) {
  using namespace v1x;
  if (rows <= 0 || kv_heads <= 0 || heads <= 0 || heads > 1024 || heads % kv_heads || table_pages <= 0) return 0;
  const Plan p = plan_for(rows, heads, kv_heads, table_pages);
  return p.ranges == 1 ? 0 : (p.ranges + 1) * 32 + p.ranges * 2 * 8 * p.tiles * (128 + 2) * 4;
}

extern "C" int v1x_kv8_attend(const void* q, int64_t qs0, int64_t qs1, const uint8_t* k_cache, const float* k_scale,
                              const uint8_t* v_cache, const float* v_scale, int64_t pages, int64_t kv_heads,
                              const int32_t* table, int64_t table_stride, int64_t table_pages, const int32_t* lens,
                              int64_t rows, int64_t heads, float scale, int dtype, void* out, float* lse,
                              void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
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
  V1X_CHECK_ARG(scale_in_range(scale), "kv8_attend: the scale must be finite and below 2^127");
  if (rows == 0) return V1X_OK;
  V1X_CHECK_ARG(q && out && lse && lens && (table || table_pages == 0) &&
                    ((k_cache && k_scale && v_cache && v_scale) || pages == 0),
                "kv8_attend: NULL argument");
  V1X_CHECK_ARG(pages * kv_heads < (int64_t(1) << 25), "kv8_attend: at most 2^25 pages x K/V heads");
  V1X_CHECK_ARG(table_pages < (int64_t(1) << 25) && kv_heads * table_pages <= (int64_t(1) << 34) / rows,
                "kv8_attend: at most 2^25 table columns, 2^34 rows x K/V heads x columns");
  const int64_t need = v1x_kv8_attend_workspace(rows, heads, kv_heads, table_pages);
  V1X_CHECK_ARG(workspace_bytes >= need && (workspace || need == 0) && aligned16(workspace),
                "kv8_attend: the workspace must be 16-byte aligned and hold %lld bytes", static_cast<long long>(need));
  if (pages == 0) table_pages = 0;   // no page is in the cache: every row is empty
  const Plan p = plan_for(rows, heads, kv_heads, table_pages);
  AttendArgs a{q, qs0, qs1, k_scale, v_scale, pages, kv_heads, table, table_stride, table_pages, lens, rows, heads,
               static_cast<int>(heads / kv_heads), static_cast<int>(p.groups), static_cast<int>(p.segments),
               static_cast<int>(p.ranges), scale * kLog2e, out, lse, nullptr, nullptr, nullptr, status};
  if (p.ranges > 1) {
    a.where = static_cast<int64_t*>(workspace);
    a.part = reinterpret_cast<float*>(a.where + 4 * (p.ranges + 1));
    a.part_ml = a.part + p.ranges * 2 * 8 * p.tiles * 128;
  }
  CUtensorMap k_map = {}, v_map = {};
  if (pages > 0) {
    if (int rc = encode_cache(&k_map, k_cache, pages * kv_heads)) return rc;
    if (int rc = encode_cache(&v_map, v_cache, pages * kv_heads)) return rc;
  }
  cudaStream_t s = as_stream(stream);
  if (dtype == 1) p.tiles == 1 ? launch_attend<__nv_bfloat16, 1>(k_map, v_map, a, s) : launch_attend<__nv_bfloat16, 2>(k_map, v_map, a, s);
  else p.tiles == 1 ? launch_attend<__half, 1>(k_map, v_map, a, s) : launch_attend<__half, 2>(k_map, v_map, a, s);
  return launch_status("v1x_kv8_attend");
}
