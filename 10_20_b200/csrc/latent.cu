// Latent attention, absorbed form, on the tensor cores: see v1x_latent_attention
// in v1x.h.
//
// Every head reads the same rows, as keys (all of a row) and as values (its first
// `latent` elements), so a tile of 64 tokens is brought into shared memory once
// and is an operand of both products:
//
//   S[64 heads x 64 tokens]      = Q . K^T        M = 64, N = 64, K = dim
//   O^T[128 of latent x heads]  += V^T . P^T      M = 128, N = heads, K = 64
//
// The output is kept transposed because its M is then the latent width, full
// 128-row operands for any number of heads, and its four accumulators of 64
// columns leave room for two score tiles.  The same bytes serve as K-major (keys)
// and MN-major (values) operand.  Softmax in one pass, in powers of two: the
// running maximum that the weights are taken against moves only when a tile
// exceeds it by more than 2^8, so that O is rescaled a few times a row at most;
// sums stay in 32 bits, the weights are rounded once, to the inputs' type, for the
// second product.
//
// What bounds it: 72 KB of queries leave room for 144 KB of tokens, two tiles, and
// a tile is held from its first load to its last product, a chain of latencies
// (load 2000 cycles, scores 1500, softmax 1400, output 600; 3600 a tile with two in
// flight, of which its MMAs need 1920).  So a tile is loaded, weighted and released
// in two halves of 32 tokens, and its scores begin on the first blocks.  128 rows of
// 2048 tokens, 64 heads: 81 us, 3.9 TB/s; 1024 rows, 128 heads: 929 us, 628 TFLOP/s.
// Measured and not kept: four tiles of 32 (80 and 1004 us: N = 32 costs the scores a
// quarter of the rate), whole pages by TMA (116 instead of 107 us on 48 ragged rows),
// each half copied by all eight warps in turn (103 us); the tensor-map gather of four
// rows moves 8 bytes a cycle and SM.
//
// Work: the tiles of all rows in a line, cut into equal ranges, one CTA each (times
// the groups of 64 heads, neighbours in the grid, which read the same tiles at the
// same time from L2).  A row that lies in several ranges leaves unnormalised parts
// in the workspace, joined by latent_join_kernel in the order of the ranges; rows
// of equal length are given to the CTAs whole where that is no longer, and a few of
// them to a cluster each, whose CTAs join their parts through shared memory (cut_for).
//
// Warp roles (512 threads, one CTA per SM):
//   0-3   softmax, rescale, epilogue (TMEM lane quarters 0-3)
//   4-11  four sets of two producer warps, a half of every other tile each: rows by
//         16-byte cp.async into the swizzled layout, each row's slot looked up a
//         tile ahead; a token that is none becomes zeros and a cleared bit of the
//         tile's mask
//   12, 14  issue the scores' MMAs of even and odd tiles (12 owns the TMEM); 13 the
//         outputs', a half of a tile at a time.  An MMA of these shapes takes 32 to 48
//         cycles and few are queued: one warp's waits between the two products left
//         the tensor cores idle (111 us instead of 92 on the decode batch)
//   15    the queries, when the row changes
// Waits are bounded (2 s, then V1X_STATUS_TIMEOUT).
#include <cooperative_groups.h>

#include <type_traits>

#include "attention.cuh"
#include "ranges.cuh"
#include "sm100.cuh"

namespace v1x {
namespace {

using namespace attn;
using namespace sm100;

constexpr int kTile = 64;                // tokens of a tile, in two halves
constexpr int kGroup = 64;               // heads of a CTA
constexpr int kBlock = 64 * 128;         // bytes of 64 elements of 64 rows (queries, tokens) or of the weights
constexpr int kMaxPairs = 4;             // tiles in shared memory: 2, or 4 where they fit
constexpr int kThreads = 512;
constexpr int kMaxCtas = 148;
constexpr uint32_t kScoreCol = 256;      // TMEM: O^T in columns 0-255, two score tiles after it
constexpr float kLazy = 8.0f;            // log2 of the growth that the weights may show before a rescale
constexpr uint64_t kWaitNs = 2000000000ull;

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
  int pairs, groups, ranges;
  int share;                   // CTAs of a cluster, which have a row's tiles together
  int64_t unit, base, extra;   // the cut of the line in units of `unit` tiles (lens: unit 1, on the device)
  float scale_log2;
  void* out;
  float* lse;
  float* part;       // [ranges * groups][2][16][latent][4]: four heads' values side by side; then [..][2][2][64] maxima, sums
  float* part_ml;
  int64_t* where;    // [ranges + 1][4]: the ranges' records
  int32_t* status;
};

// what a tile is in its segment (the tiles of one row in a CTA's range; segments
// are counted from kSegment on)
constexpr uint32_t kFirst = 1, kLastOfRow = 2, kBeforeLast = 4, kSegment = 8;

struct LatentShared {
  uint64_t full[2 * kMaxPairs];    // of a tile: its first blocks, all of it
  uint64_t empty[2 * kMaxPairs];   // its halves
  uint64_t s_full[2], p_full[2][2], pv_done[2], q_full, q_empty;   // p_full, pv_done: of a tile's halves
  uint64_t mask[kMaxPairs];
  uint32_t flags[kMaxPairs];
  alignas(16) float factor[kGroup];
  float m[kGroup], l[kGroup];      // of a cluster's CTA
  RangeBegin start;
  int64_t all;       // tiles
  int64_t cut[2];    // base, extra
  int64_t scan[kThreads / 32 + 1];
  uint32_t tmem;
  int abort, zero;
};

__device__ __forceinline__ int64_t row_len(const LatentArgs& a, int64_t r) {
  return a.lens ? min(static_cast<int64_t>(max(a.lens[r], 0)), a.count) : a.count;
}
__device__ __forceinline__ int64_t row_tiles(const LatentArgs& a, int64_t r) { return (row_len(a, r) + kTile - 1) / kTile; }

// A place in the line of tiles.
struct Place {
  int row, tile, tiles;  // the row, the tile of the row, the row's tiles
  __device__ bool first() const { return tile == 0; }
  __device__ bool last() const { return tile == tiles - 1; }
  __device__ void next(const LatentArgs& a) {
    if (++tile < tiles) return;
    tile = 0;
    do {
      ++row;
      tiles = row < a.rows ? static_cast<int>(row_tiles(a, row)) : 1;
    } while (tiles == 0);
  }
};

// The pool slot of token j of row r, or -1 if there is none.
__device__ __forceinline__ int64_t slot_of(const LatentArgs& a, int64_t r, int64_t j) {
  if (j >= row_len(a, r)) return -1;
  const int32_t* index = a.index + r * a.index_stride;
  int64_t s;
  if (a.lens) {
    s = static_cast<int64_t>(index[j >> 6]) * 64 + (j & 63);
  } else {
    s = index[j];
    if (a.req) s = s >= 0 && s < a.req_len ? a.req[s] : -1;
  }
  return s >= 0 && s < a.slots ? s : -1;
}

__device__ __forceinline__ void give_up(LatentShared& sh, int32_t* status) {
  *reinterpret_cast<volatile int*>(&sh.abort) = 1;
  if (status) atomicExch(status, V1X_STATUS_TIMEOUT);
}

// A whole warp waits, and agrees on the outcome.
__device__ __forceinline__ bool converged_wait(LatentShared& sh, int32_t* status, uint64_t* bar, int phase) {
  bool ok = __all_sync(0xffffffffu, mbar_test(bar, phase & 1));   // most phases are complete when asked for
  if (!ok) {
    ok = __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, &sh.abort, kWaitNs));
    if (!ok) give_up(sh, status);
  }
  tc_fence_after();
  return ok;
}

__device__ __forceinline__ bool any_of_128(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x))
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void sync_128() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

// Rows into the swizzled operand layout, 64 elements a block: row R of block c at
// c * kBlock + R * 128, its 16-byte pieces permuted by R & 7.  A group of eight
// lanes moves one 128-byte piece of a row at a time; the warp covers the 16 rows
// R0 .. R0 + 15, whose sources (per lane l < 16: row R0 + l, null for zeros, `any`
// then being an address that is not read) are handed over by shuffles.
struct RowCopy {
  const char* from[4];
  uint32_t to[4], bytes[4];
  __device__ __forceinline__ RowCopy(uint32_t dst, const char* src, const void* any, int R0, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * i + (lane >> 3), R = R0 + row;
      const char* p = reinterpret_cast<const char*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), row));
      bytes[i] = p ? 16 : 0;
      from[i] = p ? p + (lane & 7) * 16 : static_cast<const char*>(any);
      to[i] = dst + R * 128 + (((lane & 7) ^ (R & 7)) << 4);
    }
  }
  template <int kBegin, int kEnd>
  __device__ __forceinline__ void blocks() const {
#pragma unroll
    for (int c = kBegin; c < kEnd; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) cp_async16(to[i] + c * kBlock, from[i] + c * 128, bytes[i]);
  }
};

// kCluster: the CTAs of a cluster have one row, an equal part of its tiles each.
template <typename T, int kLatent, int kRope, bool kCluster>
__global__ void __launch_bounds__(kThreads, 1) latent_kernel(const __grid_constant__ LatentArgs a) {
  constexpr int kChunks = (kLatent + kRope) / 64, kOut = kLatent / 128;
  constexpr int kEarly = (kChunks + 1) / 2;   // the blocks that the scores begin with
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_smem = smem_u32(base);
  const uint32_t kv_smem = q_smem + kChunks * kBlock;
  uint8_t* p_ptr = base + kChunks * (1 + a.pairs) * kBlock;
  const uint32_t p_smem = smem_u32(p_ptr);
  LatentShared& sh = *reinterpret_cast<LatentShared*>(p_ptr + kBlock);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = kCluster ? blockIdx.x % a.share : 0, cta = kCluster ? blockIdx.x / a.share : blockIdx.x;
  const int group = cta % a.groups;
  const int64_t x = cta / a.groups;            // the range; kCluster: the row
  const int heads = min(kGroup, static_cast<int>(a.heads - group * kGroup));

  if (tid == 0) {
    sh.abort = 0;
    sh.zero = 0;
    for (int s = 0; s < 2 * a.pairs; ++s) {
      mbar_init(&sh.full[s], 4);
      mbar_init(&sh.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i][0], 4);
      mbar_init(&sh.p_full[i][1], 4);
      mbar_init(&sh.pv_done[i], 1);
    }
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 2);
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  // ---- this CTA's range of the line ---------------------------------------------
  if (!a.lens) {
    if (tid == 0) {
      const int64_t per = (a.count + kTile - 1) / kTile, t0 = range_start(x, a.unit, a.base, a.extra);
      const int64_t row = kCluster ? x : per ? (t0 >> 31 ? t0 / per : static_cast<uint32_t>(t0) / static_cast<uint32_t>(per)) : 0;
      sh.start = RangeBegin{row, row * per, per, t0};
      sh.all = per * a.rows;
      sh.cut[0] = a.base;
      sh.cut[1] = a.extra;
    }
    __syncthreads();
  } else {
    const int64_t chunk = (a.rows + kThreads - 1) / kThreads;
    const int64_t beg = min(tid * chunk, a.rows), end = min(beg + chunk, a.rows);
    int64_t mine = 0, all;
    for (int64_t r = beg; r < end; ++r) mine += row_tiles(a, r);
    const int64_t run = block_exclusive_scan(mine, sh.scan, &all);
    if (tid == 0) {
      sh.all = all;
      sh.cut[0] = all >> 31 ? all / a.ranges : static_cast<uint32_t>(all) / static_cast<uint32_t>(a.ranges);
      sh.cut[1] = all - sh.cut[0] * a.ranges;
    }
    __syncthreads();
    const int64_t t0 = range_start(x, 1, sh.cut[0], sh.cut[1]);
    if (t0 >= all) {
      if (tid == 0) sh.start = no_row(t0);
    } else if (run <= t0 && t0 < run + mine) {
      sh.start = find_begin(t0, beg, end, run, [&](int64_t r) { return row_tiles(a, r); });
    }
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const int64_t per = sh.start.tiles;
  const int64_t t0 = kCluster ? x * per + per * rank / a.share : range_start(x, a.unit, sh.cut[0], sh.cut[1]);
  const int64_t t1 = kCluster ? x * per + per * (rank + 1) / a.share : range_start(x + 1, a.unit, sh.cut[0], sh.cut[1]);
  const int n = static_cast<int>(t1 - t0);     // tiles of the range
  Place at{static_cast<int>(sh.start.place), static_cast<int>(t0 - sh.start.first), static_cast<int>(sh.start.tiles)};
  if (tid == 0 && group == 0 && a.where) {
    put_record(a.where, x, sh.start);
    if (x == a.ranges - 1) a.where[4 * x + 7] = sh.all;
  }

  if (warp < 4) {
    // ---------------- softmax, rescale, epilogue ----------------
    // M = 64 fills the lower half of each lane quarter: a head belongs to two
    // threads, the even and the odd tokens of a tile
    const int h = 16 * warp + (lane >> 2) + 8 * (lane & 1), odd = (lane >> 1) & 1;
    const bool mine = odd == 0;                  // the one that speaks for the head
    const uint32_t quarter = static_cast<uint32_t>(warp * 32) << 16;
    const int cols = (heads + 31) & ~31;         // accumulator columns moved, 32 at a time
    float m = -CUDART_INF_F, l = 0.0f;
    bool fresh = true;                           // the tile begins a segment: tiles of one row in this range
    int segment = 0, segment_tile = 0, pair = 0, turn = 0;
    // after a wait that gave up the loop goes on without waiting, so that all
    // four warps still meet at their barriers
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase) {
      if (ok && !mbar_test(bar, phase & 1) && !mbar_wait(bar, phase & 1, &sh.abort, kWaitNs)) {
        give_up(sh, a.status);
        ok = false;
      }
    };
    for (int it = 0; it < n; ++it) {
      wait(&sh.s_full[it & 1], it >> 1);
      tc_fence_after();
      uint32_t raw[32];
      tmem_ld16x64(tmem + quarter + kScoreCol + (it & 1) * kTile, raw);
      wait(&sh.full[2 * pair], turn);            // complete already: the producers' mask
      const uint64_t valid = *reinterpret_cast<volatile uint64_t*>(&sh.mask[pair]);
      if (++pair == a.pairs) {
        pair = 0;
        ++turn;
      }
      tmem_ld_wait();
      float s[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) s[j] = __uint_as_float(raw[j]) * a.scale_log2;
      if (valid != ~0ull) {
        const uint64_t own = valid >> odd;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!((own >> (2 * j)) & 1)) s[j] = -CUDART_INF_F;
      }
      float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int j = 4; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], s[j]);
      float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2)) - lift<T>(kLazy);   // m: the weights' reference
      if (fresh) {
        m = most;
        l = 0.0f;
        segment_tile = at.tile;
      } else {
        const bool grows = most > m + kLazy;
        if (any_of_128(grows)) {
          const float f = grows ? exp2_fast(m - most) : 1.0f;
          if (grows) m = most;
          l *= f;
          if (mine) sh.factor[h] = f;
          wait(&sh.pv_done[1], it - 1);
          sync_128();
          tc_fence_after();
          for (int t = 0; t < kOut; ++t)
            for (int c = 0; c < cols; c += 32) {
              const uint32_t addr = tmem + quarter + t * 64 + c;
              uint32_t o[32];
              tmem_ld32(addr, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * sh.factor[c + j]);
              tmem_st32(addr, o);
            }
          tmem_st_wait();
        }
      }
      fresh = false;
      const float ref = m == -CUDART_INF_F ? 0.0f : m;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      // the halves' weights are handed over one after the other
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float* const e = s + 16 * half;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          e[j] = exp2_fast(e[j] - ref);
          sum[j & 3] += e[j];
        }
        // neighbouring tokens' weights meet in one thread: the half's tokens 0-15 in the
        // even one, 16-31 in the odd one
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float got = __shfl_xor_sync(0xffffffffu, odd ? e[j] : e[j + 8], 2);
          w[j] = odd ? pack2<T>(got, e[j + 8]) : pack2<T>(e[j], got);
        }
        // their buffer is free once the previous tile's product has read it
        if (it > 0) wait(&sh.pv_done[half], it - 1);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<uint4*>(p_ptr + h * 128 + (((half * 4 + odd * 2 + c) ^ (h & 7)) << 4)) =
              make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        fence_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[it & 1][half]);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);

      if (at.last() || it == n - 1) {
        wait(&sh.pv_done[1], it);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        tc_fence_after();
        if constexpr (kCluster) {
          // the CTA's only segment: its part goes where queries and tiles were, 64 columns of
          // all heads side by side
          if (mine) {
            sh.m[h] = m;
            sh.l[h] = l;
          }
#pragma unroll 1
          for (int t = 0; t < kOut; ++t)
#pragma unroll 1
            for (int c = 0; c < cols; c += 32) {
              uint32_t o[32];
              tmem_ld32(tmem + quarter + t * 64 + c, o);
              tmem_ld_wait();
              float* const to = reinterpret_cast<float*>(base) + ((2 * t + (warp >> 1)) * kGroup + c) * 64 + (warp & 1) * 32 + lane;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j < heads) to[j * 64] = __uint_as_float(o[j]);
            }
          tc_fence_before();
          break;
        }
        const bool whole = at.last() && segment_tile == 0;   // all of the row's tiles were here
        const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (segment > 0 ? 1 : 0));
        float* part = a.part + slot * kGroup * kLatent;
        if (mine) {
          const int64_t o = static_cast<int64_t>(at.row) * a.heads + group * kGroup + h;
          if (whole) {
            sh.factor[h] = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
            if (h < heads) a.lse[o] = l > 0.0f ? (m + log2f(l)) * kLn2 : (l == 0.0f ? -CUDART_INF_F : l);
          } else if (h < heads) {
            a.part_ml[slot * 2 * kGroup + h] = m;
            a.part_ml[slot * 2 * kGroup + kGroup + h] = l;
          }
        }
        sync_128();
        T* const out = static_cast<T*>(a.out) + (static_cast<int64_t>(at.row) * a.heads + group * kGroup) * kLatent;
        const int d = warp * 32 + lane;
        if (whole) {
          // 32 heads x 32 columns at a time through the warp's quarter of the weights'
          // buffer (free: the last product has read it), so that a lane writes 16 bytes
          // of a head and four of them its 64
          uint8_t* const mine_p = p_ptr + warp * (kBlock / 4);
          uint16_t* const put = reinterpret_cast<uint16_t*>(mine_p) + lane;
          T* const to = out + warp * 32 + (lane & 3) * 8;
#pragma unroll 1
          for (int t = 0; t < kOut; ++t)
#pragma unroll 1
            for (int c = 0; c < cols; c += 32) {
              uint32_t o[32];
              tmem_ld32(tmem + quarter + t * 64 + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 f = *reinterpret_cast<const float4*>(&sh.factor[c + j]);
                const uint32_t u = pack2<T>(__uint_as_float(o[j]) * f.x, __uint_as_float(o[j + 1]) * f.y);
                const uint32_t v = pack2<T>(__uint_as_float(o[j + 2]) * f.z, __uint_as_float(o[j + 3]) * f.w);
                put[j * 32] = static_cast<uint16_t>(u);
                put[(j + 1) * 32] = static_cast<uint16_t>(u >> 16);
                put[(j + 2) * 32] = static_cast<uint16_t>(v);
                put[(j + 3) * 32] = static_cast<uint16_t>(v >> 16);
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int hh = c + 8 * i + (lane >> 2);
                const uint4 v = *reinterpret_cast<const uint4*>(mine_p + i * 512 + lane * 16);
                if (hh < heads) *reinterpret_cast<uint4*>(to + hh * kLatent + t * 128) = v;
              }
              __syncwarp();
            }
        } else {
#pragma unroll 1
          for (int t = 0; t < kOut; ++t)
#pragma unroll 1
            for (int c = 0; c < cols; c += 32) {
              uint32_t o[32];
              tmem_ld32(tmem + quarter + t * 64 + c, o);
              tmem_ld_wait();
              float* const to = part + c * kLatent + (t * 128 + d) * 4;
#pragma unroll
              for (int j = 0; j < 32; j += 4)
                if (c + j < heads)
                  *reinterpret_cast<float4*>(to + j * kLatent) =
                      make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]), __uint_as_float(o[j + 2]), __uint_as_float(o[j + 3]));
            }
        }
        tc_fence_before();
        sync_128();                              // factor is free again
        ++segment;
        fresh = true;
      }
      at.next(a);
    }
    // rows that have no tile
    if (a.lens || a.count == 0) {
      for (int64_t r = x; r < a.rows; r += a.ranges) {
        if (row_len(a, r) > 0) continue;
        uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (r * a.heads + group * kGroup) * kLatent);
        for (int i = tid; i < heads * kLatent / 8; i += 128) out[i] = make_uint4(0, 0, 0, 0);
        if (tid < heads) a.lse[r * a.heads + group * kGroup + tid] = -CUDART_INF_F;
      }
    }
  } else if (warp < 12) {
    // ---------------- producers ----------------
    const int half = (warp >> 1) & 1, turn_of = (warp - 4) >> 2, R0 = 32 * half + 16 * (warp & 1);
    int segment = 0;
    auto step = [&] {
      if (at.last()) ++segment;
      at.next(a);
    };
    int pair = turn_of, turn = 0;                // tiles turn_of, turn_of + 2, ...; the number of pairs is even
    if (turn_of < n)
      for (int i = 0; i < turn_of; ++i) step();
    auto slot_ahead = [&] {
      return lane < 16 ? slot_of(a, at.row, at.tile * static_cast<int64_t>(kTile) + R0 + lane) : -1;
    };
    int64_t slot = turn_of < n ? slot_ahead() : -1;
    for (int it = turn_of; it < n; it += 2) {
      if (!converged_wait(sh, a.status, &sh.empty[2 * pair + half], turn ^ 1)) break;
      const unsigned some = __ballot_sync(0xffffffffu, slot >= 0) & 0xFFFFu;
      if (lane == 0) {
        reinterpret_cast<volatile uint16_t*>(&sh.mask[pair])[R0 >> 4] = static_cast<uint16_t>(some);
        if (R0 == 0)
          *reinterpret_cast<volatile uint32_t*>(&sh.flags[pair]) =
              (it == 0 || at.first() ? kFirst : 0) | (at.last() ? kLastOfRow : 0) |
              (at.tile == at.tiles - 2 ? kBeforeLast : 0) | static_cast<uint32_t>(segment) * kSegment;
      }
      const char* src = slot >= 0 ? static_cast<const char*>(a.pool) + slot * a.pool_stride * 2 : nullptr;
      const RowCopy copy(kv_smem + pair * kChunks * kBlock, src, a.q, R0, lane);
      copy.template blocks<0, kEarly>();
      cp_async_commit();
      copy.template blocks<kEarly, kChunks>();
      cp_async_commit();
      if (it + 2 < n) {   // the next tile's slots arrive while this one's rows do
        step();
        step();
        slot = slot_ahead();
      }
      cp_async_wait<1>();
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.full[2 * pair]);
      cp_async_wait<0>();
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.full[2 * pair + 1]);
      pair += 2;
      if (pair >= a.pairs) {
        pair = turn_of;
        ++turn;
      }
    }
    cp_async_wait_all();
  } else if (warp == 12 || warp == 14) {
    // ---------------- scores: even tiles, odd tiles ----------------
    const uint32_t qk = idesc_16bit_f32(kBf16, kGroup, kTile, false, false), q_desc = desc_k(q_smem);
    const int mine = warp == 14;
    int pair = mine, turn = 0, scored = -1;
    // both warps take and give back every segment's queries, in order: also those of a
    // segment whose only tile is the other warp's
    int segment = 0;
    bool held = false;
    for (int it = mine; it < n; it += 2) {
      if (it >= 2 && !converged_wait(sh, a.status, &sh.p_full[it & 1][1], (it - 2) >> 1)) break;   // S is free again
      if (!converged_wait(sh, a.status, &sh.full[2 * pair], turn)) break;
      const uint32_t flags = *reinterpret_cast<volatile uint32_t*>(&sh.flags[pair]);
      bool ok = true;
      for (const int now = static_cast<int>(flags / kSegment); segment < now && ok; ++segment) {
        ok = converged_wait(sh, a.status, &sh.q_full, segment);
        if (ok) umma_commit_elect(&sh.q_empty);
      }
      if (ok && !held) ok = held = converged_wait(sh, a.status, &sh.q_full, segment);
      if (!ok) break;
      const uint32_t k_desc = desc_k(kv_smem + pair * kChunks * kBlock), d = tmem + kScoreCol + (it & 1) * kTile;
#pragma unroll
      for (int c = 0; c < kEarly; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(d, q_desc + (c * kBlock + 32 * k) / 16, k_desc + (c * kBlock + 32 * k) / 16, qk, c + k > 0 ? 1u : 0u);
      const bool whole = converged_wait(sh, a.status, &sh.full[2 * pair + 1], turn);
      if (whole) {
#pragma unroll
        for (int c = kEarly; c < kChunks; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(d, q_desc + (c * kBlock + 32 * k) / 16, k_desc + (c * kBlock + 32 * k) / 16, qk, 1u);
      }
      umma_commit_elect(&sh.s_full[it & 1]);
      scored = it;
      if (!whole) break;
      if (__any_sync(0xffffffffu, flags & (kLastOfRow | kBeforeLast))) {   // this warp's last tile of the row
        umma_commit_elect(&sh.q_empty);
        ++segment;
        held = false;
      }
      pair += 2;
      if (pair >= a.pairs) {
        pair = mine;
        ++turn;
      }
    }
    // what was issued retires before the CTA ends
    if (scored >= 0) mbar_wait(&sh.s_full[scored & 1], (scored >> 1) & 1, &sh.zero, kWaitNs);
  } else if (warp == 13) {
    // ---------------- output ----------------
    const uint32_t pv = idesc_16bit_f32(kBf16, 128, (heads + 15) & ~15, true, false), p_desc = desc_k(p_smem);
    int pair = 0, done = 0;
    for (int it = 0; it < n; ++it) {
      bool ok = true;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        ok = ok && converged_wait(sh, a.status, &sh.p_full[it & 1][half], it >> 1);
        if (!ok) break;
        const uint32_t more = (*reinterpret_cast<volatile uint32_t*>(&sh.flags[pair]) & kFirst) ^ kFirst;
        const uint32_t v_desc = desc_mn(kv_smem + pair * kChunks * kBlock, kBlock);
#pragma unroll
        for (int t = 0; t < kOut; ++t)
#pragma unroll
          for (int k = 2 * half; k < 2 * half + 2; ++k)
            umma_f16(tmem + t * 64, v_desc + (2 * t * kBlock + 2048 * k) / 16, p_desc + 32 * k / 16, pv, k > 0 ? 1u : more);
        umma_commit_elect(&sh.empty[2 * pair + half]);
        umma_commit_elect(&sh.pv_done[half]);
        ++done;
      }
      if (!ok) break;
      if (++pair == a.pairs) pair = 0;
    }
    if (done > 0) {   // halves done: the last one's commit follows all that was issued
      const int it = (done - 1) >> 1, half = (done - 1) & 1;
      mbar_wait(&sh.empty[2 * (it % a.pairs) + half], (it / a.pairs) & 1, &sh.zero, kWaitNs);
      mbar_wait(&sh.pv_done[half], it & 1, &sh.zero, kWaitNs);
    }
  } else {
    // ---------------- queries ----------------
    int rows_loaded = 0;
    for (int it = 0; it < n;) {
      if (!converged_wait(sh, a.status, &sh.q_empty, rows_loaded ^ 1)) break;
      const char* q = static_cast<const char*>(a.q) + (at.row * a.qs0 + group * kGroup * a.qs1) * 2;
      for (int w = 0; w < 4; ++w) {
        const int hh = 16 * w + lane;
        RowCopy(q_smem, lane < 16 && hh < heads ? q + hh * a.qs1 * 2 : nullptr, a.q, 16 * w, lane)
            .template blocks<0, kChunks>();
      }
      cp_async_wait_all();
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full);
      ++rows_loaded;
      it += at.tiles - at.tile;
      at.tile = at.tiles - 1;
      at.next(a);
    }
    cp_async_wait_all();
  }
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if constexpr (kCluster) {
    // ---- a CTA joins every share-th 64 columns of the cluster's parts ----------------
    auto cluster = cooperative_groups::this_cluster();
    float* const weight = reinterpret_cast<float*>(p_ptr), * const sum = weight + 8 * kGroup;   // [share][64]
    cluster.sync();                            // all parts are there
    for (int i = tid; i < a.share * kGroup; i += kThreads) {
      weight[i] = *cluster.map_shared_rank(&sh.m[i % kGroup], i / kGroup);
      sum[i] = *cluster.map_shared_rank(&sh.l[i % kGroup], i / kGroup);
    }
    __syncthreads();
    if (tid < heads) {
      float m = -CUDART_INF_F, l = 0.0f;
      for (int p = 0; p < a.share; ++p) m = fmaxf(m, weight[p * kGroup + tid]);
      const float ref = m == -CUDART_INF_F ? 0.0f : m;
      for (int p = 0; p < a.share; ++p) l += sum[p * kGroup + tid] * exp2f(weight[p * kGroup + tid] - ref);
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
      for (int p = 0; p < a.share; ++p) weight[p * kGroup + tid] = exp2f(weight[p * kGroup + tid] - ref) * inv;
      if (rank == 0)
        a.lse[x * a.heads + group * kGroup + tid] = l > 0.0f ? (m + log2f(l)) * kLn2 : (l == 0.0f ? -CUDART_INF_F : l);
    }
    __syncthreads();
    T* const out = static_cast<T*>(a.out) + (x * a.heads + group * kGroup) * kLatent;
    for (int block = rank; block < kLatent / 64; block += a.share)
      for (int i = tid; i < heads * 16; i += kThreads) {
        const int h = i >> 4, column = 4 * (i & 15);
        float4* const from = reinterpret_cast<float4*>(base) + (block * kGroup + h) * 16 + (i & 15);
        float4 o = make_float4(0, 0, 0, 0), v[8];
#pragma unroll
        for (int p = 0; p < 8; ++p)
          if (p < a.share) v[p] = *cluster.map_shared_rank(from, p);
#pragma unroll
        for (int p = 0; p < 8; ++p)
          if (p < a.share) {
            const float w = weight[p * kGroup + h];
            o = make_float4(fmaf(v[p].x, w, o.x), fmaf(v[p].y, w, o.y), fmaf(v[p].z, w, o.z), fmaf(v[p].w, w, o.w));
          }
        *reinterpret_cast<uint2*>(out + h * kLatent + 64 * block + column) = make_uint2(pack2<T>(o.x, o.y), pack2<T>(o.z, o.w));
      }
    cluster.sync();                            // read by all before it goes
  }
}

// Joins the parts of the rows that lie in several ranges, in the order of the
// ranges.  Range y's part is its first (slot 0) unless the range begins in an
// earlier row (then its last, slot 1); a range may be empty.  A warp has four heads
// (grid y) and 64 columns at a time, a lane two of them: 32 bytes of a part.
//   kShare = 1: a warp joins all parts -- two or three, many rows; the block's warps
//     have all columns.  Grid x: the row in which range x + 1 begins, if that
//     is the first range to begin inside it;
//   kShare = 16: the block's warps share the parts of 64 columns (grid z) -- a few
//     rows (grid x) spread over all ranges.
// Both kernels: one row of 131072 tokens 111 us with one, 53.5 with sixteen (62 with
// four and a head a warp); 512 tokens 15.4 and 13.1; 12 rows of 2048 30 and 38; 48
// ragged rows 107 and 123.  Around the rule's bound of 512 rows x heads, one and
// sixteen: 192 (12 rows, 16 heads) 28.7 and 28.2; 256 (4 rows of 4096, 64 heads) 38.0
// and 27.2, (of 16384) 47.9 and 40.6; 432 (18 rows of 2048, 24 heads) 25.7 and 29.7; 448
// (7 rows of 8192) 40.6 and 42.3; 512 (8 rows of 2048) 31.3 and 31.2, (of 8192) 42.9 and
// 44.9; 576 (9 rows of 2048) 28.7 and 32.0; 768 (12 rows of 8192) 50.5 and 57.8.
template <typename T, int kLatent, int kShare>
__global__ void __launch_bounds__(kShare == 1 ? kLatent / 2 : 32 * kShare) latent_join_kernel(const __grid_constant__ LatentArgs a) {
  wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = 4 * blockIdx.y;
  int x = blockIdx.x + 1;
  if constexpr (kShare > 1) {
    __shared__ int found;
    if (threadIdx.x == 0) found = kMaxCtas;
    __syncthreads();
    for (int i = threadIdx.x + 1; i < a.ranges; i += 32 * kShare)
      if (a.where[4 * i] == blockIdx.x && begins_inside(record_of(a.where, i))) atomicMin(&found, i);
    __syncthreads();
    x = found;
    if (x == kMaxCtas) return;
  }
  const RangeBegin cut = record_of(a.where, x);
  const int64_t before = begin_of(a.where, x - 1);
  if (!cuts_first(cut, before)) return;                      // the whole block
  const int64_t row = cut.place, end = cut.first + cut.tiles;
  // the part of range x - 1 + i, which may begin in an earlier row if i is 0
  const int64_t base = (static_cast<int64_t>(x - 1) * a.groups + h / kGroup) * 2, step = 2 * a.groups;
  auto part = [&](int i) { return base + i * step + (i == 0 && before < cut.first ? 1 : 0); };
  auto live = [&](int i) { return begin_of(a.where, x + i) > begin_of(a.where, x - 1 + i); };
  auto four = [](const float* p) { return *reinterpret_cast<const float4*>(p); };
  const float* const ml = a.part_ml + h % kGroup;
  float4 m = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
  int parts = 0;
  for (int i = lane; i <= a.ranges - x; i += 32) {
    if (begin_of(a.where, x - 1 + i) >= end) break;
    parts = i + 1;
    if (!live(i)) continue;
    const float4 v = four(ml + part(i) * 2 * kGroup);
    m = make_float4(fmaxf(m.x, v.x), fmaxf(m.y, v.y), fmaxf(m.z, v.z), fmaxf(m.w, v.w));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m.x = fmaxf(m.x, __shfl_xor_sync(0xffffffffu, m.x, o));
    m.y = fmaxf(m.y, __shfl_xor_sync(0xffffffffu, m.y, o));
    m.z = fmaxf(m.z, __shfl_xor_sync(0xffffffffu, m.z, o));
    m.w = fmaxf(m.w, __shfl_xor_sync(0xffffffffu, m.w, o));
    parts = max(parts, __shfl_xor_sync(0xffffffffu, parts, o));
  }
  auto ref = [](float v) { return v == -CUDART_INF_F ? 0.0f : v; };
  const float4 r = make_float4(ref(m.x), ref(m.y), ref(m.z), ref(m.w));
  auto add = [](float4& o, const float4& v, const float4& w) {
    o = make_float4(fmaf(v.x, w.x, o.x), fmaf(v.y, w.y, o.y), fmaf(v.z, w.z, o.z), fmaf(v.w, w.w, o.w));
  };
  auto inverse = [](float l) { return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l); };
  auto lse_of = [](float m_, float l) { return l > 0.0f ? (m_ + log2f(l)) * kLn2 : (l == 0.0f ? -CUDART_INF_F : l); };
  T* const out = static_cast<T*>(a.out) + (row * a.heads + h) * kLatent;
  const int heads = min(4, static_cast<int>(a.heads - h));
  const int block = kShare == 1 ? warp : static_cast<int>(blockIdx.z);
  const float4 none = make_float4(0, 0, 0, 0);
  float4 l = none, o0 = none, o1 = none;       // o0, o1: of columns 64 block + 2 lane, + 1
  const float* const from = a.part + static_cast<int64_t>(h % kGroup) * kLatent + (64 * block + 2 * lane) * 4;
#pragma unroll(kShare == 1 ? 2 : 5)
  for (int i = kShare == 1 ? 0 : warp; i < parts; i += kShare) {
    const bool some = live(i);               // the slot of an empty range holds nothing
    const float* const p = from + part(i) * kGroup * kLatent;
    const float4 v0 = some ? four(p) : none, v1 = some ? four(p + 4) : none;
    const float4 lp = some ? four(ml + part(i) * 2 * kGroup + kGroup) : none;
    const float4 mp = some ? four(ml + part(i) * 2 * kGroup) : r;
    const float4 w = make_float4(exp2f(mp.x - r.x), exp2f(mp.y - r.y), exp2f(mp.z - r.z), exp2f(mp.w - r.w));
    add(l, lp, w);
    add(o0, v0, w);
    add(o1, v1, w);
  }
  if constexpr (kShare > 1) {
    __shared__ float4 sums[kShare][64], ls[kShare];
    sums[warp][2 * lane] = o0;
    sums[warp][2 * lane + 1] = o1;
    if (lane == 0) ls[warp] = l;
    __syncthreads();
    const int column = threadIdx.x & 63, k = threadIdx.x >> 6;   // one head's column a thread
    if (k >= heads) return;
    float o = 0.0f, all = 0.0f;
#pragma unroll
    for (int w = 0; w < kShare; ++w) {
      o += reinterpret_cast<const float*>(&sums[w][column])[k];
      all += reinterpret_cast<const float*>(&ls[w])[k];
    }
    reinterpret_cast<uint16_t*>(out)[k * kLatent + 64 * block + column] = static_cast<uint16_t>(pack2<T>(o * inverse(all), 0.0f));
    if (block == 0 && column == 0) {
      const float top = k == 0 ? m.x : k == 1 ? m.y : k == 2 ? m.z : m.w;
      a.lse[row * a.heads + h + k] = lse_of(top, all);
    }
  } else {
    const float os[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w}, lk[4] = {l.x, l.y, l.z, l.w};
    const float mk[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k >= heads) break;
      const float inv = inverse(lk[k]);
      *reinterpret_cast<uint32_t*>(out + k * kLatent + 64 * block + 2 * lane) = pack2<T>(os[k] * inv, os[4 + k] * inv);
      if (block == 0 && lane == 0) a.lse[row * a.heads + h + k] = lse_of(mk[k], lk[k]);
    }
  }
}

constexpr int64_t kMaxSmem = 232448;

// How the line of tiles is cut: into `ranges` of `base` units of `unit` tiles, the
// first `extra` ones a unit more.  Ranges that cut rows cost their parts' traffic
// and a second launch, about as long as kJoinTiles tiles of a CTA, so rows of equal
// length go whole to the CTAs where the longest range is not longer by more than
// that.  128 rows of 2048 tokens, 64 heads: 81 us whole on 128 CTAs, 92 cut into 148;
// 1024 rows, 128 heads: 929 and 952.
// A few rows go to a cluster of 2, 4 or 8 CTAs each, which needs no second kernel but
// costs about kClusterTiles more than the first, while the second takes a tile's time
// for each row and group of heads up to kJoinMost.  2048 tokens, 64 heads, clusters and
// cut: 4 rows 21.5 and 21.2 us, 8 rows 21.1 and 29.4, 14 rows 23.2 and 29.8, 32 rows 33.5
// and 39.1, 64 rows 48.9 and 57.3; one row of 512 tokens 15.1 and 13.1.  15 clusters of
// 8 were resident at once, 16 were not (42.8 us).
struct Cut {
  int64_t ranges, unit, base, extra, share;
  bool whole;
};
constexpr int64_t kJoinTiles = 6, kClusterTiles = 1, kJoinMost = 5;

Cut cut_for(int64_t rows, int64_t heads, int64_t count, bool equal) {
  const int64_t groups = (heads + kGroup - 1) / kGroup, fit = kMaxCtas / groups, per = (count + kTile - 1) / kTile;
  const int64_t tiles = rows * per, ranges = tiles < fit ? (tiles > 0 ? tiles : 1) : fit;
  Cut c{ranges, 1, tiles / ranges, tiles % ranges, 1, false};
  const int64_t turns = (rows + fit - 1) / fit;
  if (equal && (ranges == 1 || turns * per <= (tiles + ranges - 1) / ranges + kJoinTiles)) {
    c.ranges = (rows + turns - 1) / turns;
    c = Cut{c.ranges, per, rows / c.ranges, rows % c.ranges, 1, true};
  }
  if (equal) {
    int64_t share = 8;
    while (share > 1 && (share > per || rows * groups * share > (share == 8 ? 112 : 128))) share /= 2;
    const int64_t join = rows * groups - 1 < kJoinMost ? rows * groups - 1 : kJoinMost;
    const int64_t each = (per + share - 1) / share, now = c.whole ? turns * per : (tiles + ranges - 1) / ranges + join;
    if (share > 1 && each + kClusterTiles <= now) c = Cut{rows, 1, per, 0, share, true};
  }
  return c;
}

template <typename... KArgs>
void launch_clusters(void (*kernel)(KArgs...), int64_t clusters, int share, size_t smem, cudaStream_t s, KArgs... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * share));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = share;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Launches the kernels of one element type and one pair of widths.
template <typename T, int kLatent, int kRope>
void launch(LatentArgs a, bool join, cudaStream_t s) {
  constexpr int kChunks = (kLatent + kRope) / 64;
  constexpr int64_t kFixed = (kChunks + 1) * kBlock + 1024 + static_cast<int64_t>(sizeof(LatentShared));
  constexpr int kPairs = kFixed + 4 * kChunks * kBlock <= kMaxSmem ? 4 : 2;
  constexpr int64_t kSmem = kFixed + static_cast<int64_t>(kPairs) * kChunks * kBlock;
  static_assert(kPairs <= kMaxPairs && kSmem <= kMaxSmem, "shared memory");
  a.pairs = kPairs;
  static DeviceOnce once;
  once.run([] {
    cudaFuncSetAttribute(latent_kernel<T, kLatent, kRope, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    cudaFuncSetAttribute(latent_kernel<T, kLatent, kRope, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (a.share > 1)
    return launch_clusters(latent_kernel<T, kLatent, kRope, true>, a.rows * a.groups, a.share, kSmem, s, a);
  launch_kernel_prio(LaunchPriority::kDefault, latent_kernel<T, kLatent, kRope, false>,
                     dim3(static_cast<unsigned>(a.ranges * a.groups)), dim3(kThreads), kSmem, s, a);
  if (!join) return;
  const unsigned cuts = static_cast<unsigned>(a.ranges - 1), fours = static_cast<unsigned>((a.heads + 3) / 4);
  if (a.ranges >= 8 * a.rows && a.rows * a.heads <= 512)
    launch_join(latent_join_kernel<T, kLatent, 16>, dim3(static_cast<unsigned>(a.rows), fours, kLatent / 64), dim3(512), s, a);
  else
    launch_join(latent_join_kernel<T, kLatent, 1>, dim3(cuts, fours), dim3(kLatent / 2), s, a);
}

template <typename T>
void launch_widths(const LatentArgs& a, int64_t latent, int64_t rope, bool join, cudaStream_t s) {
  if (latent == 512) rope ? launch<T, 512, 64>(a, join, s) : launch<T, 512, 0>(a, join, s);
  else if (latent == 384) rope ? launch<T, 384, 64>(a, join, s) : launch<T, 384, 0>(a, join, s);
  else if (latent == 256) rope ? launch<T, 256, 64>(a, join, s) : launch<T, 256, 0>(a, join, s);
  else rope ? launch<T, 128, 64>(a, join, s) : launch<T, 128, 0>(a, join, s);
}

}  // namespace
}  // namespace v1x

extern "C" int64_t v1x_latent_attention_workspace(int64_t rows, int64_t heads, int64_t count, int64_t latent,
                                                  int equal) {
  using namespace v1x;
  if (rows <= 0 || heads <= 0 || heads > 1024 || count <= 0 || latent <= 0) return 0;
  const Cut c = cut_for(rows, heads, count, equal != 0);
  if (c.whole || c.ranges == 1) return 0;
  return (c.ranges + 1) * 32 + c.ranges * ((heads + kGroup - 1) / kGroup) * 2 * kGroup * (latent + 2) * 4;
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
  V1X_CHECK_ARG(rows >= 0 && rows < (int64_t(1) << 31) && heads >= 1 && heads <= 1024 && count >= 0 &&
                    count < (int64_t(1) << 36) && slots >= 0,
                "latent_attention: bad geometry");
  V1X_CHECK_ARG(latent >= 128 && latent <= 512 && latent % 128 == 0 && (dim == latent || dim == latent + 64),
                "latent_attention: latent must be 128, 256, 384 or 512 and dim - latent 0 or 64");
  V1X_CHECK_ARG(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pool) |
                  reinterpret_cast<uintptr_t>(out)) & 15) == 0 && qs0 % 8 == 0 && qs1 % 8 == 0 && pool_stride % 8 == 0,
                "latent_attention: q, pool and out rows must be 16-byte aligned");
  V1X_CHECK_ARG(scale_in_range(scale), "latent_attention: the scale must be finite and below 2^127");
  V1X_CHECK_ARG(!lens || (count % 64 == 0 && !req), "latent_attention: a page table takes whole pages and no slot map");
  if (rows == 0) return V1X_OK;
  V1X_CHECK_ARG(q && out && lse && (index || count == 0) && (pool || slots == 0), "latent_attention: NULL argument");
  const int64_t need = v1x_latent_attention_workspace(rows, heads, count, latent, lens == nullptr);
  V1X_CHECK_ARG(workspace_bytes >= need && (workspace || need == 0) && aligned16(workspace),
                "latent_attention: the workspace must be 16-byte aligned and hold %lld bytes", static_cast<long long>(need));
  cudaStream_t s = as_stream(stream);
  const int64_t groups = (heads + kGroup - 1) / kGroup;
  const Cut c = cut_for(rows, heads, count, lens == nullptr);
  LatentArgs a{q,    qs0,  qs1,   pool, slots, pool_stride, req, req_len, index, index_stride, count, lens, rows, heads,
               0, static_cast<int>(groups), static_cast<int>(c.ranges), static_cast<int>(c.share), c.unit, c.base, c.extra, scale * kLog2e, out,
               lse, nullptr, nullptr, nullptr, status};
  if (need) {
    a.where = static_cast<int64_t*>(workspace);
    a.part = reinterpret_cast<float*>(a.where + 4 * (c.ranges + 1));
    a.part_ml = a.part + c.ranges * groups * 2 * kGroup * latent;
  }
  V1X_CHECK_ARG(c.unit * (c.base + 1) < (int64_t(1) << 31), "latent_attention: too many tokens for one call");
  if (dtype == 1) launch_widths<__nv_bfloat16>(a, latent, dim - latent, need > 0, s);
  else launch_widths<__half>(a, latent, dim - latent, need > 0, s);
  return launch_status("v1x_latent_attention");
}
