// Latent attention, expanded form, on the tensor cores: see v1x_prompt_attention
// in v1x.h.
//
// A CTA has 256 queries of one request and head, two tiles of 128, and goes over
// the keys that they see:
//
//   S_t[128 x 64]   = Q_t . [K | K_rope]^T    K = 128 + dr, operands in shared memory
//   O_t[128 x 128] += P_t . V                 P in TMEM, over S_t
//
// One query per TMEM lane: a softmax thread owns a query's row, so maxima, sums and
// the rescale of O need no exchange.  The running maximum that the weights are taken
// against moves only when a tile exceeds it by more than 2^8, so that O is rescaled
// a few times a row at most; sums stay in 32 bits, the weights are rounded once, to
// the inputs' type, for the second product.
//
// Keys go in steps of 64, two score buffers a tile: while a tile's softmax is at one
// step, the tensor cores form the output of the step before and, once that has read
// its weights, the scores of the step after over them.  Per 128 keys with dr = 64 the
// tensor cores need 3328 cycles (a 128 x 64 x 16 MMA takes 48, bound by shared
// memory; 128-key steps would need 2560, but with one buffer a tile the chain S,
// softmax, O, S took 4900), the special-function units 2048.
// 96 KB of queries leave room for three 32 KB slots that keys and values take in
// turn and two 16 KB slots of rotary keys.  Whole tiles come by TMA (a slot that is
// free is full 1100 cycles later; by cp.async, whose 48 instructions a warp took 1500
// to issue, it was 3200, more than the ring hides: 8192 tokens, 32 heads 606 us instead
// of 696, five prompts of 106-510 queries after 2.4-4 K keys 151 instead of 174); a
// request's last tile, and tensors whose heads share memory, come by 16-byte cp.async,
// which writes zeros past the last key (a neighbour's values never enter a product) and
// takes any strides.
// 8192 tokens, 32 heads: 595 us, 1155 TFLOP/s, 4280 cycles per 128 keys; both tiles'
// softmax is busy 80% of them.  An eighth to a half of the exponentials by polynomial on
// the FMA pipe made it 634 to 660 us: the warps are bound by issue, not by exp2.
//
// Warp roles (384 threads, one CTA per SM): 0-3 and 4-7 softmax and epilogue of the
// two tiles, 8 and 9 issue their MMAs (8 owns the TMEM), 10 and 11 bring the queries,
// then keys and values.  Later queries see more keys: the grid begins with the last
// ones, all heads of a tile side by side.
// Waits are bounded (2 s, then V1X_STATUS_TIMEOUT).
#include <type_traits>

#include "attention.cuh"
#include "ring.cuh"
#include "sm100.cuh"

namespace v1x {
namespace {

using namespace attn;
using namespace sm100;

constexpr int kRows = 128;                // queries of a tile, keys of a tile
constexpr int kStep = 64;                 // keys of a step: half of a key tile
constexpr int kBlock = kRows * 128;       // bytes of 64 elements of a tile's rows
constexpr int kThreads = 384;
constexpr int kSlots = 3, kRopeSlots = 2;
constexpr uint32_t kOutCol = 256;         // TMEM: S_0, S_1 in columns 0-255 (P over them), O_0, O_1
constexpr float kLazy = 8.0f;             // log2 of the growth that the weights may show before a rescale
constexpr uint64_t kWaitNs = 2000000000ull;

struct PromptArgs {
  const void *q, *k, *k_rope, *v;
  int64_t qs0, qs1, ks0, ks1, krs0, vs0, vs1;
  const int32_t *offsets, *kv_offsets;
  int64_t requests, tokens, keys, heads;
  float scale_log2;      // of |scale|
  int negative;          // the scale's sign goes into the product
  void* out;
  float* lse;
  int32_t* status;
  int tma;               // the tensor maps are there
};

struct PromptShared {
  uint64_t full[kSlots], empty[kSlots], rope_empty[kRopeSlots];   // keys: with their rotary part
  uint64_t q_full, s_full[2][2], p_full[2][2], pv_done[2][2], o_done[2];   // [tile][step & 1]
  int64_t request;
  uint32_t tmem;
  int abort, zero;
};

__device__ __forceinline__ void give_up(PromptShared& sh, int32_t* status) {
  *reinterpret_cast<volatile int*>(&sh.abort) = 1;
  if (status) atomicExch(status, V1X_STATUS_TIMEOUT);
}

__device__ __forceinline__ bool converged_wait(PromptShared& sh, int32_t* status, uint64_t* bar, int phase) {
  bool ok = __all_sync(0xffffffffu, mbar_test(bar, phase & 1));   // most phases are complete when asked for
  if (!ok) {
    ok = __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, &sh.abort, kWaitNs));
    if (!ok) give_up(sh, status);
  }
  tc_fence_after();
  return ok;
}

__device__ __forceinline__ int64_t clamped(const int32_t* offsets, int64_t i, int64_t most) {
  return min(static_cast<int64_t>(max(offsets[i], 0)), most);
}

// `kCount` rows of kBlocks x 64 elements from row `row` on, into the swizzled operand
// layout (row R of block b at b * kBlock + R * 128, its 16-byte pieces permuted by
// R & 7); rows from `rows` on become zeros.  A warp moves four rows' 128-byte pieces
// at a time.
template <int kBlocks, int kCount>
__device__ __forceinline__ void copy_tile(uint32_t dst, int R0, const char* src, int64_t stride, int64_t row, int64_t rows,
                                          const void* any, int lane) {
  const int r = lane >> 3, piece = lane & 7;
  const char* p = src + (row + r) * stride + piece * 16;
#pragma unroll 4
  for (int i = 0; i < kCount; i += 4, p += 4 * stride) {
    const int R = R0 + i + r;
    const bool live = row + i + r < rows;
    const uint32_t to = dst + R * 128 + ((piece ^ (R & 7)) << 4);
    const char* const from = live ? p : static_cast<const char*>(any);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) cp_async16(to + b * kBlock, from + (live ? b * 128 : 0), live ? 16 : 0);
  }
}

template <typename T, bool kRope>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                  const __grid_constant__ CUtensorMap rope_map, const __grid_constant__ PromptArgs a) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kQBlocks = kRope ? 3 : 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_smem = smem_u32(base), kv_smem = q_smem + 6 * kBlock, rope_smem = kv_smem + kSlots * 2 * kBlock;
  PromptShared& sh = *reinterpret_cast<PromptShared*>(base + (6 + 2 * kSlots + kRopeSlots) * kBlock);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t h = blockIdx.x, unit = static_cast<int64_t>(gridDim.y) - 1 - blockIdx.y;

  // ---- the unit's request: the last one with offsets[r] / 256 + r <= unit; a request
  // has at least as many units as tiles of 256 queries ------------------------------
  if (warp == 0) {
    int64_t lo = 0, n = a.requests;
    while (n > 1) {
      const int64_t step = (n + 31) / 32, c = lo + lane * step;
      const bool at = lane * step < n && clamped(a.offsets, c, a.tokens) / 256 + c <= unit;
      const int64_t k = max(__popc(__ballot_sync(0xffffffffu, at)) - 1, 0);
      lo += k * step;
      n = min(step, n - k * step);
    }
    if (lane == 0) sh.request = lo;
  }
  __syncthreads();
  const int64_t r = sh.request;
  const int64_t q0 = clamped(a.offsets, r, a.tokens), q1 = max(clamped(a.offsets, r + 1, a.tokens), q0);
  const int64_t k0 = clamped(a.kv_offsets, r, a.keys), k1 = max(clamped(a.kv_offsets, r + 1, a.keys), k0);
  const int64_t nq = q1 - q0, nk = k1 - k0, tile = unit - (q0 / 256 + r);
  const int64_t i0 = tile * 256;                           // the first query of the request in this CTA
  if (tile < 0 || i0 >= nq) return;
  // steps of 64 keys that a tile of queries sees: up to its last query's limit
  auto steps_seen = [&](int t) {
    const int64_t last = min(i0 + 128 * (t + 1), nq) - 1;
    if (last < i0 + 128 * t) return 0;
    const int64_t limit = min(last + 1 + nk - nq, nk);
    return limit > 0 ? static_cast<int>((limit + kStep - 1) / kStep) : 0;
  };
  const int n0 = steps_seen(0), n1 = steps_seen(1), n = (max(n0, n1) + 1) / 2;   // n: key tiles

  if (tid == 0) {
    sh.abort = 0;
    sh.zero = 0;
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh.full[i], 2);
      mbar_init(&sh.empty[i], 2);
    }
    for (int i = 0; i < kRopeSlots; ++i) mbar_init(&sh.rope_empty[i], 2);
    for (int i = 0; i < 2; ++i) {
      for (int x = 0; x < 2; ++x) {
        mbar_init(&sh.s_full[i][x], 1);
        mbar_init(&sh.p_full[i][x], 4);
        mbar_init(&sh.pv_done[i][x], 1);
      }
      mbar_init(&sh.o_done[i], 1);
    }
    mbar_init(&sh.q_full, 2);
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp < 8) {
    // ---------------- softmax, rescale, epilogue ----------------
    const int t = warp >> 2;
    const int64_t i = i0 + 128 * t + 32 * (warp & 3) + lane;     // the thread's query of the request
    const int64_t limit = i < nq ? max(min(i + 1 + nk - nq, nk), static_cast<int64_t>(0)) : 0;
    const uint32_t quarter = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + quarter + 128 * t, o_addr = tmem + quarter + kOutCol + 128 * t;
    const int mine = t ? n1 : n0;
    const float c = a.scale_log2;
    constexpr float kLift = lift<T>(kLazy);
    float m = -CUDART_INF_F, l = 0.0f;       // m: of the unscaled scores
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase) {
      if (ok && !mbar_wait(bar, phase & 1, &sh.abort, kWaitNs)) {
        give_up(sh, a.status);
        ok = false;
      }
    };
    for (int j = 0; j < mine; ++j) {
      const int x = j & 1;
      wait(&sh.s_full[t][x], j >> 1);
      if (__any_sync(0xffffffffu, !ok)) break;
      tc_fence_after();
      uint32_t s[2][32];
#pragma unroll
      for (int b = 0; b < 2; ++b) tmem_ld32(s_addr + kStep * x + 32 * b, s[b]);
      tmem_ld_wait();
      if (__any_sync(0xffffffffu, limit < static_cast<int64_t>(j + 1) * kStep)) {
        const int left = static_cast<int>(max(min(limit - static_cast<int64_t>(j) * kStep, static_cast<int64_t>(kStep)),
                                              static_cast<int64_t>(0)));
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * b + e >= left) s[b][e] = 0xFF800000u;   // -inf
      }
      float top[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        top[b] = __uint_as_float(s[b >> 1][16 * (b & 1)]);
#pragma unroll
        for (int e = 1; e < 16; ++e) top[b] = fmaxf(top[b], __uint_as_float(s[b >> 1][16 * (b & 1) + e]));
      }
      const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (j == 0) {
        m = most;
      } else {
        const bool grows = m == -CUDART_INF_F ? most > m : (most - m) * c > kLazy;
        if (__any_sync(0xffffffffu, grows)) {
          const float f = grows ? (m == -CUDART_INF_F ? 0.0f : exp2_fast((m - most) * c)) : 1.0f;
          if (grows) m = most;
          l *= f;
          wait(&sh.pv_done[t][x ^ 1], (j - 1) >> 1);   // O holds all that was given to it
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int b = 0; b < 4; ++b) {
            uint32_t o[32];
            tmem_ld32(o_addr + 32 * b, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(o_addr + 32 * b, o);
          }
        }
      }
      const float shift = m == -CUDART_INF_F ? 0.0f : kLift - m * c;
      const f32x2 c2 = two(c, c), shift2 = two(shift, shift);
      f32x2 sum[2] = {0, 0};
      uint32_t w[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const f32x2 y = fma2(two(__uint_as_float(s[e >> 4][(2 * e) & 31]), __uint_as_float(s[e >> 4][(2 * e + 1) & 31])), c2, shift2);
        const float2 v = both(y);
        const float u0 = exp2_fast(v.x), u1 = exp2_fast(v.y);
        sum[e & 1] = add2(sum[e & 1], two(u0, u1));
        w[e] = pack2<T>(u0, u1);
      }
      tmem_st32(s_addr + kStep * x, w);
      const float2 sums = both(add2(sum[0], sum[1]));
      l += sums.x + sums.y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[t][x]);
    }
    if (mine > 0 && ok && !mbar_wait(&sh.o_done[t], 0, &sh.abort, kWaitNs)) give_up(sh, a.status);
    __syncwarp();
    tc_fence_after();
    const bool empty = l == 0.0f;            // no key
    const float inv = 1.0f / l;
    T* const out = static_cast<T*>(a.out) + ((q0 + i) * a.heads + h) * 128;
#pragma unroll 1
    for (int b = 0; b < 4; ++b) {
      uint32_t o[32];
      if (mine > 0) {
        tmem_ld32(o_addr + 32 * b, o);
        tmem_ld_wait();
      }
      if (i < nq) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            w[x] = empty ? 0u
                         : pack2<T>(__uint_as_float(o[e + 2 * x]) * inv, __uint_as_float(o[e + 2 * x + 1]) * inv);
          *reinterpret_cast<uint4*>(out + 32 * b + e) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (i < nq)
      a.lse[(q0 + i) * a.heads + h] = empty ? -CUDART_INF_F : (m * c - kLift + log2f(l)) * kLn2;
    tc_fence_before();
  } else if (warp < 10) {
    // ---------------- MMA issuers, one per tile ----------------
    const int t = warp - 8, mine = t ? n1 : n0;
    const uint32_t qk = idesc_16bit_f32(kBf16, 128, kStep, false, false) | (a.negative ? 1u << 13 : 0u);
    const uint32_t pv = idesc_16bit_f32(kBf16, 128, 128, false, true);
    const uint32_t s_tmem = tmem + 128 * t, o_tmem = tmem + kOutCol + 128 * t;
    const uint32_t qd = desc_k(q_smem + t * kQBlocks * kBlock);
    bool ok = true, issued = false;
    auto wait = [&](uint64_t* bar, int phase) { return ok = ok && converged_wait(sh, a.status, bar, phase); };
    // key tile j in slot 2 j of the ring (mod kSlots), its values in slot 2 j + 1
    auto scores = [&](int j) {                   // of step j
      const int u = j & ~1, slot = u % kSlots, rope = (j >> 1) % kRopeSlots, x = j & 1;
      if (x == 0) wait(&sh.full[slot], u / kSlots);
      if (j >= 2) wait(&sh.pv_done[t][x], (j - 2) >> 1);   // the weights are read: S may be written over them
      if (!ok) return;
      const uint32_t kd = desc_k(kv_smem + slot * 2 * kBlock + x * (kBlock / 2));
      const uint32_t rd = desc_k(rope_smem + rope * kBlock + x * (kBlock / 2)), d = s_tmem + kStep * x;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(d, qd + (b * kBlock + 32 * k) / 16, kd + (b * kBlock + 32 * k) / 16, qk, b + k > 0 ? 1u : 0u);
      if (kRope) {
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16(d, qd + (2 * kBlock + 32 * k) / 16, rd + 32 * k / 16, qk, 1u);
      }
      umma_commit_elect(&sh.s_full[t][x]);
      if (x == 1 || j == mine - 1) {
        umma_commit_elect(&sh.empty[slot]);
        if (kRope) umma_commit_elect(&sh.rope_empty[rope]);
      }
      issued = true;
    };
    auto output = [&](int j) {
      const int u = j | 1, slot = u % kSlots, x = j & 1;
      if (x == 0) wait(&sh.full[slot], u / kSlots);
      wait(&sh.p_full[t][x], j >> 1);
      if (!ok) return;
      const uint32_t vd = desc_mn(kv_smem + slot * 2 * kBlock + x * (kBlock / 2), kBlock), p = s_tmem + kStep * x;
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_f16_ta(o_tmem, p + 8 * k, vd + 2048 * k / 16, pv, j + k > 0 ? 1u : 0u);
      umma_commit_elect(&sh.pv_done[t][x]);
      if (x == 1 || j == mine - 1) umma_commit_elect(&sh.empty[slot]);
    };
    if (mine > 0) wait(&sh.q_full, 0);
    if (mine > 0 && ok) scores(0);
    if (mine > 1 && ok) scores(1);
    for (int j = 0; j < mine && ok; ++j) {
      output(j);
      if (j + 2 < mine && ok) scores(j + 2);
    }
    for (int u = 2 * ((mine + 1) / 2); u < 2 * n && ok; ++u) {   // the other tile's alone
      wait(&sh.full[u % kSlots], u / kSlots);
      if (lane == 0) {
        mbar_arrive(&sh.empty[u % kSlots]);
        if (kRope && !(u & 1)) mbar_arrive(&sh.rope_empty[(u >> 1) % kRopeSlots]);
      }
      __syncwarp();
    }
    // everything that was issued retires before the CTA ends
    if (issued) {
      umma_commit_elect(&sh.o_done[t]);
      mbar_wait(&sh.o_done[t], 0, &sh.zero, kWaitNs);
    }
  } else if (n > 0) {
    // ---------------- queries, keys, values: 64 rows of a tile per warp ----------------
    const int half = warp - 10;
    const char* const q = static_cast<const char*>(a.q) + (q0 * a.qs0 + h * a.qs1) * 2;
    const char* const k = static_cast<const char*>(a.k) + (k0 * a.ks0 + h * a.ks1) * 2;
    const char* const v = static_cast<const char*>(a.v) + (k0 * a.vs0 + h * a.vs1) * 2;
    const char* const kr = static_cast<const char*>(a.k_rope) + k0 * a.krs0 * 2;
    for (int t = 0; t < 2; ++t)
      copy_tile<kQBlocks, 64>(q_smem + t * kQBlocks * kBlock, 64 * half, q, a.qs0 * 2, i0 + 128 * t + 64 * half, nq, a.q, lane);
    cp_async_commit();
    uint64_t* pending = &sh.q_full;              // a load whose arrival has not been reported
    auto report = [&] {
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(pending);
    };
    int slot = 0, turn = 0;
    LastBoxes<kSlots> boxes;
    for (int u = 0; u < 2 * n; ++u) {
      const int j = u >> 1, rope = j % kRopeSlots;
      const bool keys = (u & 1) == 0;
      if (pending && !__all_sync(0xffffffffu, mbar_test(&sh.empty[slot], (turn & 1) ^ 1))) {
        cp_async_wait<0>();
        report();
        pending = nullptr;
      }
      if (!converged_wait(sh, a.status, &sh.empty[slot], turn ^ 1)) break;
      if (kRope && keys && !converged_wait(sh, a.status, &sh.rope_empty[rope], (j / kRopeSlots) ^ 1)) break;
      if (a.tma && static_cast<int64_t>(j + 1) * kRows <= nk) {   // whole tiles come by TMA
        if (pending) {
          cp_async_wait<0>();
          report();
          pending = nullptr;
        }
        if (lane == 0) {
          uint64_t* const bar = &sh.full[slot];
          uint8_t* const to = base + (6 + slot * 2) * kBlock;
          const int y = static_cast<int>(h), z = static_cast<int>(k0) + j * kRows;
          if (half == 1) {
            mbar_arrive(bar);
          } else {
            mbar_arrive_expect_tx(bar, kRope && keys ? 3 * kBlock : 2 * kBlock);
            tma_load_3d(to, keys ? &k_map : &v_map, bar, 0, y, z);
            tma_load_3d(to + kBlock, keys ? &k_map : &v_map, bar, 64, y, z);
            if (kRope && keys) tma_load_2d(base + (6 + 2 * kSlots + rope) * kBlock, &rope_map, bar, 0, z);
          }
        }
        __syncwarp();
        boxes.box(slot, turn);
        if (++slot == kSlots) {
          slot = 0;
          ++turn;
        }
        continue;
      }
      const int64_t row = static_cast<int64_t>(j) * kRows + 64 * half;
      copy_tile<2, 64>(kv_smem + slot * 2 * kBlock, 64 * half, keys ? k : v, (keys ? a.ks0 : a.vs0) * 2, row, nk, a.q, lane);
      if (kRope && keys) copy_tile<1, 64>(rope_smem + rope * kBlock, 64 * half, kr, a.krs0 * 2, row, nk, a.q, lane);
      cp_async_commit();
      if (pending) {
        cp_async_wait<1>();
        report();
      }
      pending = &sh.full[slot];
      boxes.copy(slot);
      if (++slot == kSlots) {
        slot = 0;
        ++turn;
      }
    }
    cp_async_wait_all();
    if (pending) report();
    // boxes that are under way land before the CTA ends, whoever gives up, now or later
    if (half == 0)
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
        if (boxes.turns[i] >= 0) mbar_wait(&sh.full[i], boxes.turns[i] & 1, &sh.zero, kWaitNs);
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

constexpr int kSmem = 1024 + (6 + 2 * kSlots + kRopeSlots) * kBlock + static_cast<int>(sizeof(PromptShared));
static_assert(kSmem <= 232448, "shared memory");

// Rows [keys][heads] of 128 elements as boxes of 64 elements x 128 keys of one head
// (heads = 0: rows [keys] of 64 elements), 128-byte swizzle.  False where the driver
// takes no such map.
bool encode_rows(CUtensorMap* map, bool bf16, const void* p, int64_t keys, int64_t heads, int64_t key_stride,
                 int64_t head_stride) {
  const PFN_cuTensorMapEncodeTiled_v12000 fn = map_encoder();
  if (!fn) return false;
  const cuuint32_t steps[3] = {1, 1, 1};
  const CUtensorMapDataType type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r;
  if (heads) {
    const cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(keys)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_stride * 2), static_cast<cuuint64_t>(key_stride * 2)};
    const cuuint32_t box[3] = {64, 1, kRows};
    r = fn(map, type, 3, const_cast<void*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    const cuuint64_t dims[2] = {64, static_cast<cuuint64_t>(keys)}, strides[1] = {static_cast<cuuint64_t>(key_stride * 2)};
    const cuuint32_t box[2] = {64, kRows};
    r = fn(map, type, 2, const_cast<void*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  return r == CUDA_SUCCESS;
}

template <typename T, bool kRope>
void launch(PromptArgs a, cudaStream_t s) {
  // Maps for the whole tiles.  Strides of 0 (a dimension of one, or a broadcast one)
  // take no map: a dimension of one gets any stride, broadcast tensors go without.
  CUtensorMap k_map = {}, v_map = {}, rope_map = {};
  auto stride = [](int64_t given, int64_t count) { return given == 0 && count == 1 ? int64_t(128) : given; };
  const int64_t ks0 = stride(a.ks0, a.keys), ks1 = stride(a.ks1, a.heads), vs0 = stride(a.vs0, a.keys), vs1 = stride(a.vs1, a.heads);
  const int64_t krs0 = stride(a.krs0, a.keys);
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  a.tma = a.keys >= kRows && ks0 > 0 && ks1 > 0 && vs0 > 0 && vs1 > 0 && (!kRope || krs0 > 0) &&
          encode_rows(&k_map, kBf16, a.k, a.keys, a.heads, ks0, ks1) &&
          encode_rows(&v_map, kBf16, a.v, a.keys, a.heads, vs0, vs1) &&
          (!kRope || encode_rows(&rope_map, kBf16, a.k_rope, a.keys, 0, krs0, 0));
  static DeviceOnce once;
  once.run([] { cudaFuncSetAttribute(prompt_kernel<T, kRope>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem); });
  launch_kernel_prio(LaunchPriority::kDefault, prompt_kernel<T, kRope>,
                     dim3(static_cast<unsigned>(a.heads), static_cast<unsigned>(a.tokens / 256 + a.requests)),
                     dim3(kThreads), kSmem, s, k_map, v_map, rope_map, a);
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
  V1X_CHECK_ARG(tokens / 256 + requests <= 65535, "prompt_attention: at most 65535 tiles of 256 queries and requests");
  V1X_CHECK_ARG((dr == 0 && !k_rope) || (dr == 64 && (k_rope || keys == 0)), "prompt_attention: dr must be 0 without k_rope, 64 with it");
  V1X_CHECK_ARG(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_rope) |
                  reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                    (qs0 | qs1 | ks0 | ks1 | krs0 | vs0 | vs1) % 8 == 0,
                "prompt_attention: q, k, k_rope, v and out rows must be 16-byte aligned");
  V1X_CHECK_ARG(scale_in_range(scale), "prompt_attention: the scale must be finite and below 2^127");
  if (tokens == 0 || requests == 0) return V1X_OK;
  V1X_CHECK_ARG(q && out && lse && offsets && kv_offsets && ((k && v) || keys == 0), "prompt_attention: NULL argument");
  // a masked score, -inf, has to stay -inf under the scale, so that is never 0
  float magnitude = (scale < 0 ? -scale : scale) * kLog2e;
  if (magnitude < 1e-30f) magnitude = 1e-30f;
  const PromptArgs a{q,    k,     k_rope, v, qs0, qs1, ks0, ks1, krs0, vs0, vs1, offsets, kv_offsets, requests, tokens,
                     keys, heads, magnitude, scale < 0 ? 1 : 0, out, lse, status, 0};
  cudaStream_t s = as_stream(stream);
  if (dtype == 1) dr ? launch<__nv_bfloat16, true>(a, s) : launch<__nv_bfloat16, false>(a, s);
  else dr ? launch<__half, true>(a, s) : launch<__half, false>(a, s);
  return launch_status("v1x_prompt_attention");
}
