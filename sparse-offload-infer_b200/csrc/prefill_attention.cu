// Causal attention of packed prompts (grouped heads, sequences of different lengths) on the tcgen05 tensor cores.
//
//   o_i = sum_{j <= i + Lk - Lq} exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),   s_ij = q_i . k_j / sqrt(hd)
//
// One pass over the keys with the running maximum and sum of the softmax; scores and outputs never leave the SM.  Two
// products of 4 hd flop per pair together and one exponential per pair: at hd = 128 a 128 x 128 tile costs the tensor
// core 2 x 512 cycles and the exponential unit (16 per cycle and SM) 1024, so both bound it and have to overlap; at hd = 64
// the exponentials alone do.
//
// A CTA holds two tiles of 128 query rows that share a kv head (stages 0 and 1: two heads of the group, or two row tiles; a
// tile's rows are tokens x heads, or tokens of one head).  Their scores S (fp32, 128 columns each) and outputs O (fp32, hd
// columns each) lie in the tensor memory; the probabilities P (fp16) overwrite the scores they come from and feed the second
// product from there.
//   warps 0-3, 4-7: the softmax of stage 0 / 1, one thread per row (two threads per row: 716 against 685 us in the case
//           below; the first half's probabilities with the old maximum, beside the search for the new one: 570 against 553).
//           P is handed over in two halves, so that the second product starts after the first 64 keys, and one in four
//           pairs of exponentials is computed on the fp32 pipe.  These warps take most of the CTA's registers.
//   warp 8: loads Q, then K and V tiles of 128 keys through a ring of four slots (TMA, 128-byte swizzle).  A last V tile
//           with fewer keys has its other rows cleared: what lies behind a sequence may be anything, and 0 * NaN counts.
//   warp 9: issues the products in the order  S0(j) P1V(j-1) S1(j) P0V(j) -- while the tensor core works on one
//           stage, the other stage's softmax runs.  Products that one thread issues run in order, so S(j+1) overwrites P(j)
//           only after P(j) V has read it; a commit covers everything issued before it, so scores that have arrived say
//           that the O before them is complete.
// The running maximum moves only when a row exceeds it by 2^8 (O is rescaled in place then, by the softmax warps); the
// probabilities carry a factor 2^7 and are rounded once to fp16, which keeps 11 bits down to 2^-21 of the largest; the sum
// is fp32 over the unrounded ones and the factor cancels.
// A masked score is selected away, but a non-finite V in a masked place of a shared tile would still reach the product:
// rows whose scores or result are not finite are computed again one by one over exactly the keys they see.
//
// The grid holds one CTA per pair of tiles and kv head, an upper bound from the token counts (row bounds are read on the
// device).  Where the GPU holds two, four or eight times as many CTAs and the contexts are long, a cluster of as many
// shares a pair's keys and joins its sums through distributed shared memory: 32 / 8 heads, 512 tokens over 8000 107 -> 71 us
// and over 30000 382 -> 229, 128 over 32000 383 -> 115, four times 5 over 16000 182 -> 57, 64 over 1000 20.0 -> 19.8.
//
// Measured (8192 tokens, 40 / 8 heads, hd 128): products issued from a single lane's branch 832 us, maxima over eight chains
// and packed pairs 685, products issued by a convergent warp 600, registers / halves / fp32 pipe / coalesced output 555 in
// short runs = 1238 TFLOP/s, 0.77 of the measured burst rate of a library product; called back to back, at the power limit, 640
// to 652 = 1054 to 1075 TFLOP/s, 0.77 of its sustained rate.  7 unequal prompts (3828 tokens, 16 / 8 heads): 29 us, the longest
// one's 12 steps of 1.6 us plus 6 us of start and end and a second round of CTAs.  One in eight / three in eight / half of the
// pairs on the fp32 pipe: 31.6 / 31.7 / 32.3 us against 31.2 there.  hd 64, two chunks of 512 and 1000 rows over 4012 and 3047
// keys, 32 / 4 heads: 68 us, 192 CTAs in two rounds; P beside S in the tensor memory, so that scores run ahead, measured the
// same (the two warps of a scheduler spend their exponentials' phases together).
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace soinfer {
namespace {

constexpr int kTile = 128;            // query rows and keys per tile
constexpr int kSlots = 4;             // K / V tiles in flight
constexpr int kThreads = 384;         // 8 softmax warps, loads, products, two without work (register shares go by 4 warps)
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;  // 256 x 216 + 128 x 72 = 384 x 168, what the launch gets
constexpr uint64_t kTimeoutNs = 1000000000ull;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;          // the maximum follows when exceeded by 2^8
constexpr unsigned kFmaPairs = 0x22;  // which of 8 pairs of exponentials go to the fp32 pipe (see above)
constexpr float kLift = 7.f;          // factor 2^7 on the probabilities
constexpr int64_t kSplitKeys = 512;   // keys that a CTA of a cluster has at least

__device__ int g_prefill_error;

struct Shared {
  uint64_t q_full[2], kv_full[kSlots], kv_empty[kSlots], v_landed, s_full[2], p_full[2], p_half[2], o_full[2], drained;
  uint32_t tmem;
  int abort;
};

// Waits for a phase with a time limit; a wait that runs out tells the others and the host, and every later wait is short.
__device__ __forceinline__ bool wait(Shared& sh, uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (*reinterpret_cast<volatile int*>(&sh.abort)) return false;
    if (globaltimer_ns() - t0 > kTimeoutNs) {
      *reinterpret_cast<volatile int*>(&sh.abort) = 1;
      atomicOr(&g_prefill_error, kErrCopyTimeout);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Largest value, NaN if any is NaN.
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of both halves on the fp32 pipe: x = n + f with n the nearest integer (added to 1.5 * 2^23, whose low bits then hold
// it) and |f| <= 1/2, 2^f by a polynomial of degree 4 (least largest relative error, 2.7e-6, by exchange), 2^n added to the
// exponent.  Below 2^-126: 0 or a subnormal.
__device__ __forceinline__ void ex2_pair(uint64_t x2, float& a, float& b) {
  constexpr float kRound = 12582912.f;
  float x, y;
  unpack2(x2, x, y);
  x2 = pack2(fmaxf(x, -126.f), fmaxf(y, -126.f));
  const uint64_t t2 = add2(x2, pack2(kRound, kRound));
  const uint64_t f2 = fma2(add2(t2, pack2(-kRound, -kRound)), pack2(-1.f, -1.f), x2);
  uint64_t p2 = fma2(pack2(0.00957010220736f, 0.00957010220736f), f2, pack2(0.0559178590775f, 0.0559178590775f));
  p2 = fma2(p2, f2, pack2(0.240247443318f, 0.240247443318f));
  p2 = fma2(p2, f2, pack2(0.693121790886f, 0.693121790886f));
  p2 = fma2(p2, f2, pack2(0.999999284744f, 0.999999284744f));
  float t, u, p, q;
  unpack2(t2, t, u);
  unpack2(p2, p, q);
  a = __int_as_float((__float_as_int(t) << 23) + __float_as_int(p));
  b = __int_as_float((__float_as_int(u) << 23) + __float_as_int(q));
}

// A query tile's heads of a kv head, its rows of the sequence (128 / heads), the kv head's groups of that many heads; inv:
// 2^16 / heads, rounded up (a tile row's number times that, shifted back, is the quotient).  ranks: CTAs that share the keys
// of a pair of tiles.
struct Layout {
  int heads, rows, groups, inv, ranks;
};

// A CTA's work: two query tiles of sequence rows q0.., keys k0.., kv head kvh.
struct Work {
  int q0, lq, k0, lk, kvh;
  int row[2], head[2], tiles[2];  // first row in the sequence, first query head, key tiles (0: nothing to do)
};

// The pair of query tiles with this index (warp-wide; false: none).  Tile t of a sequence and kv head is head
// group t % groups, rows t / groups * rows ..  A sequence's pairs run from the last to the first, and of up to 32 sequences
// those with more keys come first (more: as they are given), so that short work fills the end of the launch.
template <bool kPacked>
__device__ __forceinline__ bool find_work(const PrefillParams& P, const Layout& H, int index, int lane, Work& w) {
  const int rows_tile = kPacked ? H.rows : kTile;
  auto tiles_of = [&](int n) { return (n + rows_tile - 1) / rows_tile * H.groups; };
  w.kvh = index % P.nkv;
  int want = index / P.nkv;
  for (int base = 0; base < P.seqs; base += 32) {
    const int i = base + lane;
    int q0 = 0, lq = 0, k0 = 0, lk = 0;
    if (i < P.seqs) {
      const int a = P.cu_q[i], e = P.cu_q[i + 1], c = P.cu_k[i], f = P.cu_k[i + 1];
      q0 = max(a, 0);
      lq = max(min(e, P.tokens_q) - q0, 0);
      k0 = max(c, 0);
      lk = max(min(f, P.tokens_k) - k0, 0);
    }
    const int pairs = (tiles_of(lq) + 1) / 2;
    int before = 0;
    if (P.seqs <= 32) {
      for (int o = 0; o < P.seqs; ++o) {
        const int keys = __shfl_sync(0xffffffffu, lk, o), n = __shfl_sync(0xffffffffu, pairs, o);
        if (keys > lk || (keys == lk && o < lane)) before += n;
      }
    } else {
      before = pairs;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
      }
      before -= pairs;
    }
    const unsigned owns = __ballot_sync(0xffffffffu, want >= before && want < before + pairs);
    if (owns) {
      const int src = __ffs(owns) - 1;
      w.q0 = __shfl_sync(0xffffffffu, q0, src);
      w.lq = __shfl_sync(0xffffffffu, lq, src);
      w.k0 = __shfl_sync(0xffffffffu, k0, src);
      w.lk = __shfl_sync(0xffffffffu, lk, src);
      const int last = __shfl_sync(0xffffffffu, pairs - 1 - (want - before), src);  // the pair, from the sequence's start
      const int tiles = tiles_of(w.lq);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int t = 2 * last + s;
        const int q = t / H.groups;
        w.row[s] = q * rows_tile;
        w.head[s] = (w.kvh * H.groups + t - q * H.groups) * (kPacked ? H.heads : 1);
        const int rows = w.lq - w.row[s] < rows_tile ? w.lq - w.row[s] : rows_tile;
        const int keys = max(w.row[s] + rows + w.lk - w.lq, 0);  // what the tile's last row sees
        w.tiles[s] = t < tiles ? (keys + kTile - 1) / kTile : -1;
      }
      return true;
    }
    want -= __reduce_add_sync(0xffffffffu, pairs);
  }
  return false;
}

// One row over the n keys it sees, by a whole warp (rows whose tile result is not finite).
template <int HD>
__device__ __noinline__ void redo_row(const PrefillParams& P, const half* q, int k0, int n, int kvh, half* out,
                                      float scale_log2, int lane) {
  constexpr int E = HD / 32;
  float qf[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qf[e] = __half2float(q[lane * E + e]) * scale_log2;
    acc[e] = 0.f;
  }
  for (int j = 0; j < n; ++j) {
    const half* k = P.k + (int64_t)(k0 + j) * P.k_token + kvh * P.k_head + lane * E;
    const half* v = P.v + (int64_t)(k0 + j) * P.v_token + kvh * P.v_head + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qf[e], __half2float(k[e]), s);
    s = warp_sum(s);
    const float top = fmaxf(m, s), f = m == top ? 1.f : exp2f(m - top), p = s == -INFINITY ? 0.f : exp2f(s - top);
    m = top;
    l = fmaf(l, f, p);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(p, __half2float(v[e]), acc[e] * f);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane * E + e] = __float2half_rn(acc[e] / l);
}

// kPacked: a tile holds several heads.  kSplit: the CTAs of a cluster share the keys.
template <int HD, bool kPacked, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map, const PrefillParams P, const Layout H, const float scale_log2) {
  constexpr int kBox = kTile * 128;              // bytes of a TMA box: 128 rows of 64 fp16
  constexpr int kBoxes = HD / 64;
  constexpr int kTileBytes = kBoxes * kBox;
  constexpr uint32_t kO = 2 * kTile;             // tensor memory columns: S0, S1, O0, O1
  constexpr uint32_t kColumns = 512;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;                           // two tiles
  uint8_t* s_kv = smem + 2 * kTileBytes;         // kSlots tiles
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  pdl_launch_dependents();
  pdl_wait();
  Work w;
  const int rank = kSplit ? blockIdx.x % H.ranks : 0;
  if (!find_work<kPacked>(P, H, kSplit ? blockIdx.x / H.ranks : blockIdx.x, lane, w)) return;  // alike for the whole cluster
  int first = 0;                                 // this CTA's first key tile
  if (kSplit) {
    const int each = (max(max(w.tiles[0], w.tiles[1]), 0) + H.ranks - 1) / H.ranks;
    first = rank * each;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (w.tiles[s] >= 0) w.tiles[s] = min(max(w.tiles[s] - first, 0), each);
  }
  const int steps = w.tiles[0] > w.tiles[1] ? w.tiles[0] : w.tiles[1];

  if (warp == 9) {
    tc::alloc(&sh.tmem, kColumns);
  } else if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh.q_full[s], 1);
      mbar_init(&sh.s_full[s], 1);
      mbar_init(&sh.p_full[s], 4);
      mbar_init(&sh.p_half[s], 4);
      mbar_init(&sh.o_full[s], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
    }
    mbar_init(&sh.v_landed, 1);
    mbar_init(&sh.drained, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------------------------------------------------------- softmax
    const int s = warp >> 2, r = threadIdx.x & (kTile - 1);
    const int tiles = w.tiles[s], token = kPacked ? r * H.inv >> 16 : r, row = w.row[s] + token;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t S = lanes + s * kTile, O = lanes + kO + s * HD;
    const bool valid = row < w.lq && (!kPacked || token < H.rows);
    const bool idle = !__any_sync(0xffffffffu, valid);  // whatever its P is stays in its rows
    // keys this row sees; a row behind the last one is worked on as that one (with none it would mask every tile) and dropped
    const int limit = max(min(row, w.lq - 1) + 1 + w.lk - w.lq - first * kTile, 0);  // (from this CTA's first key)
    // worst: the largest score of all, NaN if one is NaN (the polynomial loses them)
    float m = -INFINITY, l = 0.f, worst = -INFINITY;
    bool ok = true;
    for (int j = 0; j < tiles && ok; ++j) {
      ok = __all_sync(0xffffffffu, wait(sh, &sh.s_full[s], j & 1));
      if (!ok) break;
      if (idle) {
        if (lane == 0) {
          mbar_arrive(&sh.p_half[s]);
          mbar_arrive(&sh.p_full[s]);
        }
        continue;
      }
      tc::fence_after();
      uint32_t x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tc::ld32(x[c], S + 32 * c);
      tc::wait_ld();
      const int left = limit - j * kTile;
      if (__any_sync(0xffffffffu, left < kTile)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (__any_sync(0xffffffffu, left < 32 * c + 32)) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * c + i >= left) x[c][i] = 0xff800000u;  // -inf
          }
      }
      float tops[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) tops[i] = max2(__uint_as_float(x[0][2 * i]), __uint_as_float(x[0][2 * i + 1]));
#pragma unroll
      for (int i = 16; i < 128; i += 2)
        tops[(i >> 1) & 7] =
            max3(tops[(i >> 1) & 7], __uint_as_float(x[i >> 5][i & 31]), __uint_as_float(x[i >> 5][(i & 31) + 1]));
      float top = max2(max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[4]), max3(tops[5], tops[6], tops[7]));
      top *= scale_log2;
      worst = max2(worst, top);
      const bool move = top > m + kLazy;  // also the first finite maximum
      if (__any_sync(0xffffffffu, move)) {
        const float f = move ? ex2(m - top) : 1.f;
        if (move) m = top;
        l *= f;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t o[16];
            tc::ld16(o, O + 16 * c);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tc::st16(O + 16 * c, o);
          }
        }
      }
      const float shift = m == -INFINITY ? 0.f : kLift - m;
      const uint64_t scale2 = pack2(scale_log2, scale_log2), shift2 = pack2(shift, shift);
      uint64_t sum2[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float a, b;
          const uint64_t y2 = fma2(pack2(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1])), scale2, shift2);
          if (kFmaPairs >> (i & 7) & 1) {
            ex2_pair(y2, a, b);
          } else {
            unpack2(y2, a, b);
            a = ex2(a);
            b = ex2(b);
          }
          sum2[i & 1] = add2(sum2[i & 1], pack2(a, b));
          p[i] = h2_as_u32(__floats2half2_rn(a, b));
        }
        tc::st16(S + 16 * c, p);
        if (c == 1) {  // the first 64 keys' probabilities are there
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_half[s]);
        }
      }
      float sa, sb;
      unpack2(add2(sum2[0], sum2[1]), sa, sb);
      l += sa + sb;
      tc::wait_st();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[s]);
    }
    if constexpr (kSplit) {
      // The CTAs' sums, maxima and sums of weights (NaN: a score that is not finite), where the tiles were, which no product
      // and no load needs any more; every CTA then finishes its share of the 256 rows.
      float4* sums = reinterpret_cast<float4*>(smem);
      float2* stats = reinterpret_cast<float2*>(smem + 2 * kTile * HD * 4);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (w.tiles[x] > 0) ok = ok && __all_sync(0xffffffffu, wait(sh, &sh.o_full[x], 0));
      tc::fence_after();
      if (ok && tiles >= 0 && !idle) {
        if (tiles > 0) {
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tc::ld32(o, O + 32 * c);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              sums[(s * kTile + r) * (HD / 4) + ((8 * c + i) ^ (r & 7))] =
                  make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                              __uint_as_float(o[4 * i + 3]));
          }
        }
        stats[s * kTile + r] = make_float2(m, worst <= 3.4e38f ? l : __int_as_float(0x7fffffff));
      }
      __syncwarp();
      cluster_sync();
      // kRows rows at a time, two CTAs' sums at a time: their loads wait for one another only there
      constexpr int kLanes = HD / 4, kStep = 2 * kTile / kLanes, kRows = HD / 32;  // threads of a row, rows of all threads
      const int c = threadIdx.x % kLanes;
      for (int i0 = threadIdx.x / kLanes; ok && i0 < 2 * kTile / H.ranks; i0 += kStep * kRows) {
        float M[kRows], L[kRows], v[kRows][4];
#pragma unroll
        for (int u = 0; u < kRows; ++u) M[u] = -INFINITY, L[u] = v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.f;
        int at[kRows], heads_at[kRows];          // the rows' places in the sequence (-1: no such row) and heads
        bool any = false;
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          const int x = (i0 + u * kStep) * H.ranks + rank, xr = x % kTile, xt = kPacked ? xr * H.inv >> 16 : xr;
          const bool second = x >= kTile;
          at[u] = (second ? w.row[1] : w.row[0]) + xt;
          heads_at[u] = (second ? w.head[1] : w.head[0]) + (kPacked ? xr - xt * H.heads : 0);
          if ((second ? w.tiles[1] : w.tiles[0]) < 0 || at[u] >= w.lq || (kPacked && xt >= H.rows)) at[u] = -1;
          any = any || at[u] >= 0;
        }
        if (!__any_sync(0xffffffffu, any)) continue;
        for (int k = 0; k < H.ranks; k += 2) {
          float2 ml[kRows][2];
          float4 o[kRows][2];
#pragma unroll
          for (int u = 0; u < kRows; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int x = (i0 + u * kStep) * H.ranks + rank;
              ml[u][e] = cluster_read(stats + x, k + e);
              o[u][e] = cluster_read(sums + x * (HD / 4) + (c ^ (x & 7)), k + e);
            }
#pragma unroll
          for (int u = 0; u < kRows; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 t = ml[u][e];
              const float top = fmaxf(M[u], t.x), f = M[u] == top ? 1.f : ex2(M[u] - top);
              const float g = t.x == -INFINITY ? 0.f : ex2(t.x - top);
              const float4 y = t.x == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : o[u][e];  // (else never written)
              M[u] = top;
              L[u] = fmaf(g, t.y, L[u] * f);
              v[u][0] = fmaf(g, y.x, v[u][0] * f), v[u][1] = fmaf(g, y.y, v[u][1] * f);
              v[u][2] = fmaf(g, y.z, v[u][2] * f), v[u][3] = fmaf(g, y.w, v[u][3] * f);
            }
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          bool bad = false;
          if (at[u] >= 0) {
            const float inv = 1.f / L[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[u][e] *= inv;
              bad = bad || !(fabsf(v[u][e]) <= 3.4e38f);
            }
            if (at[u] + 1 + w.lk - w.lq <= 0) v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.f, bad = false;
            *reinterpret_cast<uint2*>(P.out + ((int64_t)(w.q0 + at[u]) * P.nq + heads_at[u]) * HD + 4 * c) =
                make_uint2(h2_as_u32(__floats2half2_rn(v[u][0], v[u][1])), h2_as_u32(__floats2half2_rn(v[u][2], v[u][3])));
          }
          unsigned again = __ballot_sync(0xffffffffu, bad);
          while (again) {
            const int src = (__ffs(again) - 1) / kLanes * kLanes;  // the first lane of the row
            again &= ~(kLanes == 32 ? 0xffffffffu : 0xffffu << src);
            const int rr = __shfl_sync(0xffffffffu, at[u], src), h = __shfl_sync(0xffffffffu, heads_at[u], src);
            __syncwarp();
            redo_row<HD>(P, P.q + (int64_t)(w.q0 + rr) * P.q_token + h * P.q_head, w.k0, rr + 1 + w.lk - w.lq, w.kvh,
                         P.out + ((int64_t)(w.q0 + rr) * P.nq + h) * HD, scale_log2, lane);
          }
        }
      }
      __syncwarp();
      cluster_sync();  // nobody leaves while its sums are read
    } else if (tiles >= 0 && ok && !idle) {  // the row's result
      constexpr int kPieces = HD / 8;
      uint4* stage = reinterpret_cast<uint4*>(s_q + s * kTileBytes + (warp & 3) * (32 * HD * 2));
      bool good = limit == 0 || fabsf(worst) <= 3.4e38f;
      if (tiles > 0) {
        ok = __all_sync(0xffffffffu, wait(sh, &sh.o_full[s], 0));
        tc::fence_after();
      }
      if (ok) {
        const float inv = limit > 0 ? 1.f / l : 0.f;
        const bool zero = __any_sync(0xffffffffu, limit == 0);
        uint64_t zeros = 0;                      // 0 * value: NaN where one is not finite
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          if (tiles > 0) {
            tc::ld32(o, O + 32 * c);
            tc::wait_ld();
          }
          uint4 v[4];
          uint32_t* h = reinterpret_cast<uint32_t*>(v);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t y = mul2(pack2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), both(inv));
            float a, b;
            zeros = fma2(y, 0, zeros);
            unpack2(y, a, b);
            h[i] = h2_as_u32(__floats2half2_rn(a, b));
          }
          if (zero && limit == 0)
#pragma unroll
            for (int i = 0; i < 16; ++i) h[i] = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) stage[lane * kPieces + ((4 * c + i) ^ (lane & 7))] = v[i];
        }
        float a, b;
        unpack2(zeros, a, b);
        good = limit == 0 || (good && a + b == 0.f);
        __syncwarp();
        const unsigned write = __ballot_sync(0xffffffffu, valid);
        uint4* out = reinterpret_cast<uint4*>(P.out + ((int64_t)(w.q0 + w.row[s]) * P.nq + w.head[s]) * HD);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int rr = (32 * i + lane) / kPieces, c = lane % kPieces, tr = (r & ~31) + rr;
          // the row's place behind the tile's first
          const int to = kPacked ? (tr * H.inv >> 16) * (P.nq - H.heads) + tr : tr * P.nq;
          if (write >> rr & 1) out[(int64_t)to * kPieces + c] = stage[rr * kPieces + (c ^ (rr & 7))];
        }
        unsigned again = __ballot_sync(0xffffffffu, valid && !good);
        while (again) {
          const int src = __ffs(again) - 1, rr = __shfl_sync(0xffffffffu, row, src);
          const int h = w.head[s] + (kPacked ? (r & ~31) + src - (rr - w.row[s]) * H.heads : 0);
          again &= again - 1;
          __syncwarp();
          redo_row<HD>(P, P.q + (int64_t)(w.q0 + rr) * P.q_token + h * P.q_head, w.k0, rr + 1 + w.lk - w.lq, w.kvh,
                       P.out + ((int64_t)(w.q0 + rr) * P.nq + h) * HD, scale_log2, lane);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
    // ---------------------------------------------------------------- loads
    // Key tile j is ring entry 2 j, value tile j entry 2 j + 1.
    int issued = 0;
    bool ok = true;
    if (lane == 0) {
      tc::prefetch_map(&q_map);
      tc::prefetch_map(&k_map);
      tc::prefetch_map(&v_map);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (w.tiles[s] > 0) {
          mbar_arrive_expect_tx(&sh.q_full[s], kBoxes * (kPacked ? H.rows * H.heads : kTile) * 128);
          for (int x = 0; x < kBoxes; ++x)
            tc::tma_load_3d(s_q + s * kTileBytes + x * kBox, &q_map, 64 * x, w.head[s], w.q0 + w.row[s], &sh.q_full[s]);
        }
    }
    for (int e = 0; e < 2 * steps && ok; ++e) {
      const int slot = e % kSlots, j = e >> 1;
      if (e >= kSlots) ok = wait(sh, &sh.kv_empty[slot], ((e / kSlots) - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint8_t* dst = s_kv + slot * kTileBytes;
      const int rows = w.lk - (first + j) * kTile;  // valid rows of the tile
      const bool clear = (e & 1) && rows < kTile;
      uint64_t* bar = clear ? &sh.v_landed : &sh.kv_full[slot];
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, kTileBytes);
        for (int x = 0; x < kBoxes; ++x)
          tc::tma_load_3d(dst + x * kBox, e & 1 ? &v_map : &k_map, 64 * x, w.kvh, w.k0 + (first + j) * kTile, bar);
      }
      ++issued;
      if (clear) {                               // at most once: the sequence's last tile
        ok = __all_sync(0xffffffffu, wait(sh, &sh.v_landed, 0));
        if (!ok) break;
        for (int x = 0; x < kBoxes; ++x)
          for (int i = rows * 8 + lane; i < kTile * 8; i += 32)
            reinterpret_cast<uint4*>(dst + x * kBox)[i] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.kv_full[slot]);
      }
    }
    if (!ok) {  // a wait ran out: let the copies in flight land before the CTA ends
      const uint64_t t0 = globaltimer_ns();
      for (int s = 0; s < 2; ++s)
        while (w.tiles[s] > 0 && !mbar_try_wait(&sh.q_full[s], 0) && globaltimer_ns() - t0 < kTimeoutNs) {
        }
      for (int e = issued < kSlots ? 0 : issued - kSlots; e < issued; ++e)
        while (!mbar_try_wait(&sh.kv_full[e % kSlots], (e / kSlots) & 1) && globaltimer_ns() - t0 < kTimeoutNs) {
        }
    }
    } else if (warp == 9) {
    // ---------------------------------------------------------------- products
    constexpr uint32_t kIdescS = tc::instr_desc(kTile, kTile, false), kIdescO = tc::instr_desc(kTile, HD, true);
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const int n0 = __shfl_sync(0xffffffffu, w.tiles[0], 0), n1 = __shfl_sync(0xffffffffu, w.tiles[1], 0);
    const int n = n0 > n1 ? n0 : n1;
    const uint32_t at_q = __shfl_sync(0xffffffffu, smem_u32(s_q), 0), at_kv = at_q + 2 * kTileBytes;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, wait(sh, bar, parity)); };
    bool ok = true;
    if (n0 > 0) ok = wait_all(&sh.q_full[0], 0);
    if (n1 > 0) ok = ok && wait_all(&sh.q_full[1], 0);
    auto scores = [&](int s, int j) {          // S_s = Q_s K_j^T
      const uint64_t a = tc::smem_desc(at_q + s * kTileBytes, 16, 1024);
      const uint64_t b = tc::smem_desc(at_kv + (2 * j % kSlots) * kTileBytes, 16, 1024);
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const uint32_t at = ((k / 4) * kBox + (k % 4) * 32) >> 4;
        tc::mma_ss(base + s * kTile, a + at, b + at, kIdescS, k > 0);
      }
      tc::commit(&sh.s_full[s]);
    };
    auto outputs = [&](int s, int j, int last) {  // O_s (+)= P_s V_j
      const uint64_t b = tc::smem_desc(at_kv + ((2 * j + 1) % kSlots) * kTileBytes, kBox, 1024);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        ok = ok && wait_all(f ? &sh.p_full[s] : &sh.p_half[s], j & 1);
        if (!ok) return;
        tc::fence_after();
#pragma unroll
        for (int k = 4 * f; k < 4 * f + 4; ++k)
          tc::mma_ts(base + kO + s * HD, base + s * kTile + k * 8, b + k * (2048 >> 4), kIdescO, j > 0 || k > 0);
      }
      if (j == last) tc::commit(&sh.o_full[s]);
    };
    // entry e may be overwritten; for the last ones nobody waits, and no arrival is left for after the CTA's end
    auto release = [&](int e) {
      if (e + kSlots < 2 * n) tc::commit(&sh.kv_empty[e % kSlots]);
    };
    for (int j = 0; j <= n && ok; ++j) {
      if (j < n) ok = wait_all(&sh.kv_full[2 * j % kSlots], (2 * j / kSlots) & 1);
      if (!ok) break;
      tc::fence_after();
      if (j < n0) scores(0, j);
      if (j > 0) {
        if (j - 1 < n1) {
          ok = wait_all(&sh.kv_full[(2 * j - 1) % kSlots], ((2 * j - 1) / kSlots) & 1);
          if (ok) outputs(1, j - 1, n1 - 1);
          if (!ok) break;
        }
        release(2 * j - 1);
      }
      if (j == n) break;
      if (j < n1) scores(1, j);
      release(2 * j);
      if (j < n0) {
        ok = wait_all(&sh.kv_full[(2 * j + 1) % kSlots], ((2 * j + 1) / kSlots) & 1);
        if (ok) outputs(0, j, n0 - 1);
      }
    }
    if (!ok) {  // let the products in flight end before the tensor memory is given back
      tc::commit(&sh.drained);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&sh.drained, 0) && globaltimer_ns() - t0 < kTimeoutNs) {
      }
    }
    __syncwarp();
    }
    if (kSplit) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 9) {
    tc::fence_after();
    tc::dealloc(tmem, kColumns);
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Map of rows [tokens, heads, hd] with boxes of 64 values x box_heads x 128 / box_heads tokens.
cudaError_t make_map(CUtensorMap* map, const half* data, int64_t tokens, int64_t heads, int hd, int64_t token_stride,
                     int64_t head_stride, int box_heads) {
  const EncodeTiled encode = encoder();
  if (!encode) return cudaErrorNotSupported;
  // a dimension of one entry may have any stride
  if (heads == 1) head_stride = hd;
  if (tokens == 1) token_stride = heads * hd;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)(kTile / box_heads)}, ones[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<half*>(data), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Query heads per tile: all of a kv head's unless that takes more tiles for sequences of the average length (5 heads leave 3
// of 128 rows empty), which also lets a tile's rows see keys that differ less.  32 / 8 heads, one against all heads a tile:
// 128 sequences of one token over 2001 450 against 210 us, 256 of 20 tokens 340 against 165, 64 of 200 135.6 against 126.8,
// 100 of 10 to 910 580 against 535, 16 of 1000 196.9 against 197.0; 64 / 8 heads, 20 of 450 194 against 176.
Layout layout_of(const PrefillParams& P) {
  const int64_t rep = P.nq / P.nkv, length = (P.tokens_q + P.seqs - 1) / P.seqs;
  int heads = 1;
  if (rep <= kTile) {
    const int64_t rows = kTile / rep;
    if ((length + rows - 1) / rows <= (length + kTile - 1) / kTile * rep) heads = (int)rep;
  }
  return {heads, kTile / heads, (int)rep / heads, (65536 + heads - 1) / heads, 1};
}

// CTAs that share the keys of a pair of tiles: as many as the GPU holds at once, with at least kSplitKeys keys each on the
// average (one long context among many short sequences is not seen: 5 tokens over 16000 beside 40 of one token 180 us).  A
// cluster lies within one group of SMs, so that fewer than 148 / 4 and 148 / 8 clusters fit at one CTA per SM.  One token each
// of 8 / 1 heads over 16000: clusters of eight 34.2 us for 15 pairs and 63.6 for 16, of four 55 for 16 and 57 for 33 but 107
// for 34, of two 99 for 34.
int ranks_for(int64_t ctas, int64_t keys) {
  constexpr int64_t kFit[3] = {74, 33, 15};  // clusters of 2, 4, 8
  int ranks = 1;
  for (int i = 0; i < 3 && ctas <= kFit[i] && keys >= kSplitKeys * ranks * 2; ++i) ranks *= 2;
  return ranks;
}

template <int HD>
cudaError_t prefill_hd(const PrefillParams& P, cudaStream_t stream) {
  CUtensorMap q, k, v;
  Layout H = layout_of(P);
  cudaError_t e = make_map(&q, P.q, P.tokens_q, P.nq, HD, P.q_token, P.q_head, H.heads);
  if (e != cudaSuccess) return e;
  k = v = q;  // no keys: never read
  if (P.tokens_k > 0) {
    if ((e = make_map(&k, P.k, P.tokens_k, P.nkv, HD, P.k_token, P.k_head, 1)) != cudaSuccess) return e;
    if ((e = make_map(&v, P.v, P.tokens_k, P.nkv, HD, P.v_token, P.v_head, 1)) != cudaSuccess) return e;
  }
  // the most that sum over sequences of ceil(n t / 2), t = ceil(lq / rows), may be with seqs of them not empty: t is at most
  // (lq + rows - 1) / rows, and a half is rounded up only where n is odd
  const int64_t n = H.groups, seqs = P.seqs < P.tokens_q ? P.seqs : P.tokens_q;
  const int64_t tiles = (P.tokens_q + seqs * (H.rows - 1)) / H.rows;
  const int64_t pairs = (n * tiles + n % 2 * seqs) / 2;
  if (pairs * P.nkv > 0x7fffffff) return cudaErrorInvalidValue;
  const float scale_log2 = (1.0f / sqrtf((float)HD)) * kLog2e;
  const int smem = (2 + kSlots) * kTile * HD * 2 + 1024;
  H.ranks = ranks_for(pairs * P.nkv, P.tokens_k / P.seqs);
  auto launch = [&](auto packed, auto split) {
    constexpr auto kernel = prefill_kernel<HD, decltype(packed)::value, decltype(split)::value>;
    const cudaError_t error = ensure_smem_attr<kernel>(smem);
    if (error != cudaSuccess) return error;
    return launch_ex(kernel, dim3((unsigned)(pairs * P.nkv * H.ranks)), dim3(kThreads), (size_t)smem, stream,
                     dim3((unsigned)H.ranks), true, q, k, v, P, H, scale_log2);
  };
  using Yes = std::true_type;
  using No = std::false_type;
  if (H.heads > 1) return H.ranks > 1 ? launch(Yes{}, Yes{}) : launch(Yes{}, No{});
  return H.ranks > 1 ? launch(No{}, Yes{}) : launch(No{}, No{});
}

}  // namespace

cudaError_t launch_prefill_attention(const PrefillParams& P, cudaStream_t stream) {
  return P.hd == 128 ? prefill_hd<128>(P, stream) : prefill_hd<64>(P, stream);
}

cudaError_t read_and_clear_prefill_error(int* out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_prefill_error, sizeof(int));
  if (e != cudaSuccess) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_prefill_error, &zero, sizeof(int));
}

}  // namespace soinfer
