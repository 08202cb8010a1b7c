// Decode attention over a paged cache: one query per sequence, grouped heads, fp16 or 4-bit rows.
//
//   s_p = (q . k_p) / sqrt(hd) for p < len,   o = sum_p exp(s_p - m) v_p / sum_p exp(s_p - m)
//
// Memory bounds it: every cached row is read once and serves the query heads of its group.  Both products run on the
// matrix instruction with the cached rows as its 16-row operand and up to 8 query heads as its 8 columns, so the work a
// 4-bit value costs is its unpacking, not its dot products:
//   scores:  16 positions x 16 values times 16 values x 8 heads.  One LOP3 turns a nibble into an fp16 number: half of the
//            codes enter as 72 + c and the product starts at -72 sum q over their values, the others are freed of their
//            1032 first (the integer and the fp16 pipe share the work).  The group's scale multiplies the fp32 result --
//            no code is rounded.
//   output:  16 values x 16 positions times 16 positions x 8 heads.  4-bit rows: the codes are exact fp16 numbers and a
//            position's scale multiplies its probability.  The running maximum is taken over score + exponent of the
//            scale, so that the product p * scale lies in (0, 2^8] whatever the scales are; it is lifted by 2^7 and rounded
//            once to fp16 (11 bits, down to 2^-21 of the largest).  fp16 rows: the same with the scale 1.
// The softmax statistics and both sums are fp32.
//
// Work split.  A sequence's kv head with up to 8 of its query heads is a unit.
//   Few units (cluster_units) over tables that name few positions (kClusterMost): a unit is one cluster of eight CTAs, each
//   an eighth of the positions; they join through distributed shared memory.  One launch, no workspace: 777 4-bit positions of
//   8 kv heads 5.2 us against 7.3 by ranges; 8 unequal sequences of up to 4096 fp16 positions, 4 kv heads, 12.5 against 14.0.
//   What a table can name decides, not the lengths, which the host does not know: short sequences under wide tables go by ranges.
//   Beyond, a cluster's idle CTAs and the eight-fold start cost more than they bring (64 unequal sequences of up to 4000 4-bit
//   positions 91 us against 56, 256 of 500 252 against 58; one of 8000 fp16 positions 14.3 against 11.3, 4-bit 11.0 against
//   11.3).
//   Else the positions of all units form one line that is cut into equal ranges, one per CTA that the GPU holds, computed on
//   the device from the lengths (no host read; a captured launch serves any lengths).  A CTA works through the pieces of
//   sequences in its range; a sequence inside one range is finished in place, the pieces (m, l, acc) of the others go to the
//   workspace, whose size follows from the GPU, and a second kernel joins them in order.  (Chunks of equal length, as many as
//   CTAs where that fits: 20 sequences of 50000 316 us against 219, 30 of 12000 141 against 93; two long ones 61.8 against
//   61.4.)
// A CTA has four warps, each with every fourth tile of the CTA's positions; they are joined in shared memory.
//
// Feeding: each warp has its own ring of tiles in shared memory, filled by 16-byte asynchronous copies, so loads run ahead and
// the registers hold only what is being multiplied.  The pieces' places are exchanged within 128 bytes by row, since rows
// that lie end to end put the lanes of a load on the same banks (fp16, 8 sequences of up to 4096, 4 kv heads: bulk copies
// without exchange 15.5 us, a bulk copy per padded row 18.2, this 12.3, all at an earlier state of the kernel).
//
// Measured (GPU time): 4 bits, two sequences of 131072 and 100003, 40 / 8 heads: 62 us for 255 MB = 4.1 TB/s (0.63 of the
// measured copy rate), bound by issuing 303 instructions per 16 positions and kv head (integer pipe 47%, fp16 / fp32 pipe
// 25%, tensor pipe 25% busy); register tiles without a ring 96 us, 32-position tiles 81.  One sequence of 777
// positions: 5.2 us in one launch (an earlier form with a second kernel that joins: 8.7).
#include <algorithm>

#include "launch.cuh"
#include "paged_cache.cuh"

namespace soinfer {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kCluster = 8;
// The most units that go to clusters: two CTAs per SM, or as many clusters as the GPU holds at once where those are fewer.  (A
// cluster lies within one group of SMs: 33 with fp16 rows of 128, whose rings let an SM hold two; 48 and more with the
// others.  fp16, hd 128, 34 units of 500 / 2000 / 4000 positions: 9.0 / 13.8 / 19.5 us against 8.9 / 11.3 / 15.3 by ranges,
// 33 units 7.2 / 10.4 / 14.9 against 8.9 / 11.2 / 15.3.)
constexpr int cluster_units(bool q4, int64_t hd) { return !q4 && hd == 128 ? 33 : 148 * 2 / kCluster; }
constexpr int kCols = 8;          // query heads per CTA
constexpr int kMostLen = 1 << 30;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;      // the running maximum follows when exceeded by 2^8 (it moves in a few tiles, not in half)
constexpr float kLift = 7.f;      // factor 2^7 on the probabilities (it cancels)
constexpr float kNoScore = -3.0e38f;  // the maximum of positions without a finite score: below every score, above no position

// Positions a warp takes at a time, tiles in its ring, CTAs that an SM holds (shared memory and registers), the split's limit
// and units (see above and below).
template <bool Q4>
struct Plan {
  static constexpr int kTile = Q4 ? 64 : 16;
  static constexpr int kStages = Q4 ? 2 : 3;
  static constexpr int kPerSm = Q4 ? 3 : 2;
  static constexpr int kCtas = 148 * kPerSm;
  static constexpr int kMinChunk = kTile * kWarps;
  static constexpr int kStart = Q4 ? 1 : 2;
  static constexpr int64_t kClusterMost = Q4 ? 8192 : 4096;
};

// d = a b + c.
__device__ __forceinline__ void mma_from(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1, float c0, float c1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

// Transpose of an 8 x 8 block of 16-bit values spread over the warp (lane i: row i / 4, columns 2 (i % 4), + 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Positions of sequence b: its length, at most what its table can name (the length limit keeps positions in 32 bits).
__device__ __forceinline__ int seq_len(const PagedDecodeParams& P, int b) {
  const int64_t table = (int64_t)P.cache.table_cols << P.cache.page_shift;
  const int most = table < kMostLen ? (int)table : kMostLen, n = ld_i32(P.lens + b);
  return n < 0 ? 0 : n > most ? most : n;
}

// The split by ranges: a sequence counts as its positions in units of kMinChunk and kStart units more, what beginning it
// costs (without them 67 against 62 us in the file comment's case: the CTAs with two pieces were the last).  All sequences of
// a head group follow one another, and the head groups; CTA i takes the units [i per, (i + 1) per) of that line, per =
// ceil(all / CTAs).  Its range falls into pieces, one per sequence that it touches; a sequence that lies in one range is
// finished by its CTA, the others' pieces go to the workspace: slot 2 i for a piece that begins the range, 2 i + 1 for one
// that ends it.
struct Piece {
  int b, group, begin, end;        // sequence (-1: none), head group, positions
  int slot;                        // workspace slot (-1: the whole sequence)
  int later;                       // units that later CTAs do (-1: not the sequence's first piece)
};
struct Range {
  long long left, per;             // units still to do, units of a range
  int b, group, inside;            // where they begin: sequence, head group, units of the sequence before
};
// A split sequence, noted by the CTA that begins it: its pieces are slot first and slots 2 (first / 2 + 1) .. 2 last.
struct Split {
  int b, group, first, last;       // b -1: none
};
struct Workspace {
  Split* splits;                   // per head group and sequence where those are fewer than the CTAs, else per CTA
  float* pieces;                   // [2 CTAs][heads][hd + 2]: sums, maximum, sum of weights
};
template <bool Q4>
__device__ __forceinline__ Workspace workspace(const PagedDecodeParams& P) {
  return {reinterpret_cast<Split*>(P.ws), P.ws + Plan<Q4>::kCtas * (sizeof(Split) / sizeof(float))};
}

template <bool Q4>
__device__ __forceinline__ int units_of(int len) {
  return (len + Plan<Q4>::kMinChunk - 1) / Plan<Q4>::kMinChunk + Plan<Q4>::kStart;
}

// The next piece of the range (one thread).
template <bool Q4>
__device__ __forceinline__ void next_piece(const PagedDecodeParams& P, Range& R, bool first, Piece& out) {
  if (R.left <= 0) {
    out.b = -1;
    return;
  }
  constexpr int kMin = Plan<Q4>::kMinChunk, kStart = Plan<Q4>::kStart;
  const int n = seq_len(P, R.b), rest = units_of<Q4>(n) - R.inside;
  const int take = rest < R.left ? rest : (int)R.left;
  const int from = max(R.inside - kStart, 0) * kMin, to = max(R.inside + take - kStart, 0) * kMin;
  out.b = R.b;
  out.group = R.group;
  out.begin = from;
  out.end = n < to ? n : to;
  out.slot = R.inside == 0 && take == rest ? -1 : 2 * (int)blockIdx.x + (first ? 0 : 1);
  out.later = R.inside == 0 ? rest - take : -1;
  R.left -= take;
  R.inside = 0;
  if (++R.b == P.seqs) R.b = 0, ++R.group;
}

// Notes whether the sequence that this piece begins is split (one thread).
template <bool Q4>
__device__ __forceinline__ void note_split(const PagedDecodeParams& P, int groups_all, const Piece& piece, long long per) {
  constexpr int kCtas = Plan<Q4>::kCtas;
  const bool by_sequence = (long long)P.seqs * groups_all <= kCtas;
  if (piece.later < 0 || (piece.later == 0 && !by_sequence)) return;
  Split* at = workspace<Q4>(P).splits + (by_sequence ? piece.group * P.seqs + piece.b : (int)blockIdx.x);
  if (piece.later == 0)
    at->b = -1;
  else
    *at = {piece.b, piece.group, piece.slot, (int)(blockIdx.x + (piece.later + per - 1) / per)};
}

// This CTA's range and its first two pieces (one warp).
template <bool Q4>
__device__ __forceinline__ void first_piece(const PagedDecodeParams& P, int groups_all, int lane, Range& R, Piece* out) {
  constexpr int kCtas = Plan<Q4>::kCtas;
  long long total = 0;
  for (int base = 0; base < P.seqs; base += 32)
    total += __reduce_add_sync(0xffffffffu, base + lane < P.seqs ? (unsigned)units_of<Q4>(seq_len(P, base + lane)) : 0u);
  const long long all = total * groups_all, per = (all + kCtas - 1) / kCtas, at = per * blockIdx.x;
  long long want = at, group = 0;
  if (at < all) {
    group = all >> 31 ? at / total : (unsigned)at / (unsigned)total;
    want -= group * total;
  }
  int b = 0, inside = 0;
  for (int base = 0; at < all && base < P.seqs; base += 32) {
    const int mine = base + lane < P.seqs ? units_of<Q4>(seq_len(P, base + lane)) : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned owns = __ballot_sync(0xffffffffu, want < sum);
    if (owns) {
      const int src = __ffs(owns) - 1;
      b = base + src;
      inside = (int)want - __shfl_sync(0xffffffffu, sum - mine, src);
      break;
    }
    want -= __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane != 0) return;
  R.per = per;
  R.left = at + per < all ? per : at < all ? all - at : 0;
  R.b = b;
  R.group = (int)group;
  R.inside = inside;
  next_piece<Q4>(P, R, true, out[0]);
  next_piece<Q4>(P, R, false, out[1]);
  if ((long long)P.seqs * groups_all > kCtas) workspace<Q4>(P).splits[blockIdx.x].b = -1;
}

// A tile in shared memory: key codes (rows), their scales, value codes (rows), their scales; where it holds 16-byte piece c
// of a key row p and of a value row m (4 bits: a pair of positions): what a load of a quarter warp takes lies on all banks.
template <int HD, bool Q4>
struct Tile {
  static constexpr int kTile = Plan<Q4>::kTile;
  static constexpr int kKeyRow = Q4 ? HD / 2 : 2 * HD, kValueRow = Q4 ? HD : 2 * HD;
  static constexpr int kScales = kTile * kKeyRow;  // offset of the key scales
  static constexpr int kValues = kScales + (Q4 ? kTile * (HD / 16) : 0);
  static constexpr int kValueScales = kValues + (Q4 ? kTile / 2 : kTile) * kValueRow;
  static constexpr int kBytes = kValueScales + (Q4 ? 2 * kTile : 0);
  static __device__ __forceinline__ int key(int p, int c) { return p * kKeyRow + ((Q4 ? c : c ^ (p & 1) << 2) << 4); }
  static __device__ __forceinline__ int value(int m, int c) {
    return kValues + m * kValueRow + ((c ^ (!Q4 ? m & 6 : HD == 128 ? (m & 3) << 1 : m & 2)) << 4);
  }
};

template <int N>
__device__ __forceinline__ void lds_words(uint32_t* d, const uint8_t* p) {
  if constexpr (N == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    d[0] = u.x, d[1] = u.y, d[2] = u.z, d[3] = u.w;
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    d[0] = u.x, d[1] = u.y;
  } else {
    d[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Scores of the 16 positions at slot0: D rows are positions g and g + 8, columns heads 2 t and 2 t + 1.
template <int HD, bool Q4>
__device__ __forceinline__ void scores(float s[4], const uint8_t* tile, int slot0, const uint32_t (*qf)[4],
                                       const float (*bias)[2], int g, int t) {
  using T = Tile<HD, Q4>;
  constexpr int G = HD / 32;
  if constexpr (Q4) {
    const half2 k1032 = __floats2half2_rn(1032.f, 1032.f);
    uint32_t k[2][G], ks[2][G / 2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int p = slot0 + g + 8 * r;
      lds_words<G>(k[r], tile + p * (HD / 2) + t * (4 * G));
      lds_words<G / 2>(ks[r], tile + T::kScales + p * (2 * G));
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      uint32_t x[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // nibbles at bits 0..3: fp16 1024 + (c + 8), made c; at bits 4..7: fp16 64 + (c + 8), left with its 72
        const uint32_t w = k[r][j], top = w >> 8;
        x[r][0] = h2_as_u32(__hsub2(u32_as_h2(lop3_and_xor(w, 0x000f000fu, 0x64086408u)), k1032));
        x[r][1] = lop3_and_xor(w, 0x00f000f0u, 0x54805480u);
        x[r][2] = h2_as_u32(__hsub2(u32_as_h2(lop3_and_xor(top, 0x000f000fu, 0x64086408u)), k1032));
        x[r][3] = lop3_and_xor(top, 0x00f000f0u, 0x54805480u);
      }
      float d[4];
      const uint32_t a0[4] = {x[0][0], x[1][0], x[0][1], x[1][1]}, a1[4] = {x[0][2], x[1][2], x[0][3], x[1][3]};
      mma_from(d, a0, qf[j][0], qf[j][1], bias[j][0], bias[j][1]);
      mma_16816(d, a1, qf[j][2], qf[j][3]);
      const half2 h0 = u32_as_h2(ks[0][j >> 1]), h1 = u32_as_h2(ks[1][j >> 1]);
      const float s0 = j & 1 ? __high2float(h0) : __low2float(h0), s1 = j & 1 ? __high2float(h1) : __low2float(h1);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = j == 0 ? d[e] * (e < 2 ? s0 : s1) : fmaf(d[e], e < 2 ? s0 : s1, s[e]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < G; ++j) {
      uint32_t k[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) lds_words<4>(k[r], tile + T::key(slot0 + g + 8 * r, 4 * j + t));
      const uint32_t a0[4] = {k[0][0], k[1][0], k[0][1], k[1][1]}, a1[4] = {k[0][2], k[1][2], k[0][3], k[1][3]};
      if (j == 0)
        mma_from(s, a0, qf[j][0], qf[j][1], 0.f, 0.f);
      else
        mma_16816(s, a0, qf[j][0], qf[j][1]);
      mma_16816(s, a1, qf[j][2], qf[j][3]);
    }
  }
}

// acc += V^T w.  w: weights of positions g, g + 8 (rows) for heads 2 t, 2 t + 1 (0 for positions that do not count);
// n_valid positions of the 16 count: fp16 rows beyond them are taken as zeros.  acc[i] rows are values value_of(i, 0 / 1).
template <int HD, bool Q4>
__device__ __forceinline__ void accumulate(float (*acc)[4], const uint8_t* tile, int slot0, const float w[4], int n_valid,
                                           int g, int t) {
  using T = Tile<HD, Q4>;
  uint32_t b[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) b[r] = transpose8x8(h2_as_u32(__floats2half2_rn(w[2 * r], w[2 * r + 1])));
  if constexpr (Q4) {
    uint32_t v[2][HD / 32];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      lds_words<HD / 32>(v[r], tile + T::value(slot0 / 2 + t + 4 * r, g * (HD / 8) / 16) + g * (HD / 8) % 16);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      uint32_t x[2][4];  // values 4 i + (0..3) of the lane's, at position pairs t and t + 4
      unpack_int4x8(v[0][i], x[0]);
      unpack_int4x8(v[1][i], x[1]);
      const uint32_t a0[4] = {x[0][0], x[0][1], x[1][0], x[1][1]}, a1[4] = {x[0][2], x[0][3], x[1][2], x[1][3]};
      mma_16816(acc[2 * i], a0, b[0], b[1]);
      mma_16816(acc[2 * i + 1], a1, b[0], b[1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) {
      uint32_t v[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = 2 * t + (r & 1) + 8 * (r >> 1);
        lds_words<4>(v[r], tile + T::value(slot0 + p, 8 * j + g));
        if (n_valid < 16 && p >= n_valid)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[r][i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // value pair 2 i, 2 i + 1 of the 8
        const uint32_t a[4] = {__byte_perm(v[0][i], v[1][i], 0x5410), __byte_perm(v[0][i], v[1][i], 0x7632),
                               __byte_perm(v[2][i], v[3][i], 0x5410), __byte_perm(v[2][i], v[3][i], 0x7632)};
        mma_16816(acc[4 * j + i], a, b[0], b[1]);
      }
    }
  }
}

// The output.  The maximum M is -inf without positions only, and the output 0 then; it is kNoScore where every score is
// -inf or NaN, and the sum of weights 0 or NaN, which the output 0 / 0 or NaN is too.  Else the sum is at least 2^(7 - 16)
// (the weight of the position whose score and scale, below 2^16, set the maximum), or NaN: a NaN of the query or of a key
// never becomes the maximum, but its weight is one.
__device__ __forceinline__ half result(float num, float den, float M) {
  return __float2half_rn(M == -INFINITY ? 0.f : num / den);
}

// Value index of row half r (0: row g, 1: row g + 8) of accumulator i.
template <int HD, bool Q4>
__device__ __forceinline__ int value_of(int i, int r, int g) {
  return Q4 ? g * (HD / 8) + 2 * i + r : 64 * (i >> 2) + 8 * g + 2 * (i & 3) + r;
}

// The four warps' sums of head h, value d; a warp's lie kStride floats behind the one's before.
template <int HD, int kStride>
__device__ __forceinline__ void join_warps(const float* s_acc, const float (*s_m)[kCols], const float (*s_l)[kCols], int h,
                                           int d, float& num, float& den, float& M) {
  M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][h]);
  num = den = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float f = s_m[w][h] == -INFINITY ? 0.f : ex2(s_m[w][h] - M);
    den = fmaf(f, s_l[w][h], den);
    num = fmaf(f, s_acc[w * kStride + h * (HD + 4) + d], num);
  }
}

// kRuns: a tile's runs (more than one where a page is smaller than a 4-bit tile).
template <int HD, bool Q4, int kRuns, bool kJoined>
__global__ void __launch_bounds__(kThreads, Plan<Q4>::kPerSm)
    paged_decode_kernel(const PagedDecodeParams P, const int groups, const float scale_log2) {
  constexpr int G = HD / 32, kTile = Plan<Q4>::kTile, kSub = kTile / 16, kBytes = Tile<HD, Q4>::kBytes;
  constexpr int kStages = Plan<Q4>::kStages;
  constexpr int kMin = Plan<Q4>::kMinChunk, kRun = kTile / kRuns;
  extern __shared__ __align__(128) uint8_t smem[];  // kWarps rings of kStages tiles, then the warps' results
  __shared__ float s_m[kWarps][kCols], s_l[kWarps][kCols];
  __shared__ Range s_range;
  __shared__ Piece s_piece[3];  // this one, the next, the one after
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (kStages * kBytes);
  pdl_launch_dependents();
  pdl_wait();
  const PagedCache& C = P.cache;
  const int rep = P.nq / C.nkv;
  Piece piece;
  if (kJoined) {
    // an eighth of a sequence, by the rank in the cluster
    const int len = seq_len(P, blockIdx.y), L = (len + kCluster * kMin - 1) / (kCluster * kMin) * kMin;
    const int begin = blockIdx.z * L;
    piece = {(int)blockIdx.y, (int)blockIdx.x, begin, len - begin < L ? len : begin + L, -1, -1};
  } else {
    if (warp == 0) first_piece<Q4>(P, C.nkv * groups, lane, s_range, s_piece);
    __syncthreads();
    piece = s_piece[0];
    if (piece.b < 0) return;
  }

  // the ring: tile i of this warp starts at position p_warp + i kWarps kTile and consists of runs of positions inside a page;
  // lane r knows the page of run r
  using T = Tile<HD, Q4>;
  constexpr int stride = kWarps * kTile;
  const int page = 1 << C.page_shift;
  const int64_t k_block = k_block_bytes(page, HD, Q4), v_block = v_block_bytes(page, HD, Q4);
  const uint32_t ring_at = smem_u32(ring);
  int b, kvh, heads, qh0, p_end, p_warp, tiles;
  unsigned there;                                // per ring slot, which runs hold data
  auto take = [&] {
    b = piece.b, kvh = piece.group / groups;
    const int h0 = (piece.group - kvh * groups) * kCols;
    heads = rep - h0 < kCols ? rep - h0 : kCols;
    qh0 = kvh * rep + h0;
    p_end = piece.end;
    p_warp = piece.begin + warp * kTile;
    tiles = p_warp < p_end ? (p_end - p_warp + stride - 1) / stride : 0;
    there = 0;
  };
  auto page_id = [&](int i) {
    const int p = p_warp + i * stride + lane * kRun;
    return i < tiles && lane < kRuns && p < p_end ? page_of(C, b, p) : -1;
  };
  auto issue = [&](int i, int slot, int ids) {
    const unsigned on = __ballot_sync(0xffffffffu, ids >= 0);
    there = (there & ~(15u << (4 * slot))) | on << (4 * slot);
    const uint32_t to = ring_at + slot * kBytes;
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const int id = __shfl_sync(0xffffffffu, ids, r);
      if (id < 0) continue;
      const int slot0 = (p_warp + i * stride + r * kRun) & (page - 1);
      const uint8_t* kb = C.k + ((int64_t)id * C.nkv + kvh) * k_block;
      const uint8_t* vb = C.v + ((int64_t)id * C.nkv + kvh) * v_block;
      const uint8_t* kc = kb + slot0 * T::kKeyRow;
      const uint8_t* vc = vb + (Q4 ? slot0 / 2 : slot0) * T::kValueRow;
      constexpr int kPieces = kRun * T::kKeyRow / 16, kKeyPieces = T::kKeyRow / 16, kValuePieces = T::kValueRow / 16;
      static_assert(kPieces == (Q4 ? kRun / 2 : kRun) * kValuePieces, "keys and values have as many");
#pragma unroll
      for (int o0 = 0; o0 < kPieces; o0 += 32) {
        const int o = o0 + lane;
        copy16(to + T::key(r * kRun + o / kKeyPieces, o % kKeyPieces), kc + 16 * o);
        copy16(to + T::value((Q4 ? r * kRun / 2 : r * kRun) + o / kValuePieces, o % kValuePieces), vc + 16 * o);
      }
      if constexpr (Q4) {
        constexpr int kKeyScales = kRun * (HD / 16) / 16, kScales = kKeyScales + kRun * 2 / 16;
        const uint8_t* ks = kb + page * (HD / 2) + slot0 * (HD / 16);
        const uint8_t* vs = vb + page * (HD / 2) + slot0 * 2;
#pragma unroll
        for (int o0 = 0; o0 < kScales; o0 += 32) {
          const int o = o0 + lane, n = o - kKeyScales;
          if (o < kScales)
            copy16(to + (n < 0 ? T::kScales + r * kRun * (HD / 16) + 16 * o : T::kValueScales + r * kRun * 2 + 16 * n),
                   n < 0 ? ks + 16 * o : vs + 16 * n);
        }
      }
    }
  };
  int id[kStages];
  auto look_up = [&] {
#pragma unroll
    for (int i = 0; i < kStages; ++i) id[i] = page_id(i);
  };
  auto start = [&](int i) {
    if (i < tiles) issue(i, i, id[i]);
    copy_commit();
  };
  take();
  look_up();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) start(i);
  for (int turn = 1;; turn = turn == 2 ? 0 : turn + 1) {  // turn: where the next piece is
    start(kStages - 1);
    int next_id = page_id(kStages);
    if (!kJoined && threadIdx.x == 0) {
      note_split<Q4>(P, C.nkv * groups, piece, s_range.per);
      next_piece<Q4>(P, s_range, false, s_piece[turn == 2 ? 0 : turn + 1]);
    }

    // the queries as the product's column operand: head g, values 32 j + 8 t + (0..7)
    uint32_t qf[G][4];
    float bias[G][2];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (g < heads)
        u = reinterpret_cast<const uint4*>(P.q + b * P.q_token + (qh0 + g) * P.q_head)[4 * j + t];
      qf[j][0] = u.x, qf[j][1] = u.y, qf[j][2] = u.z, qf[j][3] = u.w;
      if (Q4) {
        float sum = 0.f;
#pragma unroll
        for (int i = 1; i < 4; i += 2) {  // the values whose codes carry the 72
          const float2 f = __half22float2(u32_as_h2(qf[j][i]));
          sum += f.x + f.y;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        bias[j][0] = -72.f * __shfl_sync(0xffffffffu, sum, 8 * t);
        bias[j][1] = -72.f * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      }
    }

    float acc[HD / 16][4];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // heads 2 t, 2 t + 1

    int slot = 0;
    for (int i = 0; i < tiles; ++i) {
      copy_wait<kStages - 1>();
      __syncwarp();
      const int p0 = p_warp + i * stride;
      const unsigned held = there >> (4 * slot);
      const uint8_t* tile = ring + slot * kBytes;
      const bool full_tile = p0 + kTile <= p_end && (held & ((1u << kRuns) - 1)) == (1u << kRuns) - 1;
      float s[kSub][4], sv[kSub][2];
      float top[2];
      top[0] = top[1] = held & ((1u << kRuns) - 1) ? kNoScore : -INFINITY;
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        scores<HD, Q4>(s[u], tile, 16 * u, qf, bias, g, t);
        uint32_t scale[2];  // fp16 bits
        if (Q4) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
            scale[r] = reinterpret_cast<const uint16_t*>(tile + T::kValueScales)[16 * u + g + 8 * r];
        }
        if (!full_tile) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (!(p0 + 16 * u + g + 8 * r < p_end && (held >> (16 * u / kRun) & 1))) {
              s[u][2 * r] = s[u][2 * r + 1] = -INFINITY;
              scale[r] = 0x3c00;
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          // exponent of the scale, rounded up: scale * 2^-e < 1 (an integer put into a float's mantissa); -14 for the scale 0
          // of zeroed pages, whose weights stay finite so
          float e = 0.f;
          if (Q4) {
            e = __uint_as_float(scale[r] >> 10 | 0x4b000000u) - (8388608.f + 14.f);
            sv[u][r] = __half2float(__ushort_as_half((unsigned short)scale[r]));
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) top[c] = fmaxf(top[c], fmaf(s[u][2 * r + c], scale_log2, e));
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] + kLazy || top[1] > m[1] + kLazy)) {
        float f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[c] = fmaxf(top[c], m[c]);
          f[c] = m[c] == top[c] ? 1.f : ex2(m[c] - top[c]);
          m[c] = top[c];
          l[c] *= f[c];
        }
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] *= f[e & 1];
      }
      const float shift[2] = {m[0] == -INFINITY ? 0.f : kLift - m[0], m[1] == -INFINITY ? 0.f : kLift - m[1]};
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[u][e] = ex2(fmaf(s[u][e], scale_log2, shift[e & 1]));
          l[e & 1] += s[u][e];
          if (Q4) s[u][e] *= sv[u][e >> 1];
        }
        accumulate<HD, Q4>(acc, tile, 16 * u, s[u], full_tile ? 16 : (held >> (16 * u / kRun) & 1) ? p_end - p0 - 16 * u : 0,
                           g, t);
      }
      __syncwarp();  // every lane has read the tile
      if (i + kStages < tiles) {
        issue(i + kStages, slot, next_id);
        next_id = page_id(i + kStages + 1);
      }
      copy_commit();
      if (++slot == kStages) slot = 0;
    }

    // join the warps: lane (g, t) holds heads 2 t, 2 t + 1 and HD/8 of the values
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], o);
      if (g == 0) {
        s_m[warp][2 * t + c] = m[c];
        s_l[warp][2 * t + c] = l[c];
      }
    }
    // each warp's sums where its last ring slot was; the next piece's first tiles are on their way to the others meanwhile
    constexpr int kRow = HD + 4, kStride = kStages * kBytes / 4;
    static_assert(kCols * kRow * 4 <= kBytes, "the results fit into a ring slot");
    float* s_acc = reinterpret_cast<float*>(smem + (kStages - 1) * kBytes);
    const int64_t row = (int64_t)b * P.nq + qh0;
    const int done_heads = heads, done_slot = piece.slot;
    if (!kJoined) {
      piece = s_piece[turn];
      if (piece.b >= 0) {
        take();
        look_up();
      }
    }
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s_acc[warp * kStride + (2 * t + (e & 1)) * kRow + value_of<HD, Q4>(i, e >> 1, g)] = acc[i][e];
    if (!kJoined && piece.b >= 0) {
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) start(i);
    }
    __syncthreads();
    if constexpr (kJoined) {
      // this CTA's sums, over the first warp's; then every CTA finishes an eighth of the cluster's values
      for (int e = threadIdx.x; e < done_heads * HD; e += kThreads) {
        const int h = e / HD, d = e - h * HD;
        float num, den, M;
        join_warps<HD, kStride>(s_acc, s_m, s_l, h, d, num, den, M);
        s_acc[h * kRow + d] = num;
        if (d == 0) s_acc[h * kRow + HD] = M, s_acc[h * kRow + HD + 1] = den;
      }
      cluster_sync();
      for (int e = blockIdx.z * kThreads + threadIdx.x; e < done_heads * HD; e += kCluster * kThreads) {
        const int h = e / HD, d = e - h * HD;
        const float* sums = s_acc + h * kRow;
        float m8[kCluster], M = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll
        for (int r = 0; r < kCluster; ++r) M = fmaxf(M, m8[r] = cluster_read(sums + HD, r));
#pragma unroll
        for (int r = 0; r < kCluster; ++r) {
          const float f = m8[r] == -INFINITY ? 0.f : ex2(m8[r] - M);
          den = fmaf(f, cluster_read(sums + HD + 1, r), den);
          num = fmaf(f, cluster_read(sums + d, r), num);
        }
        P.out[(row + h) * HD + d] = result(num, den, M);
      }
      cluster_sync();  // nobody leaves while its sums are read
    } else {
      for (int e = threadIdx.x; e < done_heads * HD; e += kThreads) {
        const int h = e / HD, d = e - h * HD;
        float num, den, M;
        join_warps<HD, kStride>(s_acc, s_m, s_l, h, d, num, den, M);
        if (done_slot < 0) {
          P.out[(row + h) * HD + d] = result(num, den, M);
        } else {
          float* ws = workspace<Q4>(P).pieces + (done_slot * (rep < kCols ? rep : kCols) + h) * (HD + 2);
          ws[d] = num;
          if (d == 0) ws[HD] = M, ws[HD + 1] = den;
        }
      }
    }
    if (kJoined || piece.b < 0) return;
    __syncthreads();  // the sums are read: their place becomes a ring slot again
  }
}

// Joins the pieces of a split sequence; one CTA per split and query head, in kParts parts of the pieces that are joined in
// order.  The loads of a part's first pieces wait for nothing but the note of the split.
constexpr int kParts = 4, kAtOnce = 8;
template <int HD, bool Q4>
__global__ void __launch_bounds__(HD * kParts) paged_join_kernel(const PagedDecodeParams P, const int groups) {
  __shared__ float s_num[kParts][HD], s_den[kParts], s_top[kParts];
  const int part = threadIdx.x / HD, d = threadIdx.x % HD;
  pdl_launch_dependents();
  pdl_wait();
  const Workspace w = workspace<Q4>(P);
  const Split split = w.splits[blockIdx.y];
  if (split.b < 0) return;
  const int rep = P.nq / P.cache.nkv, kvh = split.group / groups, h = (split.group - kvh * groups) * kCols + blockIdx.x;
  if (h >= rep) return;
  const int count = split.last - split.first / 2 + 1;
  float M = -INFINITY, num = 0.f, den = 0.f;
  for (int c0 = part * kAtOnce; c0 < count; c0 += kParts * kAtOnce) {
    float x[kAtOnce];
    float2 ml[kAtOnce];
    float top = M;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int c = c0 + i;
      const float* at = w.pieces + ((c == 0 ? split.first : (split.first & ~1) + 2 * c) * gridDim.x + blockIdx.x) * (HD + 2);
      x[i] = c < count ? at[d] : 0.f;
      ml[i] = c < count ? *reinterpret_cast<const float2*>(at + HD) : make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, ml[i].x);
    const float f = M == top ? 1.f : ex2(M - top);
    num *= f, den *= f, M = top;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float fi = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - M);
      num = fmaf(fi, x[i], num);
      den = fmaf(fi, ml[i].y, den);
    }
  }
  s_num[part][d] = num;
  if (d == 0) s_den[part] = den, s_top[part] = M;
  __syncthreads();
  if (part > 0) return;
#pragma unroll
  for (int i = 1; i < kParts; ++i) M = fmaxf(M, s_top[i]);
  num = den = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const float f = s_top[i] == -INFINITY ? 0.f : ex2(s_top[i] - M);
    num = fmaf(f, s_num[i][d], num);
    den = fmaf(f, s_den[i], den);
  }
  P.out[((int64_t)split.b * P.nq + kvh * rep + h) * HD + d] = result(num, den, M);
}

int64_t head_groups(int64_t nq, int64_t nkv) { return (nq / nkv + kCols - 1) / kCols; }

template <int HD, bool Q4, int kRuns>
cudaError_t decode_runs(const PagedDecodeParams& P, cudaStream_t stream) {
  const int rep = P.nq / P.cache.nkv, groups = (int)head_groups(P.nq, P.cache.nkv), units = P.cache.nkv * groups;
  const float scale_log2 = (1.0f / sqrtf((float)HD)) * kLog2e;
  constexpr int kSmem = kWarps * Plan<Q4>::kStages * Tile<HD, Q4>::kBytes, kCtas = Plan<Q4>::kCtas;
  cudaError_t e;
  const int64_t all = (int64_t)P.seqs * units;
  if (all <= cluster_units(Q4, HD) && (int64_t)P.cache.table_cols << P.cache.page_shift <= Plan<Q4>::kClusterMost) {
    if ((e = ensure_smem_attr<paged_decode_kernel<HD, Q4, kRuns, true>>(kSmem)) != cudaSuccess) return e;
    return launch_ex(paged_decode_kernel<HD, Q4, kRuns, true>, dim3((unsigned)units, (unsigned)P.seqs, kCluster),
                     dim3(kThreads), kSmem, stream, dim3(1, 1, kCluster), true, P, groups, scale_log2);
  }
  if ((e = ensure_smem_attr<paged_decode_kernel<HD, Q4, kRuns, false>>(kSmem)) != cudaSuccess) return e;
  e = launch_ex(paged_decode_kernel<HD, Q4, kRuns, false>, dim3(kCtas), dim3(kThreads), kSmem, stream, 1, true, P, groups,
                scale_log2);
  if (e != cudaSuccess) return e;
  return launch_ex(paged_join_kernel<HD, Q4>, dim3((unsigned)(rep < kCols ? rep : kCols), (unsigned)(all < kCtas ? all : kCtas)),
                   dim3(HD * kParts), 0, stream, 1, true, P, groups);
}

template <int HD>
cudaError_t decode_hd(const PagedDecodeParams& P, cudaStream_t stream) {
  if (!P.cache.q4) return decode_runs<HD, false, 1>(P, stream);
  static_assert(Plan<true>::kTile == 64, "the runs of a tile below");
  switch (P.cache.page_shift) {
    case 4: return decode_runs<HD, true, 4>(P, stream);
    case 5: return decode_runs<HD, true, 2>(P, stream);
    default: return decode_runs<HD, true, 1>(P, stream);
  }
}

}  // namespace

int64_t paged_decode_workspace_bytes(int64_t seqs, int64_t nq, int64_t nkv, int64_t hd, int64_t positions) {
  // for either type of page
  const int64_t most = std::min(Plan<true>::kClusterMost, Plan<false>::kClusterMost);
  const int64_t units = std::min(cluster_units(true, hd), cluster_units(false, hd));
  if (seqs * nkv * head_groups(nq, nkv) <= units && positions <= most) return 0;
  const int64_t ctas = std::max(Plan<true>::kCtas, Plan<false>::kCtas), heads = std::min<int64_t>(nq / nkv, kCols);
  return ctas * (int64_t)(sizeof(Split) + 2 * heads * (hd + 2) * sizeof(float));
}

cudaError_t launch_paged_decode(const PagedDecodeParams& P, cudaStream_t stream) {
  return P.cache.hd == 128 ? decode_hd<128>(P, stream) : decode_hd<64>(P, stream);
}

}  // namespace soinfer
