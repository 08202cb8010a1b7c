// Decode attention over a paged cache: one query per sequence, grouped heads, fp16 or 4-bit rows.
//
//   s_p = (q . k_p) / sqrt(hd) for p < len,   o = sum_p exp(s_p - m) v_p / sum_p exp(s_p - m)
//
// Memory bounds it: every cached row is read once and serves the query heads of its group.  Both products run on the
// matrix instruction with the cached rows as its 16-row operand and up to 8 query heads as its 8 columns, so the work a
// 4-bit value costs is its unpacking, not its dot products:
//   scores:  16 positions x 16 values times 16 values x 8 heads.  4-bit codes enter as 72 + c (one LOP3 turns a nibble
//            into the fp16 number 64 + (c + 8)), the product starts at -72 sum q, and the group's scale multiplies the
//            fp32 result -- no code is rounded.
//   output:  16 values x 16 positions times 16 positions x 8 heads.  A position's scale multiplies its probability; that
//            product is split into two bf16 terms (error 2^-17), because its range is the scales' range and one rounding
//            to 8 bits would show.  fp16 rows: the probability times 2^14 is rounded once to fp16 (11 bits; the factor
//            keeps probabilities down to 2^-28 normal).
// The softmax statistics and both sums are fp32.
//
// Work split: positions of all sequences together are cut into chunks of equal length, about as many as the GPU holds
// CTAs, computed on the device from the lengths (no host read; a captured launch serves any lengths).  A CTA of four
// warps takes a chunk of one sequence for one kv head and up to 8 of its query heads, each warp every fourth tile, and
// joins the warps in shared memory.  A sequence cut into several chunks leaves (m, l, acc) per chunk in the workspace and
// a second kernel joins them in order; one chunk is finished in place.
#include <cuda_bf16.h>

#include "launch.cuh"
#include "paged_cache.cuh"

namespace soinfer {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 32;         // positions a warp takes at a time
constexpr int kTargetCtas = 148 * 3;
constexpr int kMinChunk = kTile * kWarps;
constexpr int kCols = 8;          // query heads per CTA
constexpr int kMostLen = 1 << 30;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void mma_bf16_16816(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 block of 16-bit values spread over the warp (lane i: row i / 4, columns 2 (i % 4), + 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint32_t bf2_as_u32(__nv_bfloat162 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Positions of sequence b: its length, at most what its table can name (the length limit keeps positions in 32 bits).
__device__ __forceinline__ int seq_len(const PagedDecodeParams& P, int b) {
  const int64_t table = (int64_t)P.cache.table_cols << P.cache.page_shift;
  const int most = table < kMostLen ? (int)table : kMostLen, n = __ldg(P.lens + b);
  return n < 0 ? 0 : n > most ? most : n;
}

// Chunk length for the batch: a multiple of kMinChunk that gives about kTargetCtas chunks x head groups (warp-wide).
__device__ __forceinline__ int chunk_len(const PagedDecodeParams& P, int units, int lane) {
  long long total = 0;
  for (int b = lane; b < P.seqs; b += 32) total += seq_len(P, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const long long want = (total * units + kTargetCtas - 1) / kTargetCtas;
  const long long c = (want + kMinChunk - 1) / kMinChunk * kMinChunk;
  return (int)(c < kMinChunk ? kMinChunk : c > kMostLen ? kMostLen : c);
}

template <int HD, bool Q4>
struct Tile;  // one 16-position piece in registers

template <int HD>
struct Tile<HD, true> {
  static constexpr int G = HD / kKGroup;
  uint32_t k[2][G];       // words t G + j of positions g and g + 8
  uint32_t ks[2][G / 2];  // their scales
  uint32_t v[2][HD / 32]; // words of position pairs t and t + 4, values g HD/8 ..
  uint32_t vs[2];         // scales of positions g (low half) and g + 8
};

template <int HD>
struct Tile<HD, false> {
  static constexpr int G = HD / 32;
  uint4 k[2][G];   // values 32 j + 8 t .. of positions g and g + 8
  uint4 v[4][HD / 64];  // positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9; values 64 j + 8 g ..
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t* d, const void* p) {
  if constexpr (N == 4) {
    const uint4 u = ldg_stream_u4(p);
    d[0] = u.x, d[1] = u.y, d[2] = u.z, d[3] = u.w;
  } else if constexpr (N == 2) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    d[0] = u.x, d[1] = u.y;
  } else {
    d[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// Loads the 16 positions at slot0 of pool page id (id < 0: zeros) for kv head kvh.
template <int HD>
__device__ __forceinline__ void load_tile(Tile<HD, true>& T, const PagedCache& C, int id, int slot0, int kvh, int g,
                                          int t) {
  constexpr int G = HD / kKGroup;
  if (id < 0) {
    T = Tile<HD, true>{};
    return;
  }
  const int page = 1 << C.page_shift;
  const int64_t at = (int64_t)id * C.nkv + kvh;
  const uint8_t* kb = C.k + at * k_block_bytes(page, HD, true);
  const uint8_t* vb = C.v + at * v_block_bytes(page, HD, true);
  const int code = page * (HD / 2);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int p = slot0 + g + 8 * r;
    load_words<G>(T.k[r], kb + p * (HD / 2) + t * (4 * G));
    load_words<G / 2>(T.ks[r], kb + code + p * (2 * G));
    load_words<HD / 32>(T.v[r], vb + (slot0 / 2 + t + 4 * r) * HD + g * (HD / 8));
    T.vs[r] = __ldg(reinterpret_cast<const unsigned short*>(vb + code) + p);
  }
}

template <int HD>
__device__ __forceinline__ void load_tile(Tile<HD, false>& T, const PagedCache& C, int id, int slot0, int kvh, int g,
                                          int t) {
  if (id < 0) {
    T = Tile<HD, false>{};
    return;
  }
  const int64_t at = (((int64_t)id * C.nkv + kvh) << C.page_shift) + slot0;
  const uint4* kb = reinterpret_cast<const uint4*>(C.k) + at * (HD / 8);
  const uint4* vb = reinterpret_cast<const uint4*>(C.v) + at * (HD / 8);
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) T.k[r][j] = ldg_stream_u4(kb + (g + 8 * r) * (HD / 8) + 4 * j + t);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < HD / 64; ++j)
      T.v[r][j] = ldg_stream_u4(vb + (2 * t + (r & 1) + 8 * (r >> 1)) * (HD / 8) + 8 * j + g);
}

// Scores of the tile: D rows are positions g and g + 8, columns heads 2 t and 2 t + 1.
template <int HD>
__device__ __forceinline__ void scores(float s[4], const Tile<HD, true>& T, const uint32_t (*qf)[4],
                                       const float (*bias)[2]) {
  constexpr int G = HD / kKGroup;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = 0.f;
#pragma unroll
  for (int j = 0; j < G; ++j) {
    float d[4] = {bias[j][0], bias[j][1], bias[j][0], bias[j][1]};
    uint32_t x[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t w = T.k[r][j];  // nibble n at bits 4..7 and 20..23: fp16 64 + (c + 8)
      x[r][0] = lop3_and_xor(w << 4, 0x00f000f0u, 0x54805480u);
      x[r][1] = lop3_and_xor(w, 0x00f000f0u, 0x54805480u);
      x[r][2] = lop3_and_xor(w >> 4, 0x00f000f0u, 0x54805480u);
      x[r][3] = lop3_and_xor(w >> 8, 0x00f000f0u, 0x54805480u);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t a[4] = {x[0][2 * h], x[1][2 * h], x[0][2 * h + 1], x[1][2 * h + 1]};
      mma_16816(d, a, qf[j][2 * h], qf[j][2 * h + 1]);
    }
    const float s0 = __half2float(__ushort_as_half((unsigned short)(T.ks[0][j >> 1] >> (16 * (j & 1)))));
    const float s1 = __half2float(__ushort_as_half((unsigned short)(T.ks[1][j >> 1] >> (16 * (j & 1)))));
    s[0] = fmaf(d[0], s0, s[0]);
    s[1] = fmaf(d[1], s0, s[1]);
    s[2] = fmaf(d[2], s1, s[2]);
    s[3] = fmaf(d[3], s1, s[3]);
  }
}

template <int HD>
__device__ __forceinline__ void scores(float s[4], const Tile<HD, false>& T, const uint32_t (*qf)[4],
                                       const float (*)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = 0.f;
#pragma unroll
  for (int j = 0; j < HD / 32; ++j) {
    const uint32_t a0[4] = {T.k[0][j].x, T.k[1][j].x, T.k[0][j].y, T.k[1][j].y};
    const uint32_t a1[4] = {T.k[0][j].z, T.k[1][j].z, T.k[0][j].w, T.k[1][j].w};
    mma_16816(s, a0, qf[j][0], qf[j][1]);
    mma_16816(s, a1, qf[j][2], qf[j][3]);
  }
}

// acc += V^T p.  p: probabilities of positions g, g + 8 (rows) for heads 2 t, 2 t + 1; n_valid positions of the tile
// count (the rest holds anything: its p is 0 and so must be its values).  acc[i]: rows are values of_row(i, 0 / 1).
template <int HD>
__device__ __forceinline__ void accumulate(float (*acc)[4], const Tile<HD, true>& T, const float p[4], int n_valid,
                                           int g, int) {
  uint32_t hi[2], lo[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float sv = g + 8 * r < n_valid ? __half2float(__ushort_as_half((unsigned short)T.vs[r])) : 0.f;
    const float x0 = p[2 * r] * sv, x1 = p[2 * r + 1] * sv;
    const uint32_t h = bf2_as_u32(__floats2bfloat162_rn(x0, x1));
    const float r0 = x0 - __uint_as_float(h << 16), r1 = x1 - __uint_as_float(h & 0xffff0000u);
    hi[r] = transpose8x8(h);
    lo[r] = transpose8x8(bf2_as_u32(__floats2bfloat162_rn(r0, r1)));
  }
  const __nv_bfloat162 bias = __floats2bfloat162_rn(136.f, 136.f);
#pragma unroll
  for (int w = 0; w < HD / 32; ++w) {
    uint32_t x[2][4];  // values 4 w + (0..3) of the lane's, at position pairs t and t + 4
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t u = lop3_and_xor(T.v[r][w] >> (4 * i), 0x000f000fu, 0x43084308u);  // bf16 128 + (c + 8)
        x[r][i] = bf2_as_u32(__hsub2(*reinterpret_cast<__nv_bfloat162*>(&u), bias));
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t a[4] = {x[0][2 * h], x[0][2 * h + 1], x[1][2 * h], x[1][2 * h + 1]};
      mma_bf16_16816(acc[2 * w + h], a, hi[0], hi[1]);
      mma_bf16_16816(acc[2 * w + h], a, lo[0], lo[1]);
    }
  }
}

template <int HD>
__device__ __forceinline__ void accumulate(float (*acc)[4], Tile<HD, false>& T, const float p[4], int n_valid, int,
                                           int t) {
  uint32_t b[2];
#pragma unroll
  for (int r = 0; r < 2; ++r)
    b[r] = transpose8x8(h2_as_u32(__floats2half2_rn(p[2 * r] * 16384.f, p[2 * r + 1] * 16384.f)));
  if (n_valid < 16) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (2 * t + (r & 1) + 8 * (r >> 1) >= n_valid)
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) T.v[r][j] = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < HD / 64; ++j) {
    const uint32_t* v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = reinterpret_cast<const uint32_t*>(&T.v[r][j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // value pair 2 i, 2 i + 1 of the 8
      const uint32_t a[4] = {__byte_perm(v[0][i], v[1][i], 0x5410), __byte_perm(v[0][i], v[1][i], 0x7632),
                             __byte_perm(v[2][i], v[3][i], 0x5410), __byte_perm(v[2][i], v[3][i], 0x7632)};
      mma_16816(acc[4 * j + i], a, b[0], b[1]);
    }
  }
}

// Value index of row half r (0: row g, 1: row g + 8) of accumulator i.
template <int HD, bool Q4>
__device__ __forceinline__ int value_of(int i, int r, int g) {
  return Q4 ? g * (HD / 8) + 2 * i + r : 64 * (i >> 2) + 8 * g + 2 * (i & 3) + r;
}

template <int HD, bool Q4>
__global__ void __launch_bounds__(kThreads, 3)
    paged_decode_kernel(const PagedDecodeParams P, const int groups, const float scale_log2) {
  constexpr int G = HD / 32, kSub = kTile / 16;
  __shared__ float s_acc[kWarps][kCols][HD + 4];
  __shared__ float s_m[kWarps][kCols], s_l[kWarps][kCols];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const PagedCache& C = P.cache;
  const int rep = P.nq / C.nkv, units = C.nkv * groups;

  // which chunk of which sequence (every warp finds it for itself)
  const int L = chunk_len(P, units, lane);
  int b = -1, len = 0, chunk = 0, count = 0;
  for (int base = 0, before = 0; base < P.seqs; base += 32) {
    const int i = base + lane;
    const int n = i < P.seqs ? seq_len(P, i) : 0;
    const int mine = i < P.seqs ? (n > L ? (n + L - 1) / L : 1) : 0;  // an empty sequence has one chunk: its zeros
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const int c = (int)blockIdx.y - before;
    const unsigned owns = __ballot_sync(0xffffffffu, c >= sum - mine && c < sum);
    if (owns) {
      const int src = __ffs(owns) - 1;
      b = base + src;
      len = __shfl_sync(0xffffffffu, n, src);
      count = __shfl_sync(0xffffffffu, mine, src);
      chunk = c - __shfl_sync(0xffffffffu, sum - mine, src);
      break;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (b < 0) return;
  const int kvh = blockIdx.x / groups, h0 = (blockIdx.x - kvh * groups) * kCols;
  const int heads = rep - h0 < kCols ? rep - h0 : kCols;
  const int qh0 = kvh * rep + h0;
  const int p_begin = chunk * L, p_end = len - p_begin < L ? len : p_begin + L;

  // the queries as the product's column operand: head g, values 32 j + 8 t + (0..7)
  uint32_t qf[G][4];
  float bias[G][2];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (g < heads)
      u = __ldg(reinterpret_cast<const uint4*>(P.q + b * P.q_token + (qh0 + g) * P.q_head) + 4 * j + t);
    qf[j][0] = u.x, qf[j][1] = u.y, qf[j][2] = u.z, qf[j][3] = u.w;
    if (Q4) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
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

  const int page_mask = (1 << C.page_shift) - 1;
  int id[kSub];
  int p0 = p_begin + warp * kTile;
#pragma unroll
  for (int u = 0; u < kSub; ++u) id[u] = p0 + 16 * u < p_end ? page_of(C, b, p0 + 16 * u) : -1;
  for (; p0 < p_end; p0 += kMinChunk) {
    Tile<HD, Q4> tile[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) load_tile<HD>(tile[u], C, id[u], (p0 + 16 * u) & page_mask, kvh, g, t);
    int next[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const int p = p0 + kMinChunk + 16 * u;
      next[u] = p < p_end ? page_of(C, b, p) : -1;
    }
    float s[kSub][4];
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      scores<HD>(s[u], tile[u], qf, bias);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p = p0 + 16 * u + g + 8 * (e >> 1);
        s[u][e] = p < p_end && id[u] >= 0 ? s[u][e] * scale_log2 : -INFINITY;
        top[e & 1] = fmaxf(top[e & 1], s[u][e]);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
      top[c] = fmaxf(top[c], m[c]);
    }
    if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f[c] = m[c] == top[c] ? 1.f : exp2f(m[c] - top[c]);
        m[c] = top[c];
        l[c] *= f[c];
      }
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= f[e & 1];
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[u][e] = s[u][e] == -INFINITY ? 0.f : exp2f(s[u][e] - m[e & 1]);
        l[e & 1] += s[u][e];
      }
      accumulate<HD>(acc, tile[u], s[u], p_end - p0 - 16 * u, g, t);
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) id[u] = next[u];
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
#pragma unroll
  for (int i = 0; i < HD / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s_acc[warp][2 * t + (e & 1)][value_of<HD, Q4>(i, e >> 1, g)] = acc[i][e];
  __syncthreads();
  constexpr float kUndo = Q4 ? 1.f : 1.f / 16384.f;
  for (int e = threadIdx.x; e < heads * HD; e += kThreads) {
    const int h = e / HD, d = e - h * HD;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][h]);
    float den = 0.f, num = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_m[w][h] == -INFINITY ? 0.f : exp2f(s_m[w][h] - M);
      den = fmaf(f, s_l[w][h], den);
      num = fmaf(f, s_acc[w][h][d], num);
    }
    num *= kUndo;
    if (count == 1) {
      P.out[((int64_t)b * P.nq + qh0 + h) * HD + d] = __float2half_rn(M == -INFINITY ? 0.f : num / den);
    } else {
      float* ws = P.ws + ((int64_t)blockIdx.y * P.nq + qh0 + h) * (HD + 2);
      ws[d] = num;
      if (d == 0) ws[HD] = M, ws[HD + 1] = den;
    }
  }
}

// Joins the chunks of a sequence that has several, in order; one CTA per (sequence, query head).
template <int HD>
__global__ void __launch_bounds__(HD) paged_join_kernel(const PagedDecodeParams P, const int units) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 31;
  const int n = seq_len(P, b);
  const int L = chunk_len(P, units, lane);
  if (n <= L) return;  // finished by its only chunk
  int first = 0;
  for (int i = lane; i < b; i += 32) {
    const int x = seq_len(P, i);
    first += x > L ? (x + L - 1) / L : 1;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(0xffffffffu, first, o);
  const int count = (n + L - 1) / L;
  const float* ws = P.ws + ((int64_t)first * P.nq + h) * (HD + 2);
  const int64_t step = (int64_t)P.nq * (HD + 2);
  float M = -INFINITY;
  for (int c = 0; c < count; ++c) M = fmaxf(M, ws[c * step + HD]);
  float num = 0.f, den = 0.f;
  for (int c = 0; c < count; ++c) {
    const float mc = ws[c * step + HD];
    const float f = mc == -INFINITY ? 0.f : exp2f(mc - M);
    den = fmaf(f, ws[c * step + HD + 1], den);
    num = fmaf(f, ws[c * step + threadIdx.x], num);
  }
  P.out[((int64_t)b * P.nq + h) * HD + threadIdx.x] = __float2half_rn(M == -INFINITY ? 0.f : num / den);
}

// Chunks of any lengths: sum over sequences of max(1, ceil(len / L)) with L >= total * units / kTargetCtas.
int64_t most_chunks(int64_t seqs, int64_t units) { return seqs + (kTargetCtas + units - 1) / units; }

int64_t head_groups(int64_t nq, int64_t nkv) { return (nq / nkv + kCols - 1) / kCols; }

template <int HD>
cudaError_t decode_hd(const PagedDecodeParams& P, cudaStream_t stream) {
  const int groups = (int)head_groups(P.nq, P.cache.nkv), units = P.cache.nkv * groups;
  const float scale_log2 = (1.0f / sqrtf((float)HD)) * kLog2e;
  cudaError_t e = launch_ex(P.cache.q4 ? paged_decode_kernel<HD, true> : paged_decode_kernel<HD, false>,
                            dim3((unsigned)units, (unsigned)most_chunks(P.seqs, units)), dim3(kThreads), 0, stream, 1,
                            true, P, groups, scale_log2);
  if (e != cudaSuccess) return e;
  // a table that holds no more than one chunk never splits
  if (((int64_t)P.cache.table_cols << P.cache.page_shift) <= kMinChunk) return cudaSuccess;
  return launch_ex(paged_join_kernel<HD>, dim3((unsigned)P.nq, (unsigned)P.seqs), dim3(HD), 0, stream, 1, true, P,
                   units);
}

}  // namespace

int64_t paged_decode_workspace_bytes(int64_t seqs, int64_t nq, int64_t nkv, int64_t hd) {
  return most_chunks(seqs, nkv * head_groups(nq, nkv)) * nq * (hd + 2) * (int64_t)sizeof(float);
}

cudaError_t launch_paged_decode(const PagedDecodeParams& P, cudaStream_t stream) {
  return P.cache.hd == 128 ? decode_hd<128>(P, stream) : decode_hd<64>(P, stream);
}

}  // namespace soinfer
