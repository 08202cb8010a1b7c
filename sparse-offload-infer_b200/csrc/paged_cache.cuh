// Pages of a KV cache: addressing and the 4-bit row format shared by the append, read and decode kernels.
//
// A (page, kv head) pair owns one block of K bytes and one of V bytes.
//   fp16:   [page][hd] halves each.
//   4 bits: K = page * hd/2 bytes of codes, then page * hd/32 fp16 scales (one per 32 values);
//           V = page * hd/2 bytes of codes, then page fp16 scales (one per position).
// Codes are two's-complement nibbles in [-7, 7] and a value is code * scale.  The words are ordered for the matrix
// instruction that reads them, so that a lane's share of a tile is one contiguous piece:
//   K: word t * (hd/32) + j of a position holds values 32 j + 8 t + (0..7), value 2 i in nibble i and 2 i + 1 in nibble
//      i + 4 (masking one nibble of each 16-bit half gives two consecutive values).  Lane t of a quad reads words
//      t * (hd/32) ..: 16 bytes at hd = 128, every pair of matrix steps inside one scale group.
//   V: positions 2 m and 2 m + 1 share hd/4 words; word w holds values 4 w + (0..3), the even position's in the low half
//      and the odd one's in the high half (masking gives one value at two positions, the product's reduction axis).  Each
//      position owns whole 16-bit units, so rows are appended without reading what is there.
// A scale is fp16(max(amax / 7, 2^-14)) and the code is chosen against the rounded scale.  A row (K: group) that holds
// an infinity or a NaN, or whose scale is beyond fp16, gets code 0 and the scale NaN: it reads as NaN throughout.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace soinfer {

// Tables, lengths, rows and pages may all be written by the kernel before, whose end these kernels' start overlaps, so they are
// read by ordinary loads behind pdl_wait; only norm weights and the rotation's tables take the read-only path.  (Decode of 8
// fp16 sequences 12.4 -> 12.55 us, of one of 777 4-bit positions 5.1 -> 5.2, of two long ones 61.8 either way.)

constexpr int kKGroup = 32;                 // values of a key that share a scale
constexpr float kMinScale = 6.103515625e-5f;  // 2^-14, the smallest normal fp16

__host__ __device__ __forceinline__ int64_t k_block_bytes(int page, int hd, bool q4) {
  return q4 ? (int64_t)page * (hd / 2 + hd / 16) : (int64_t)page * hd * 2;
}
__host__ __device__ __forceinline__ int64_t v_block_bytes(int page, int hd, bool q4) {
  return q4 ? (int64_t)page * (hd / 2 + 2) : (int64_t)page * hd * 2;
}

// Pool page of position pos (>= 0) of sequence b, or -1 when the table or the pool does not hold it.
__device__ __forceinline__ int page_of(const PagedCache& c, int b, int pos) {
  const int col = pos >> c.page_shift;
  if (col >= c.table_cols) return -1;
  int id;  // (movable among asynchronous copies; `pos` comes from what was loaded behind the wait, so the load stays there too)
  asm("ld.global.s32 %0, [%1];" : "=r"(id) : "l"(c.table + (int64_t)b * c.table_stride + col));
  return (id >= 0 && id < c.num_pages) ? id : -1;
}

// Sequence that owns packed row t (all lanes get it; n = no sequence owns the row), its first and last row, and x[its
// index] where x is given.  Everything is loaded at once: what follows waits for one load, not for a chain.
struct Owner {
  int b, first, end, x;
};
__device__ __forceinline__ Owner owner_of(const int32_t* cu, int n, int t, int lane, const int32_t* x = nullptr) {
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane;
    int first = 0, end = 0x7fffffff, xi = 0;
    if (i < n) {
      first = cu[i];
      end = cu[i + 1];
      if (x) xi = x[i];
    }
    const unsigned behind = __ballot_sync(0xffffffffu, i >= n || end > t);
    if (behind) {
      const int src = __ffs(behind) - 1;
      if (base + src >= n) break;
      return {base + src, __shfl_sync(0xffffffffu, first, src), __shfl_sync(0xffffffffu, end, src),
              __shfl_sync(0xffffffffu, xi, src)};
    }
  }
  return {n, 0, 0, 0};
}

// fp16 scale of a group with largest magnitude amax; NaN where that is not finite.  (An infinite scale would be lost where
// a product with the codes 0 leaves a rounding error below zero: a score of -inf, which has no weight.)
__device__ __forceinline__ half scale_of(float amax) {
  const float s = __fdiv_rn(amax, 7.f);
  const half h = __float2half_rn(s < kMinScale ? kMinScale : s);
  return __hisinf(h) ? __ushort_as_half(0x7fff) : h;
}

// Codes against the fp16 scale s (inv = 1 / s): rint(x / s), which needs no clamp since s is at least (1 - 2^-11) of the
// largest magnitude's seventh.  x * inv is within 2^-23 |x / s| < 1e-6 of the quotient, so it rounds alike unless it lies
// that near to a half, where the division decides.  An integer is rounded to by adding 1.5 * 2^23; digits r in base 16 are
// summed up as exact fp32 numbers with 8 added to each, so that the low bits are the offset nibbles.
constexpr float kDigits = 8388608.f + 8.f * (1.f + 16.f + 256.f + 4096.f);  // 2^23 + 0x8888

// The rounded quotients of two values; far: the largest distance from an integer so far.
__device__ __forceinline__ uint64_t quotients2(uint64_t x, uint64_t inv, float& far) {
  const uint64_t y = mul2(x, inv);
  const uint64_t r = add2(add2(y, both(12582912.f)), both(-12582912.f));
  float d, e;
  unpack2(fma2(r, both(-1.f), y), d, e);
  far = fmaxf(far, fmaxf(fabsf(d), fabsf(e)));
  return r;
}
__device__ __forceinline__ uint64_t divided2(uint64_t x, float s) {
  float a, b;
  unpack2(x, a, b);
  return pack2(rintf(__fdiv_rn(a, s)), rintf(__fdiv_rn(b, s)));
}
// The four two's-complement nibbles whose digits v holds.
__device__ __forceinline__ uint32_t nibbles(float v) { return (__float_as_uint(v) & 0xffffu) ^ 0x8888u; }

// Key word of eight values x[4] (pairs of neighbours): value 2 i in nibble i, 2 i + 1 in nibble i + 4; a non-finite s gives
// zeros.
__device__ __forceinline__ uint32_t key_word(const uint64_t x[4], float s, float inv) {
  constexpr float kUnit[4] = {1.f, 16.f, 256.f, 4096.f};
  uint64_t r[4], v = both(kDigits);
  float far = 0.f, lo, hi;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = quotients2(x[i], both(inv), far);
  if (far > 0.499998f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = divided2(x[i], s);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v = fma2(r[i], both(kUnit[i]), v);
  unpack2(v, lo, hi);
  return s <= 65504.f ? nibbles(lo) | nibbles(hi) << 16 : 0u;
}

// Value halves of eight values: the low 16 bits hold values 0..3 in order, the high ones values 4..7.
__device__ __forceinline__ uint32_t value_word(const uint64_t x[4], float s, float inv) {
  uint64_t r[4];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = quotients2(x[i], both(inv), far);
  if (far > 0.499998f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = divided2(x[i], s);
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float a, b;
    unpack2(fma2(r[2 * i + 1], pack2(256.f, 4096.f), fma2(r[2 * i], pack2(1.f, 16.f), pack2(kDigits, 0.f))), a, b);
    w[i] = nibbles(a + b);
  }
  return s <= 65504.f ? w[0] | w[1] << 16 : 0u;
}

// The larger magnitude, NaN if either is NaN.
__device__ __forceinline__ float amax_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(fabsf(b)));
  return m;
}

}  // namespace soinfer
