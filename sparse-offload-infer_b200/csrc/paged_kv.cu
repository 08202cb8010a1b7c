// Appending rotated keys and values to a paged cache, and reading cached rows back.
//
// Both move rows of hd fp16 values once: what bounds them is memory (a prompt) or the launch (one token).
// Measured (GPU time): 8675 tokens of 40 / 8 heads of 128 into fp16 pages 50 us for 266 MB (0.82 of the measured copy rate);
// one token 2.3 us; 65431 4-bit positions of 8 heads read back 61 us for 340 MB (0.86); 3759 tokens of 16 / 8 heads into 4
// bits 20 us, where 58 MB alone would take 9: 0.53 instructions per cycle and scheduler from the 3.9 warps that 96 registers a
// thread leave, DRAM 17% busy -- latency that few warps leave open -- and 2.5 waves of CTAs.
#include "launch.cuh"
#include "paged_cache.cuh"

namespace soinfer {
namespace {

constexpr int kWarps = 4;  // warps per CTA

// Eight fp16 values as pairs of fp32, and back.
__device__ __forceinline__ void unpack8(const uint4& u, uint64_t x[4]) {
  const half2* p = reinterpret_cast<const half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(p[i]);
    x[i] = pack2(f.x, f.y);
  }
}
__device__ __forceinline__ uint4 pack8(const float x[8]) {
  uint4 u;
  half2* p = reinterpret_cast<half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
  return u;
}
__device__ __forceinline__ uint4 pack8(const uint64_t x[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(x[i], f[2 * i], f[2 * i + 1]);
  return pack8(f);
}

__device__ __forceinline__ float amax8(const uint64_t x[4]) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f, g;
    unpack2(x[i], f, g);
    a = amax_nan(amax_nan(a, f), g);
  }
  return a;
}

// Stores this lane's keys (x[half]: values half hd/2 + 8 l ..) of one position; the lanes of a row take part.
template <int HD>
__device__ __forceinline__ void store_key_q4(uint8_t* block, int page, int slot, int l, bool on, const uint64_t (*x)[4]) {
  constexpr int G = HD / kKGroup;
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    float a = amax8(x[f]);
    a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));  // the 4 lanes of a 32-value group
    a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const half sh = scale_of(a);
    const float s = __half2float(sh);
    const uint32_t w = key_word(x[f], s, __fdiv_rn(1.f, s));
    if (!on) continue;
    const int j = f * (G / 2) + (l >> 2), t = l & 3;
    *reinterpret_cast<uint32_t*>(block + (int64_t)slot * (HD / 2) + 4 * (t * G + j)) = w;
    if (t == 0) reinterpret_cast<half*>(block + (int64_t)page * (HD / 2))[slot * G + j] = sh;
  }
}

// Stores this lane's values of one position.
template <int HD>
__device__ __forceinline__ void store_value_q4(uint8_t* block, int page, int slot, int l, bool on, const uint64_t (*x)[4]) {
  float a = amax_nan(amax8(x[0]), amax8(x[1]));
#pragma unroll
  for (int o = 1; o < HD / 16; o <<= 1) a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  const half sh = scale_of(a);
  const float s = __half2float(sh), inv = __fdiv_rn(1.f, s);
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const uint32_t w = value_word(x[f], s, inv);
    if (!on) continue;
    uint8_t* at = block + (int64_t)(slot >> 1) * HD + f * (HD / 2) + 8 * l + 2 * (slot & 1);
    *reinterpret_cast<uint16_t*>(at) = (uint16_t)w;
    *reinterpret_cast<uint16_t*>(at + 4) = (uint16_t)(w >> 16);
  }
  if (on && l == 0) reinterpret_cast<half*>(block + (int64_t)page * (HD / 2))[slot] = sh;
}

// A warp takes `per` steps of one token; a step is 512/HD rows of one kind (q heads, then k, then v).  A row is hd/16
// lanes, each with 8 values of the row's first half and the same 8 of its second, so that a rotation's pairs lie in one
// lane; the token's position, page, cosines and sines are looked up once, and the next R steps' rows are on their way
// while R are worked on.
//   norm:   x^ = x / sqrt(mean x^2 + eps) * w    (optional; a key's sum in 64 bits: a code may lie next to a border, and
//                                                 the 64-bit sum makes it the same whatever the order of the sum)
//   rotate: y_i = x^_i c_i - x^_{i+h/2} s_i,  y_{i+h/2} = x^_{i+h/2} c_i + x^_i s_i
// in fp32 with each operation rounded by itself, and one rounding to fp16 or to a code at the end.
template <int HD, bool Q4, int R>
__global__ void __launch_bounds__(32 * kWarps, 5) paged_append_kernel(const PagedAppendParams P, const int per) {
  constexpr int kLanes = HD / 16, kRows = 32 / kLanes;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, l = lane % kLanes, sub = lane / kLanes;
  const int q_steps = (P.nq + kRows - 1) / kRows, kv_steps = (P.nkv + kRows - 1) / kRows;
  const int steps = q_steps + 2 * kv_steps, parts = (steps + per - 1) / per;
  const int64_t warp = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (warp >= (int64_t)P.tokens * parts) return;
  const int t = (int)(warp / parts), s0 = (int)(warp - (int64_t)t * parts) * per;
  const int s_end = s0 + per < steps ? s0 + per : steps;

  auto load = [&](int s, uint4 (&x)[2]) {
    const bool is_q = s < q_steps, is_k = !is_q && s < q_steps + kv_steps;
    const int h = (is_q ? s : is_k ? s - q_steps : s - q_steps - kv_steps) * kRows + sub;
    const half* src = is_q ? P.q + t * P.q_token + h * P.q_head
                           : is_k ? P.k + t * P.k_token + h * P.k_head : P.v + t * P.v_token + h * P.v_head;
    x[0] = x[1] = make_uint4(0, 0, 0, 0);
    if (s < s_end && h < (is_q ? P.nq : P.nkv)) {
      x[0] = ld_stream_u4(src + 8 * l);
      x[1] = ld_stream_u4(src + HD / 2 + 8 * l);
    }
  };
  // the first rows before anything else: their loads do not wait for the position
  uint4 raw[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r) load(s0 + r, raw[r]);

  int b = t;
  int64_t pos = -1;
  if (P.cu) {
    const Owner o = owner_of(P.cu, P.seqs, t, lane, P.start);
    b = o.b;
    if (b < P.seqs && t >= o.first) pos = (int64_t)o.x + (t - o.first);
  } else if (t < P.seqs) {
    pos = P.start[t];
  }
  if (pos < 0 || pos >= P.table_rows) {  // of no sequence, or beyond the tables: zeros, whatever the row and the norm hold
    for (int s = s0; s < s_end && s < q_steps + kv_steps; ++s) {
      const bool is_q = s < q_steps;
      const int h = (is_q ? s : s - q_steps) * kRows + sub;
      half* out = is_q ? P.q_out + ((int64_t)t * P.nq + h) * HD : P.k_out + ((int64_t)t * P.nkv + h) * HD;
      if (h < (is_q ? P.nq : P.nkv) && (is_q || P.k_out)) {
        reinterpret_cast<uint4*>(out)[l] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(out)[kLanes + l] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  const int page = 1 << P.cache.page_shift;
  const int id = page_of(P.cache, b, (int)pos);
  const int slot = (int)pos & (page - 1);
  const int64_t k_block = k_block_bytes(page, HD, Q4), v_block = v_block_bytes(page, HD, Q4);
  uint8_t* k_base = P.cache.k + (int64_t)id * P.nkv * k_block;
  uint8_t* v_base = P.cache.v + (int64_t)id * P.nkv * v_block;

  uint64_t c[4], sn[4];  // pairs, as the rows'
  {
    const int64_t row = pos * (HD / 2) + 8 * l;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(P.cos_t + row) + i);
      const float4 e = __ldg(reinterpret_cast<const float4*>(P.sin_t + row) + i);
      c[2 * i] = pack2(a.x, a.y), c[2 * i + 1] = pack2(a.z, a.w);
      sn[2 * i] = pack2(e.x, e.y), sn[2 * i + 1] = pack2(e.z, e.w);
    }
  }

  for (int s1 = s0; s1 < s_end; s1 += R) {
    uint4 cur[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) cur[r][0] = raw[r][0], cur[r][1] = raw[r][1];
    if (s1 + R < s_end)
#pragma unroll
      for (int r = 0; r < R; ++r) load(s1 + R + r, raw[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int s = s1 + r;
      if (s >= s_end) break;
      const bool is_q = s < q_steps, is_k = !is_q && s < q_steps + kv_steps;
      const int h = (is_q ? s : is_k ? s - q_steps : s - q_steps - kv_steps) * kRows + sub;
      const bool on = h < (is_q ? P.nq : P.nkv);
      const bool cached = on && id >= 0;
      uint64_t x[2][4];
      unpack8(cur[r][0], x[0]);
      unpack8(cur[r][1], x[1]);
      if (!is_q && !is_k) {
        uint8_t* vb = v_base + h * v_block;
        if (Q4) {
          store_value_q4<HD>(vb, page, slot, l, cached, x);
        } else if (cached) {
          uint4* dst = reinterpret_cast<uint4*>(vb) + (int64_t)slot * (HD / 8) + l;
          dst[0] = cur[r][0];
          dst[kLanes] = cur[r][1];
        }
        continue;
      }
      const half* w = is_q ? P.q_norm : P.k_norm;
      if (w) {
        float inv;
        uint64_t wf[2][4];
        unpack8(__ldg(reinterpret_cast<const uint4*>(w) + l), wf[0]);
        unpack8(__ldg(reinterpret_cast<const uint4*>(w) + kLanes + l), wf[1]);
        if (is_q) {
          uint64_t ss2 = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) ss2 = fma2(x[0][i], x[0][i], fma2(x[1][i], x[1][i], ss2));
          float ss, other;
          unpack2(ss2, ss, other);
          ss += other;
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          inv = rsqrtf(ss / (float)HD + P.eps);
        } else {
          double ss = 0.0;  // the squares are exact in fp32
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a, b, c2, d;
            unpack2(mul2(x[0][i], x[0][i]), a, b);
            unpack2(mul2(x[1][i], x[1][i]), c2, d);
            ss += ((double)a + (double)b) + ((double)c2 + (double)d);
          }
#pragma unroll
          for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          // 1 / sqrt by Newton's iteration r += r (1 - a r^2) / 2 from the fp32 value: 2^-22 -> 2^-43 -> 64-bit rounding
          // (not from the 0 of an infinite mean square, which is the result)
          const double a = ss * (1.0 / HD) + (double)P.eps;
          double r = (double)rsqrtf((float)a);
          if (r != 0.0) {
            r = fma(0.5 * r, fma(-a * r, r, 1.0), r);
            r = fma(0.5 * r, fma(-a * r, r, 1.0), r);
          }
          inv = (float)r;
        }
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[f][i] = mul2(mul2(x[f][i], both(inv)), wf[f][i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (sums one by one: products and sums of pairs may be contracted, which these must not be)
        const uint64_t a = x[0][i], e = x[1][i];
        float p0, p1, q0, q1;
        unpack2(mul2(a, c[i]), p0, p1);
        unpack2(mul2(e, sn[i]), q0, q1);
        x[0][i] = pack2(__fsub_rn(p0, q0), __fsub_rn(p1, q1));
        unpack2(mul2(e, c[i]), p0, p1);
        unpack2(mul2(a, sn[i]), q0, q1);
        x[1][i] = pack2(__fadd_rn(p0, q0), __fadd_rn(p1, q1));
      }
      const uint4 lo = pack8(x[0]), hi = pack8(x[1]);
      half* out = is_q ? P.q_out + ((int64_t)t * P.nq + h) * HD : P.k_out + ((int64_t)t * P.nkv + h) * HD;
      if (on && (is_q || P.k_out)) {
        reinterpret_cast<uint4*>(out)[l] = lo;
        reinterpret_cast<uint4*>(out)[kLanes + l] = hi;
      }
      if (is_q) continue;
      uint8_t* kb = k_base + h * k_block;
      if (Q4) {
        store_key_q4<HD>(kb, page, slot, l, cached, x);
      } else if (cached) {
        uint4* dst = reinterpret_cast<uint4*>(kb) + (int64_t)slot * (HD / 8) + l;
        dst[0] = lo;
        dst[kLanes] = hi;
      }
    }
  }
}

// Reads two packed rows t, t + 1 (mostly positions 2 m, 2 m + 1 of one sequence, which share their 4-bit values' words).
// fp16: hd/8 lanes copy a row.  4 bits: 8 lanes take a kv head at a pair of positions: 4 lanes a position's key codes,
// all of them the pair's values (hd = 64: half as many bytes each).  Every lane reads 16 + 16 bytes of codes and writes 128.
template <int HD, bool Q4>
__global__ void __launch_bounds__(32 * kWarps)
    paged_read_kernel(const PagedCache C, const int32_t* cu, const int seqs, const int tokens, half* k_out, half* v_out) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int t0 = 2 * (blockIdx.x * kWarps + (threadIdx.x >> 5));
  if (t0 >= tokens) return;
  const int page = 1 << C.page_shift;
  const int64_t kbb = k_block_bytes(page, HD, Q4), vbb = v_block_bytes(page, HD, Q4);
  for (int t = t0, n; t < t0 + 2 && t < tokens; t += n) {
    n = 1;
    const Owner o = owner_of(cu, seqs, t, lane);
    const int b = o.b, pos = t - o.first;
    if (b >= seqs) return;  // behind the last sequence: left as it was
    if (pos < 0) continue;
    if (t == t0 && !(pos & 1) && t + 1 < tokens && t + 1 < o.end) n = 2;
    const int slot = pos & (page - 1), id = page_of(C, b, pos);
    const uint8_t* k_base = C.k + (int64_t)id * C.nkv * kbb;
    const uint8_t* v_base = C.v + (int64_t)id * C.nkv * vbb;
    if constexpr (!Q4) {
      constexpr int kLanes = HD / 8, kRows = 32 / kLanes;
      const int l = lane % kLanes;
      for (int r = 0; r < n; ++r)
#pragma unroll 4
        for (int h = lane / kLanes; h < C.nkv; h += kRows) {
          uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
          if (id >= 0) {
            ko = ld_stream_u4(reinterpret_cast<const uint4*>(k_base + h * kbb) + (int64_t)(slot + r) * kLanes + l);
            vo = ld_stream_u4(reinterpret_cast<const uint4*>(v_base + h * vbb) + (int64_t)(slot + r) * kLanes + l);
          }
          const int64_t o = ((int64_t)(t + r) * C.nkv + h) * kLanes + l;
          reinterpret_cast<uint4*>(k_out)[o] = ko;
          reinterpret_cast<uint4*>(v_out)[o] = vo;
        }
    } else {
      constexpr int G = HD / kKGroup;
      const int l = lane & 7, tq = l & 3, first = slot & 1;
      const int kr = n == 2 ? l >> 2 : 0;  // which of the rows this lane's keys belong to
#pragma unroll 2
      for (int h = lane >> 3; h < C.nkv; h += 4) {
        const bool keys = n == 2 || l < 4;
        uint32_t kw[G], ks[G / 2], vw[G];
        float vs[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < G; ++j) kw[j] = vw[j] = 0;
#pragma unroll
        for (int j = 0; j < G / 2; ++j) ks[j] = 0;
        if (id >= 0) {
          const uint8_t *kb = k_base + h * kbb, *vb = v_base + h * vbb;
          const uint32_t* kc = reinterpret_cast<const uint32_t*>(kb + (int64_t)(slot + kr) * (HD / 2)) + tq * G;
          const uint32_t* kg = reinterpret_cast<const uint32_t*>(kb + (int64_t)page * (HD / 2) + (slot + kr) * (2 * G));
          const uint32_t* vc = reinterpret_cast<const uint32_t*>(vb + (int64_t)(slot >> 1) * HD) + l * G;
          if constexpr (G == 4) {
            const uint4 a = *reinterpret_cast<const uint4*>(kc), e = *reinterpret_cast<const uint4*>(vc);
            const uint2 f = *reinterpret_cast<const uint2*>(kg);
            kw[0] = a.x, kw[1] = a.y, kw[2] = a.z, kw[3] = a.w, vw[0] = e.x, vw[1] = e.y, vw[2] = e.z, vw[3] = e.w;
            ks[0] = f.x, ks[1] = f.y;
          } else {
            const uint2 a = *reinterpret_cast<const uint2*>(kc), e = *reinterpret_cast<const uint2*>(vc);
            kw[0] = a.x, kw[1] = a.y, vw[0] = e.x, vw[1] = e.y;
            ks[0] = *kg;
          }
          const half2 v2 = u32_as_h2(reinterpret_cast<const uint32_t*>(vb + (int64_t)page * (HD / 2))[slot >> 1]);
          vs[0] = __low2float(v2), vs[1] = __high2float(v2);
        }
        uint4* ko = reinterpret_cast<uint4*>(k_out + ((int64_t)(t + kr) * C.nkv + h) * HD);
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const half2 sc = u32_as_h2(ks[j >> 1]);
          const float s = j & 1 ? __high2float(sc) : __low2float(sc);
          uint32_t u[4];
          unpack_int4x8(kw[j], u);
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(u32_as_h2(u[i]));
            x[2 * i] = f.x * s;
            x[2 * i + 1] = f.y * s;
          }
          if (keys) ko[4 * j + tq] = pack8(x);
        }
        // words 4 values x 2 positions: the low halves of the unpacked pairs are the even position's
        float x[2][4 * G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
          uint32_t u[4];
          unpack_int4x8(vw[j], u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(u32_as_h2(u[i]));
            x[0][4 * j + i] = f.x * vs[0];
            x[1][4 * j + i] = f.y * vs[1];
          }
        }
        for (int r = 0; r < n; ++r) {
          uint4* vo = reinterpret_cast<uint4*>(v_out + ((int64_t)(t + r) * C.nkv + h) * HD) + l * (G / 2);
          const bool odd = first + r;
#pragma unroll
          for (int j = 0; j < G / 2; ++j) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = odd ? x[1][8 * j + i] : x[0][8 * j + i];
            vo[j] = pack8(y);
          }
        }
      }
    }
  }
}

template <int HD, bool Q4>
cudaError_t append_hd(const PagedAppendParams& P, cudaStream_t stream) {
  constexpr int kRows = 512 / HD;
  const int steps = (P.nq + kRows - 1) / kRows + 2 * ((P.nkv + kRows - 1) / kRows);
  // as many steps per warp as still leave the GPU full of warps: a warp's look-ups then serve more rows.  fp16 pages take
  // two steps at a time (50 against 53 us for 8675 tokens), 4-bit ones one, whose code is long (38.9 against 40.5 us for
  // 3759 tokens and their context).
  const int64_t all = (int64_t)P.tokens * steps;
  int per = (int)(all / (148 * 32));
  per = per < 1 ? 1 : per > steps ? steps : per;
  const int parts = (steps + per - 1) / per;
  per = (steps + parts - 1) / parts;
  const int64_t warps = (int64_t)P.tokens * ((steps + per - 1) / per);
  const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps)), block(32 * kWarps);
  if constexpr (!Q4) {
    if (per > 1) return launch_ex(paged_append_kernel<HD, Q4, 2>, grid, block, 0, stream, 1, true, P, per);
  }
  return launch_ex(paged_append_kernel<HD, Q4, 1>, grid, block, 0, stream, 1, true, P, per);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& P, cudaStream_t stream) {
  if (P.cache.hd == 128) return P.cache.q4 ? append_hd<128, true>(P, stream) : append_hd<128, false>(P, stream);
  return P.cache.q4 ? append_hd<64, true>(P, stream) : append_hd<64, false>(P, stream);
}

cudaError_t launch_paged_read(const PagedCache& C, const int32_t* cu, int seqs, int tokens, half* k_out, half* v_out,
                              cudaStream_t stream) {
  const dim3 grid((unsigned)((tokens + 2 * kWarps - 1) / (2 * kWarps))), block(32 * kWarps);
  if (C.hd == 128)
    return launch_ex(C.q4 ? paged_read_kernel<128, true> : paged_read_kernel<128, false>, grid, block, 0, stream, 1,
                     true, C, cu, seqs, tokens, k_out, v_out);
  return launch_ex(C.q4 ? paged_read_kernel<64, true> : paged_read_kernel<64, false>, grid, block, 0, stream, 1, true,
                   C, cu, seqs, tokens, k_out, v_out);
}

}  // namespace soinfer
