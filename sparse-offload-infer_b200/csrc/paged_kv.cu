// Appending rotated keys and values to a paged cache, and reading cached rows back.
//
// Both move rows of hd fp16 values once: what bounds them is memory (a prompt) or the launch (one token).  A row is
// hd/8 lanes x 16 bytes, so a warp holds 256/hd rows; it works on one token, whose position, page, cosines and sines it
// looks up once, and has up to four row loads in flight per lane.
#include "launch.cuh"
#include "paged_cache.cuh"

namespace soinfer {
namespace {

constexpr int kWarps = 8;  // warps per CTA

__device__ __forceinline__ void unpack8(const uint4& u, float x[8]) {
  const half2* p = reinterpret_cast<const half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(p[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float x[8]) {
  uint4 u;
  half2* p = reinterpret_cast<half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
  return u;
}

// Stores this lane's 8 keys (values 8 l .. 8 l + 7) of one position; all lanes of the row take part.
template <int HD>
__device__ __forceinline__ void store_key_q4(uint8_t* block, int page, int slot, int l, bool on, const float x[8]) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = amax_nan(a, x[i]);
  a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));  // the 4 lanes of a 32-value group
  a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
  const half sh = scale_of(a);
  const float s = __half2float(sh);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= (uint32_t)(code_of(x[i], s) & 15) << (4 * ((i >> 1) + 4 * (i & 1)));
  if (!on) return;
  constexpr int G = HD / kKGroup;
  const int j = l >> 2, t = l & 3;
  *reinterpret_cast<uint32_t*>(block + (int64_t)slot * (HD / 2) + 4 * (t * G + j)) = w;
  if (t == 0) reinterpret_cast<half*>(block + (int64_t)page * (HD / 2))[slot * G + j] = sh;
}

// Stores this lane's 8 values of one position.
template <int HD>
__device__ __forceinline__ void store_value_q4(uint8_t* block, int page, int slot, int l, bool on, const float x[8]) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = amax_nan(a, x[i]);
#pragma unroll
  for (int o = 1; o < HD / 8; o <<= 1) a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  const half sh = scale_of(a);
  const float s = __half2float(sh);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= (uint32_t)(code_of(x[i], s) & 15) << (4 * (i & 3));
  if (!on) return;
  uint8_t* at = block + (int64_t)(slot >> 1) * HD + 8 * l + 2 * (slot & 1);
  *reinterpret_cast<uint16_t*>(at) = (uint16_t)w[0];
  *reinterpret_cast<uint16_t*>(at + 4) = (uint16_t)w[1];
  if (l == 0) reinterpret_cast<half*>(block + (int64_t)page * (HD / 2))[slot] = sh;
}

// A warp takes steps [s R, s R + R) of one token; a step is 256/HD rows of one kind (q heads, then k, then v).
//   norm:   x^ = x / sqrt(mean x^2 + eps) * w    (optional; a key's sum in 64 bits: a code may lie next to a border, and
//                                                 the 64-bit sum makes it the same whatever the order of the sum)
//   rotate: y_i = x^_i c_i - x^_{i+h/2} s_i,  y_{i+h/2} = x^_{i+h/2} c_i + x^_i s_i
// in fp32 with each operation rounded by itself, and one rounding to fp16 or to a code at the end.
template <int HD, bool Q4, int R>
__global__ void __launch_bounds__(32 * kWarps) paged_append_kernel(const PagedAppendParams P) {
  constexpr int kLanes = HD / 8, kRows = 32 / kLanes;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, l = lane % kLanes, sub = lane / kLanes;
  const int q_steps = (P.nq + kRows - 1) / kRows, kv_steps = (P.nkv + kRows - 1) / kRows;
  const int steps = q_steps + 2 * kv_steps, per_token = (steps + R - 1) / R;
  const int64_t warp = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (warp >= (int64_t)P.tokens * per_token) return;
  const int t = (int)(warp / per_token), s0 = (int)(warp - (int64_t)t * per_token) * R;

  // the rows first: their loads do not wait for the position
  uint4 raw[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int s = s0 + r;
    const bool is_q = s < q_steps, is_k = !is_q && s < q_steps + kv_steps;
    const int h = (is_q ? s : is_k ? s - q_steps : s - q_steps - kv_steps) * kRows + sub;
    const half* src = is_q ? P.q + t * P.q_token + h * P.q_head
                           : is_k ? P.k + t * P.k_token + h * P.k_head : P.v + t * P.v_token + h * P.v_head;
    raw[r] = make_uint4(0, 0, 0, 0);
    if (s < steps && h < (is_q ? P.nq : P.nkv)) raw[r] = ldg_stream_u4(src + 8 * l);
  }

  int b = t, at = 0;
  if (P.cu) {
    b = owner_of(P.cu, P.seqs, t, lane);
    at = b < P.seqs ? t - __ldg(P.cu + b) : -1;
  } else if (t >= P.seqs) {
    at = -1;
  }
  int64_t pos = -1;
  if (at >= 0) pos = (int64_t)__ldg(P.start + b) + at;
  const bool placed = pos >= 0 && pos < P.table_rows;  // a token of no sequence, or beyond the tables: zeros, no row
  const int page = 1 << P.cache.page_shift;
  int id = -1;
  if (placed && P.cache.k) id = page_of(P.cache, b, (int)pos);
  const int slot = (int)pos & (page - 1);

  float c[8], sn[8], wq[8], wk[8];
  const bool first = l < kLanes / 2;
  {
    const int64_t row = (placed ? pos : 0) * (HD / 2) + 8 * (first ? l : l - kLanes / 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(P.cos_t + row) + i);
      const float4 e = __ldg(reinterpret_cast<const float4*>(P.sin_t + row) + i);
      c[4 * i] = a.x, c[4 * i + 1] = a.y, c[4 * i + 2] = a.z, c[4 * i + 3] = a.w;
      sn[4 * i] = e.x, sn[4 * i + 1] = e.y, sn[4 * i + 2] = e.z, sn[4 * i + 3] = e.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sn[i] = first ? -sn[i] : sn[i];
    if (P.q_norm) unpack8(__ldg(reinterpret_cast<const uint4*>(P.q_norm) + l), wq);
    if (P.k_norm) unpack8(__ldg(reinterpret_cast<const uint4*>(P.k_norm) + l), wk);
  }

#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int s = s0 + r;
    if (s >= steps) break;
    const bool is_q = s < q_steps, is_k = !is_q && s < q_steps + kv_steps;
    const int h = (is_q ? s : is_k ? s - q_steps : s - q_steps - kv_steps) * kRows + sub;
    const bool on = h < (is_q ? P.nq : P.nkv);
    const bool cached = on && id >= 0;
    uint8_t* kb = nullptr;
    uint8_t* vb = nullptr;
    if (cached) {
      kb = P.cache.k + ((int64_t)id * P.nkv + h) * k_block_bytes(page, HD, Q4);
      vb = P.cache.v + ((int64_t)id * P.nkv + h) * v_block_bytes(page, HD, Q4);
    }
    if (!is_q && !is_k) {
      if (Q4) {
        float x[8];
        unpack8(raw[r], x);
        store_value_q4<HD>(vb, page, slot, l, cached, x);
      } else if (cached) {
        reinterpret_cast<uint4*>(vb)[(int64_t)slot * kLanes + l] = raw[r];
      }
      continue;
    }
    float x[8], y[8];
    unpack8(raw[r], x);
    if (is_q ? P.q_norm != nullptr : P.k_norm != nullptr) {
      float inv;
      if (is_q) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        inv = rsqrtf(ss / (float)HD + P.eps);
      } else {
        double ss = 0.0;  // the squares are exact in fp32
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += (double)__fmul_rn(x[i], x[i]);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        inv = (float)(1.0 / sqrt(ss / (double)HD + (double)P.eps));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inv), is_q ? wq[i] : wk[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl_xor_sync(0xffffffffu, x[i], kLanes / 2);
      y[i] = placed ? __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(o, sn[i])) : 0.f;
    }
    if (is_q) {
      if (on) *reinterpret_cast<uint4*>(P.q_out + ((int64_t)t * P.nq + h) * HD + 8 * l) = pack8(y);
      continue;
    }
    const uint4 packed = pack8(y);
    if (on && P.k_out) *reinterpret_cast<uint4*>(P.k_out + ((int64_t)t * P.nkv + h) * HD + 8 * l) = packed;
    if (Q4)
      store_key_q4<HD>(kb, page, slot, l, cached, y);
    else if (cached)
      reinterpret_cast<uint4*>(kb)[(int64_t)slot * kLanes + l] = packed;
  }
}

// A warp reads one position's rows of every kv head, keys then values.
template <int HD, bool Q4>
__global__ void __launch_bounds__(32 * kWarps)
    paged_read_kernel(const PagedCache C, const int32_t* __restrict__ cu, const int seqs, const int tokens,
                      half* __restrict__ k_out, half* __restrict__ v_out) {
  constexpr int kLanes = HD / 8, kRows = 32 / kLanes;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, l = lane % kLanes, sub = lane / kLanes;
  const int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const int b = owner_of(cu, seqs, t, lane);
  if (b >= seqs) return;  // behind the last sequence: left as it was
  const int pos = t - __ldg(cu + b);
  if (pos < 0) return;
  const int page = 1 << C.page_shift, slot = pos & (page - 1);
  const int id = page_of(C, b, pos);
  const int64_t kbb = k_block_bytes(page, HD, Q4), vbb = v_block_bytes(page, HD, Q4);
#pragma unroll 4
  for (int h = sub; h < C.nkv; h += kRows) {
    uint4 ko = make_uint4(0, 0, 0, 0), vo = make_uint4(0, 0, 0, 0);
    if (id >= 0) {
      const uint8_t* kb = C.k + ((int64_t)id * C.nkv + h) * kbb;
      const uint8_t* vb = C.v + ((int64_t)id * C.nkv + h) * vbb;
      if (Q4) {
        constexpr int G = HD / kKGroup;
        const int j = l >> 2, tq = l & 3;
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(kb + (int64_t)slot * (HD / 2)) + tq * G + j);
        const float ks = __half2float(reinterpret_cast<const half*>(kb + (int64_t)page * (HD / 2))[slot * G + j]);
        const uint2 vw = __ldg(reinterpret_cast<const uint2*>(vb + (int64_t)(slot >> 1) * HD + 8 * l));
        const float vs = __half2float(reinterpret_cast<const half*>(vb + (int64_t)page * (HD / 2))[slot]);
        float kx[8], vx[8];
        const int sh = 16 * (slot & 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int n = (w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15;
          kx[i] = (float)((n ^ 8) - 8) * ks;
          const int m = ((i < 4 ? vw.x : vw.y) >> (sh + 4 * (i & 3))) & 15;
          vx[i] = (float)((m ^ 8) - 8) * vs;
        }
        ko = pack8(kx);
        vo = pack8(vx);
      } else {
        ko = ldg_stream_u4(reinterpret_cast<const uint4*>(kb) + (int64_t)slot * kLanes + l);
        vo = ldg_stream_u4(reinterpret_cast<const uint4*>(vb) + (int64_t)slot * kLanes + l);
      }
    }
    const int64_t o = ((int64_t)t * C.nkv + h) * kLanes + l;
    reinterpret_cast<uint4*>(k_out)[o] = ko;
    reinterpret_cast<uint4*>(v_out)[o] = vo;
  }
}

template <int HD, bool Q4>
cudaError_t append_hd(const PagedAppendParams& P, cudaStream_t stream) {
  constexpr int kRows = 256 / HD;
  const int steps = (P.nq + kRows - 1) / kRows + 2 * ((P.nkv + kRows - 1) / kRows);
  // few tokens: one step per warp, for latency; many: four, so that a warp's look-ups serve more rows
  const bool wide = (int64_t)P.tokens * steps >= 148 * 64;
  const int per_token = wide ? (steps + 3) / 4 : steps;
  const unsigned ctas = (unsigned)(((int64_t)P.tokens * per_token + kWarps - 1) / kWarps);
  return launch_ex(wide ? paged_append_kernel<HD, Q4, 4> : paged_append_kernel<HD, Q4, 1>, dim3(ctas),
                   dim3(32 * kWarps), 0, stream, 1, true, P);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& P, cudaStream_t stream) {
  if (P.cache.hd == 128) return P.cache.q4 ? append_hd<128, true>(P, stream) : append_hd<128, false>(P, stream);
  return P.cache.q4 ? append_hd<64, true>(P, stream) : append_hd<64, false>(P, stream);
}

cudaError_t launch_paged_read(const PagedCache& C, const int32_t* cu, int seqs, int tokens, half* k_out, half* v_out,
                              cudaStream_t stream) {
  const dim3 grid((unsigned)((tokens + kWarps - 1) / kWarps)), block(32 * kWarps);
  if (C.hd == 128)
    return launch_ex(C.q4 ? paged_read_kernel<128, true> : paged_read_kernel<128, false>, grid, block, 0, stream, 1,
                     true, C, cu, seqs, tokens, k_out, v_out);
  return launch_ex(C.q4 ? paged_read_kernel<64, true> : paged_read_kernel<64, false>, grid, block, 0, stream, 1, true,
                   C, cu, seqs, tokens, k_out, v_out);
}

}  // namespace soinfer
