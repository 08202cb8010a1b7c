// Causal attention of packed prompts (grouped heads, sequences of different lengths).
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace soinfer {
namespace {

constexpr int kWarps = 4;

// One warp per (query row, head): row i of a sequence sees keys j <= i + len_k - len_q.
template <int HD>
__global__ void __launch_bounds__(32 * kWarps) prefill_rows_kernel(const PrefillParams P, const float scale_log2) {
  constexpr int E = HD / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5), h = blockIdx.y;
  if (row >= P.tokens_q) return;
  int b = 0;
  while (b < P.seqs && P.cu_q[b + 1] <= row) ++b;
  if (b >= P.seqs || row < P.cu_q[b]) return;
  const int q0 = max(P.cu_q[b], 0), lq = min(P.cu_q[b + 1], P.tokens_q) - q0;
  const int k0 = max(P.cu_k[b], 0), lk = max(min(P.cu_k[b + 1], P.tokens_k) - k0, 0);
  const int kvh = h / (P.nq / P.nkv), n = row - q0 + 1 + lk - lq;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    q[e] = __half2float(P.q[row * P.q_token + h * P.q_head + lane * E + e]) * scale_log2;
    acc[e] = 0.f;
  }
  for (int j = 0; j < n; ++j) {
    const half* k = P.k + (k0 + j) * P.k_token + kvh * P.k_head + lane * E;
    const half* v = P.v + (k0 + j) * P.v_token + kvh * P.v_head + lane * E;
    float s = 0.f;
    for (int e = 0; e < E; ++e) s = fmaf(q[e], __half2float(k[e]), s);
    s = warp_sum(s);
    const float top = fmaxf(m, s), f = m == top ? 1.f : exp2f(m - top), p = exp2f(s - top);
    m = top;
    l = fmaf(l, f, p);
    for (int e = 0; e < E; ++e) acc[e] = fmaf(p, __half2float(v[e]), acc[e] * f);
  }
  for (int e = 0; e < E; ++e)
    P.out[((int64_t)row * P.nq + h) * HD + lane * E + e] = __float2half_rn(n > 0 ? acc[e] / l : 0.f);
}

}  // namespace

cudaError_t launch_prefill_attention(const PrefillParams& P, cudaStream_t stream) {
  const float scale_log2 = (1.0f / sqrtf((float)P.hd)) * 1.4426950408889634f;
  const dim3 grid((unsigned)((P.tokens_q + kWarps - 1) / kWarps), (unsigned)P.nq);
  return launch_ex(P.hd == 128 ? prefill_rows_kernel<128> : prefill_rows_kernel<64>, grid, dim3(32 * kWarps), 0, stream,
                   1, true, P, scale_log2);
}

}  // namespace soinfer
