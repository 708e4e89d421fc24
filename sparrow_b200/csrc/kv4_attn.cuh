// kv4_attn.cuh -- attention of the newest tokens over a 4-bit cache.
//
// Token t of the m newest of sequence b sees the slots j < len[b] - (m - 1 - t):
//   s_j = scale * q . k_j,  p = softmax(s),  out = sum_j p_j v_j
// (no slot visible: out = 0), and, where asked for, the weight that each slot
// received: w_out[j] = w_in[j] + the sum of p_j over the m tokens and over the
// query heads that share the kv head (w_in counts as 0 for the m newest slots).
#pragma once
#include "kv4.cuh"

namespace vmlm {

struct Kv4Attn {
  const float* q;
  float* out;
  long long ldq, ldo;
  const int32_t* len;
  const float* w_in;
  float* w_out;
  float* lse;    // [n_seq][m][n_q], log2 of the softmax's denominator with the maximum in it
  float scale2;  // scale * log2(e)
  int m, n_q;
};

// One warp per (sequence, token, query head), one slot at a time: a lane has
// d/32 columns, the score is a warp sum, the softmax runs with the largest
// score so far and rescales what it has when that grows. Sums run over blocks
// of 64 slots before they join the total, so that many small weights behind a
// large one are not rounded away one by one.
template <int D>
__global__ void __launch_bounds__(128) kv4_attn_kernel(const Kv4Attn p, const Kv4View c, int* __restrict__ err) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(c.n_seq) * p.m * p.n_q) return;
  const long long tok = row / p.n_q;
  const int head = static_cast<int>(row % p.n_q);
  const long long b = tok / p.m;
  const int t = static_cast<int>(tok % p.m);
  const int kvh = head / (p.n_q / c.n_kv);
  long long n = __ldg(p.len + b);
  if (n > c.cap) {
    if (lane == 0) atomicCAS(err, 0, kDevKv4Slot);
    n = c.cap;
  }
  n -= p.m - 1 - t;
  float q[V], o[V], ob[V];
  #pragma unroll
  for (int i = 0; i < V; ++i)
    q[i] = p.q[tok * p.ldq + static_cast<long long>(head) * D + lane * V + i], o[i] = 0.f, ob[i] = 0.f;
  float top = -INFINITY, sum = 0.f, sum_b = 0.f;
  const long long base_row = (b * c.n_kv + kvh) * c.cap;
  for (long long j = 0; j < n; ++j) {
    if (j % 64 == 0) {
      sum += sum_b, sum_b = 0.f;
      #pragma unroll
      for (int i = 0; i < V; ++i) o[i] += ob[i], ob[i] = 0.f;
    }
    const long long r = base_row + j;
    float k[V], v[V];
    const uint32_t ksb = __ldg(c.ks + r * (D / 32) + lane * V / 32), vsb = __ldg(c.vs + r * (D / 32) + lane * V / 32);
    const __half2 k2 = *reinterpret_cast<const __half2*>(&ksb), v2 = *reinterpret_cast<const __half2*>(&vsb);
    #pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = lane * V + i;
      const uint32_t kc = (__ldg(c.k + r * (D / 2) + col / 2) >> (4 * (col & 1))) & 15u;
      const uint32_t vc = (__ldg(c.v + r * (D / 2) + col / 2) >> (4 * (col & 1))) & 15u;
      k[i] = __half2float(__hfma(__ushort2half_rn(16 + kc), __low2half(k2), __high2half(k2)));
      v[i] = __half2float(__hfma(__ushort2half_rn(16 + vc), __low2half(v2), __high2half(v2)));
    }
    float s = 0.f;
    #pragma unroll
    for (int i = 0; i < V; ++i) s = fmaf(q[i], k[i], s);
    #pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale2;
    if (s > top) {
      const float f = exp2f(top - s);
      sum *= f, sum_b *= f;
      #pragma unroll
      for (int i = 0; i < V; ++i) o[i] *= f, ob[i] *= f;
      top = s;
    }
    const float e = exp2f(s - top);
    sum_b += e;
    #pragma unroll
    for (int i = 0; i < V; ++i) ob[i] = fmaf(e, v[i], ob[i]);
  }
  sum += sum_b;
  #pragma unroll
  for (int i = 0; i < V; ++i) o[i] += ob[i];
  #pragma unroll
  for (int i = 0; i < V; ++i)
    p.out[tok * p.ldo + static_cast<long long>(head) * D + lane * V + i] = n > 0 ? o[i] / sum : 0.f;
  if (p.lse && lane == 0) p.lse[row] = n > 0 ? top + log2f(sum) : 0.f;
}

// The weights: one warp per (sequence, kv head, slot) forms the slot's scores
// again and adds exp2(s - lse) over the rows that see it.
template <int D>
__global__ void __launch_bounds__(128) kv4_weights_kernel(const Kv4Attn p, const Kv4View c) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const long long r = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (r >= static_cast<long long>(c.n_seq) * c.n_kv * c.cap) return;
  const long long j = r % c.cap;
  const int kvh = static_cast<int>(r / c.cap % c.n_kv);
  const long long b = r / c.cap / c.n_kv;
  long long n = __ldg(p.len + b);
  if (n > c.cap) n = c.cap;
  if (j >= n) return;
  const int group = p.n_q / c.n_kv;
  float k[V];
  const uint32_t ksb = __ldg(c.ks + r * (D / 32) + lane * V / 32);
  const __half2 k2 = *reinterpret_cast<const __half2*>(&ksb);
  #pragma unroll
  for (int i = 0; i < V; ++i) {
    const int col = lane * V + i;
    const uint32_t kc = (__ldg(c.k + r * (D / 2) + col / 2) >> (4 * (col & 1))) & 15u;
    k[i] = __half2float(__hfma(__ushort2half_rn(16 + kc), __low2half(k2), __high2half(k2)));
  }
  float w = 0.f;
  for (int t = 0; t < p.m; ++t) {
    if (j >= n - (p.m - 1 - t)) continue;
    for (int g = 0; g < group; ++g) {
      const long long tok = b * p.m + t;
      const int head = kvh * group + g;
      float s = 0.f;
      #pragma unroll
      for (int i = 0; i < V; ++i) s = fmaf(p.q[tok * p.ldq + static_cast<long long>(head) * D + lane * V + i], k[i], s);
      #pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      w += exp2f(s * p.scale2 - p.lse[tok * p.n_q + head]);
    }
  }
  if (lane == 0) p.w_out[r] = (p.w_in && j < n - p.m ? p.w_in[r] : 0.f) + w;
}

}  // namespace vmlm
