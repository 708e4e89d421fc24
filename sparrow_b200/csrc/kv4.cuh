// kv4.cuh -- the 4-bit key/value cache: its format, the kernels that write rows
// (per-head RMSNorm and position rotation of queries and keys, quantisation),
// read them back, and move the kept rows of an evicted cache.
//
// Format. A row is one slot's d values (d = 64, 128 or 256) of one kv head:
// d/2 bytes of codes, column p in byte p/2, the low nibble when p is even (the
// packing of the int4 weights), and for every 32 columns one 32-bit word
// (step, base) of two halves, step in the low one. A code c stands for
//     half(step * (16 + c) + base),
// one rounding. 16 + c because a nibble placed in the top four mantissa bits of
// the half 16.0 (0x4C00) is the half 16 + c: unpacking costs a shift and one
// LOP3 for two values, and one HFMA2 makes them the halves that the tensor
// cores take, so a product with a cached value is exact. Rounding the value
// to a half costs at most 2^-11 of it, where half a code step is about 1/30 of
// the group's range; halves for step and base make 5 bits a value in all.
//
// Rows are [n_seq][n_kv][cap], so one head's slots are contiguous.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"

namespace vmlm {

constexpr int kKv4Group = 32;             // columns that share a step and a base
constexpr float kKv4Clamp = 16384.f;      // |x| saturates here, so that base stays a finite half
constexpr int kDevKv4Slot = 104;          // "KV4: slot outside the cache"
constexpr int kDevRopePos = 105;          // "ROPE: position outside the table"

struct Kv4View {
  uint8_t* k;
  uint8_t* v;
  uint32_t* ks;
  uint32_t* vs;
  long long cap;
  int n_seq, n_kv;
};

struct Kv4Rows {
  const float *q, *k, *v;     // [tokens] rows, strides ldq, ldk, ldv
  float *qo, *ko;             // normalised and rotated rows (ko only without a cache)
  long long ldq, ldk, ldv, ldqo, ldko;
  const float *gq, *gk;       // gains [d], or null: no norm
  const float *cos_t, *sin_t; // [n_pos][rot/2], or null: no rotation
  const int32_t* pos;         // [tokens]
  const int32_t* len;         // [n_seq] slots in use before the call (cache only)
  long long tokens, n_pos, m; // m tokens of each sequence
  float eps;
  int n_q, n_kv, rot, interleaved;
  int vec;                    // every row starts on a 16-byte boundary
};

__device__ __forceinline__ uint32_t kv4_pack_sb(float step, float base) {
  return static_cast<uint32_t>(__half_as_ushort(__float2half_rn(step))) |
         (static_cast<uint32_t>(__half_as_ushort(__float2half_rn(base))) << 16);
}

// min and max that keep a NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// V consecutive floats at p; vec: p is aligned to the widest load that V allows.
template <int V>
__device__ __forceinline__ void load_row(const float* __restrict__ p, bool vec, float (&x)[V]) {
  if (vec) {
    if constexpr (V == 2) {
      const float2 t = *reinterpret_cast<const float2*>(p);
      x[0] = t.x, x[1] = t.y;
    } else {
      #pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 t = *reinterpret_cast<const float4*>(p + i);
        x[i] = t.x, x[i + 1] = t.y, x[i + 2] = t.z, x[i + 3] = t.w;
      }
    }
  } else {
    #pragma unroll
    for (int i = 0; i < V; ++i) x[i] = p[i];
  }
}

template <int V>
__device__ __forceinline__ void store_row(float* __restrict__ p, bool vec, const float (&x)[V]) {
  if (vec) {
    if constexpr (V == 2) {
      *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
    } else {
      #pragma unroll
      for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
  } else {
    #pragma unroll
    for (int i = 0; i < V; ++i) p[i] = x[i];
  }
}

// Quantise the row that a warp holds (lane l has columns V*l .. V*l + V - 1)
// and store it. Every step is one IEEE operation in f32, so the codes are those
// of the definition evaluated in f32 by any other program.
template <int D>
__device__ __forceinline__ void kv4_store_row(const float (&x)[D / 32], uint8_t* codes, uint32_t* sb, long long row) {
  constexpr int V = D / 32;
  constexpr int kLanes = kKv4Group / V;  // lanes of one group
  const int lane = threadIdx.x & 31;
  float c[V];
  #pragma unroll
  for (int i = 0; i < V; ++i) c[i] = min_nan(max_nan(x[i], -kKv4Clamp), kKv4Clamp);
  float lo = c[0], hi = c[0];
  #pragma unroll
  for (int i = 1; i < V; ++i) lo = min_nan(lo, c[i]), hi = max_nan(hi, c[i]);
  #pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float step = __half2float(__float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)));
  const float base = __half2float(__float2half_rn(__fsub_rn(lo, __fmul_rn(16.f, step))));
  const float inv = step > 0.f ? __fdiv_rn(1.f, step) : 0.f;
  uint32_t bits = 0;
  #pragma unroll
  for (int i = 0; i < V; ++i) {
    const float t = __fsub_rn(rintf(__fmul_rn(__fsub_rn(c[i], base), inv)), 16.f);
    bits |= static_cast<uint32_t>(fminf(fmaxf(t, 0.f), 15.f)) << (4 * i);
  }
  uint8_t* dst = codes + row * (D / 2) + lane * (V / 2);
  if constexpr (V == 2) *dst = static_cast<uint8_t>(bits);
  if constexpr (V == 4) *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(bits);
  if constexpr (V == 8) *reinterpret_cast<uint32_t*>(dst) = bits;
  if (lane % kLanes == 0) sb[row * (D / kKv4Group) + lane / kLanes] = kv4_pack_sb(step, base);
}

// One warp per row (token, head): heads 0 .. n_q-1 are queries, then n_kv keys,
// then (with a cache) n_kv values.
//   y = x * (1 / sqrt(sum(x^2) / d + eps)) * gain        (gain given)
//   (a, b) -> (a cos - b sin, b cos + a sin)             (table given)
// on the pairs (i, i + rot/2) or (2i, 2i + 1) of the first rot columns. The sum
// of squares adds halves (i and i + d/2, then d/4, ...), a tree whose order does
// not depend on the lane layout. Products and sums are rounded one by one: a
// key's code must not depend on whether a compiler fused them.
// Bound by HBM: each value is read once and written once.
template <int D, bool kCache>
__global__ void __launch_bounds__(256) kv4_rows_kernel(const Kv4Rows p, const Kv4View c, int* __restrict__ err) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const int heads = p.n_q + p.n_kv + (kCache ? p.n_kv : 0);
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const long long tok = row / heads;
  if (tok >= p.tokens) return;
  const int head = static_cast<int>(row - tok * heads);
  const bool is_q = head < p.n_q;
  const int kvh = is_q ? 0 : (head - p.n_q) % p.n_kv;
  const bool is_v = head >= p.n_q + p.n_kv;
  const float* src = is_q ? p.q + tok * p.ldq + static_cast<long long>(head) * D
                          : (is_v ? p.v + tok * p.ldv : p.k + tok * p.ldk) + static_cast<long long>(kvh) * D;
  float x[V];
  load_row<V>(src + lane * V, p.vec, x);
  if (!is_v) {
    const float* gain = is_q ? p.gq : p.gk;
    if (gain) {
      float s[V];
      #pragma unroll
      for (int i = 0; i < V; ++i) s[i] = __fmul_rn(x[i], x[i]);
      #pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        #pragma unroll
        for (int i = 0; i < V; ++i) s[i] = __fadd_rn(s[i], __shfl_xor_sync(0xffffffffu, s[i], o));
      #pragma unroll
      for (int h = V / 2; h > 0; h /= 2)
        #pragma unroll
        for (int i = 0; i < h; ++i) s[i] = __fadd_rn(s[i], s[i + h]);
      const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(s[0], static_cast<float>(D)), p.eps)));
      #pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inv), __ldg(gain + lane * V + i));
    }
    if (p.cos_t) {
      const long long at = __ldg(p.pos + tok);
      if (at < 0 || at >= p.n_pos) {
        if (lane == 0) atomicCAS(err, 0, kDevRopePos);
        return;
      }
      const int half = p.rot / 2;
      const float *ct = p.cos_t + at * half, *sn = p.sin_t + at * half;
      const int d0 = lane * V;
      if (p.interleaved) {
        #pragma unroll
        for (int i = 0; i < V; i += 2) {
          if (d0 + i < p.rot) {
            const float cv = __ldg(ct + (d0 + i) / 2), sv = __ldg(sn + (d0 + i) / 2);
            const float a = x[i], b = x[i + 1];
            x[i] = __fsub_rn(__fmul_rn(a, cv), __fmul_rn(b, sv));
            x[i + 1] = __fadd_rn(__fmul_rn(b, cv), __fmul_rn(a, sv));
          }
        }
      } else {
        const bool first = d0 < half;  // rot is a multiple of 16, so a lane's columns lie on one side
        const int other = first ? lane + half / V : lane - half / V;
        #pragma unroll
        for (int i = 0; i < V; ++i) {
          const float y = __shfl_sync(0xffffffffu, x[i], other & 31);
          if (d0 < p.rot) {
            const int e = first ? d0 + i : d0 + i - half;
            const float cv = __ldg(ct + e), sv = __ldg(sn + e);
            x[i] = first ? __fsub_rn(__fmul_rn(x[i], cv), __fmul_rn(y, sv))
                         : __fadd_rn(__fmul_rn(x[i], cv), __fmul_rn(y, sv));
          }
        }
      }
    }
  }
  if (is_q) {
    store_row<V>(p.qo + tok * p.ldqo + static_cast<long long>(head) * D + lane * V, p.vec, x);
    return;
  }
  if constexpr (!kCache) {
    store_row<V>(p.ko + tok * p.ldko + static_cast<long long>(kvh) * D + lane * V, p.vec, x);
  } else {
    const long long b = tok / p.m;
    const long long had = __ldg(p.len + b);
    if (had < 0) return;  // an idle sequence
    const long long slot = had + (tok - b * p.m);
    if (slot >= c.cap) {
      if (lane == 0) atomicCAS(err, 0, kDevKv4Slot);
      return;
    }
    kv4_store_row<D>(x, is_v ? c.v : c.k, is_v ? c.vs : c.ks, (b * c.n_kv + kvh) * c.cap + slot);
  }
}

// The eight halves of a code word as four half2 of columns (i, i + 4), i = 0..3.
__device__ __forceinline__ void kv4_unpack(uint32_t w, __half2 step, __half2 base, __half2 (&h)[4]) {
  constexpr uint32_t kMask = 0x03C003C0u, kSixteen = 0x4C004C00u;
  const uint32_t t[4] = {w << 6, w << 2, w >> 2, w >> 6};
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = (t[i] & kMask) | kSixteen;
    h[i] = __hfma2(*reinterpret_cast<const __half2*>(&u), step, base);
  }
}

// Values as halves: one thread per code word (8 columns) of K and of V. Rows
// start[b] + i, i < count; a row at or behind end[b] reads as zeros. Bound by
// the halves it writes (4 d bytes a slot against 1.25 d read).
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4View c, const int32_t* __restrict__ start,
                                                       const int32_t* __restrict__ end, long long count,
                                                       __half* __restrict__ ko, __half* __restrict__ vo,
                                                       int* __restrict__ err) {
  constexpr int W = D / 8;
  const long long rows = static_cast<long long>(c.n_seq) * c.n_kv * count;
  for (long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; t < rows * W * 2;
       t += static_cast<long long>(gridDim.x) * 256) {
    const bool is_v = t >= rows * W;
    const long long u = is_v ? t - rows * W : t;
    const long long r = u / W;
    const int w = static_cast<int>(u % W);
    const long long bh = r / count;
    const long long b = bh / c.n_kv;
    const long long slot = __ldg(start + b) + (r - bh * count);
    uint4 o = make_uint4(0, 0, 0, 0);
    if (slot < __ldg(end + b)) {
      if (slot < 0 || slot >= c.cap) {
        atomicCAS(err, 0, kDevKv4Slot);
      } else {
        const long long at = bh * c.cap + slot;
        const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(is_v ? c.v : c.k) + at * W + w);
        const uint32_t sb = __ldg((is_v ? c.vs : c.ks) + at * (D / kKv4Group) + w / 4);
        const __half2 sb2 = *reinterpret_cast<const __half2*>(&sb);
        __half2 h[4];
        kv4_unpack(word, __low2half2(sb2), __high2half2(sb2), h);
        const __half2 p01 = __lows2half2(h[0], h[1]), p23 = __lows2half2(h[2], h[3]);
        const __half2 p45 = __highs2half2(h[0], h[1]), p67 = __highs2half2(h[2], h[3]);
        o = make_uint4(*reinterpret_cast<const uint32_t*>(&p01), *reinterpret_cast<const uint32_t*>(&p23),
                       *reinterpret_cast<const uint32_t*>(&p45), *reinterpret_cast<const uint32_t*>(&p67));
      }
    }
    *reinterpret_cast<uint4*>((is_v ? vo : ko) + r * D + w * 8) = o;
  }
}

// ------------------------------------------------------------------ eviction

// An order-preserving key of a weight: a NaN is the lowest, -0 equals +0.
__device__ __forceinline__ uint32_t kv4_weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(__fadd_rn(w, 0.f));
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kEvictThreads = 1024;

// One CTA per (sequence, kv head) picks the slots to keep. The first `first`
// and the last `recent` are kept; of the others the `keep - first - recent`
// largest weights, found by a radix select of 8 bits a pass (histogram, then
// the bin that holds the wanted rank): T, the key of the last one kept, and how
// many keys equal to T are kept, lowest slots first. A last pass writes the kept
// slots in order. len_out[b] = min(len, keep).
__global__ void __launch_bounds__(kEvictThreads)
    kv4_select_kernel(const float* __restrict__ w, const int32_t* __restrict__ len, long long cap, int n_kv, int keep,
                      int first, int recent, int32_t* __restrict__ idx, float* __restrict__ w_out,
                      int32_t* __restrict__ len_out, int* __restrict__ err) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_rank;
  __shared__ uint32_t warp_eq[32], warp_kept[32];
  const int bh = blockIdx.x, b = bh / n_kv, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  long long n = __ldg(len + b);
  if (n > cap) {
    if (tid == 0) atomicCAS(err, 0, kDevKv4Slot);
    n = cap;
  }
  if (n < 0) n = 0;
  const float* wr = w + static_cast<long long>(bh) * cap;
  int32_t* io = idx + static_cast<long long>(bh) * keep;
  float* wo = w_out ? w_out + static_cast<long long>(bh) * keep : nullptr;
  if (bh % n_kv == 0 && tid == 0) len_out[b] = static_cast<int32_t>(n < keep ? n : keep);
  if (keep == 0) return;  // w and idx may be null
  if (n <= keep) {
    for (int i = tid; i < keep; i += kEvictThreads) {
      io[i] = i < n ? i : -1;
      if (wo) wo[i] = i < n ? wr[i] : 0.f;
    }
    return;
  }
  const int lo = first, hi = static_cast<int>(n) - recent;  // candidates
  const uint32_t want = static_cast<uint32_t>(keep - first - recent);
  uint32_t prefix = 0, rank = want;  // the rank-th largest among keys with this prefix
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kEvictThreads) {
        const uint32_t key = kv4_weight_key(wr[i]);
        if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0;
        int bin = 255;
        for (; bin > 0; --bin) {
          if (above + hist[bin] >= rank) break;
          above += hist[bin];
        }
        s_prefix = (prefix << 8) | static_cast<uint32_t>(bin);
        s_rank = rank - above;
      }
      __syncthreads();
      prefix = s_prefix;
      rank = s_rank;
      __syncthreads();
    }
  }
  // prefix = T, rank = how many of the keys equal to T are kept (0 where nothing is wanted)
  uint32_t eq_seen = 0, kept = 0;
  for (int i0 = 0; i0 < n; i0 += kEvictThreads) {
    const int i = i0 + tid;
    const bool in = i < n;
    const bool cand = in && i >= lo && i < hi;
    const float x = in ? wr[i] : 0.f;
    const uint32_t key = kv4_weight_key(x);
    const bool eq = cand && want > 0 && key == prefix;
    const uint32_t below = (1u << lane) - 1u;
    const uint32_t eq_mask = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_eq[wid] = __popc(eq_mask);
    __syncthreads();
    uint32_t eq_before = eq_seen, eq_total = 0;
    for (int j = 0; j < 32; ++j) {
      if (j < wid) eq_before += warp_eq[j];
      eq_total += warp_eq[j];
    }
    const bool take = in && (!cand || (want > 0 && key > prefix) ||
                             (eq && eq_before + __popc(eq_mask & below) < rank));
    const uint32_t mask = __ballot_sync(0xffffffffu, take);
    if (lane == 0) warp_kept[wid] = __popc(mask);
    __syncthreads();
    uint32_t at = kept, total = 0;
    for (int j = 0; j < 32; ++j) {
      if (j < wid) at += warp_kept[j];
      total += warp_kept[j];
    }
    at += __popc(mask & below);
    if (take && at < static_cast<uint32_t>(keep)) {
      io[at] = i;
      if (wo) wo[at] = x;
    }
    eq_seen += eq_total;
    kept += total;
    __syncthreads();
  }
}

// Kept rows to the other cache: one thread per 16 bytes of codes of K or V, the
// steps and bases beside them.
template <int D>
__global__ void __launch_bounds__(256) kv4_move_kernel(const Kv4View src, const Kv4View dst, const int32_t* __restrict__ idx,
                                                       int keep) {
  constexpr int U = D / 32;  // 16-byte units of codes in a row, and words of (step, base)
  const long long rows = static_cast<long long>(src.n_seq) * src.n_kv * keep;
  for (long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; t < rows * U * 2;
       t += static_cast<long long>(gridDim.x) * 256) {
    const bool is_v = t >= rows * U;
    const long long u = is_v ? t - rows * U : t;
    const long long r = u / U;
    const int i = static_cast<int>(u % U);
    const int from = __ldg(idx + r);
    if (from < 0) continue;
    const long long bh = r / keep;
    const long long s = bh * src.cap + from, d = bh * dst.cap + (r - bh * keep);
    reinterpret_cast<uint4*>(is_v ? dst.v : dst.k)[d * U + i] =
        __ldg(reinterpret_cast<const uint4*>(is_v ? src.v : src.k) + s * U + i);
    (is_v ? dst.vs : dst.ks)[d * U + i] = __ldg((is_v ? src.vs : src.ks) + s * U + i);
  }
}

}  // namespace vmlm
