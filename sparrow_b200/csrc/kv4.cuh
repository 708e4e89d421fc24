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
// the half 16.0 (0x4C00) is the half 16 + c: unpacking costs a LOP3 and a shift or
// a multiply-add for two values, and one HFMA2 makes them the halves that the
// tensor cores take, so a product with a cached value is exact. Rounding the value
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
  int steps;                  // times 256 / d rows that a warp takes
  uint32_t sets;              // warps of a token
  int vec, vec_g, vec_t;      // every row starts on a 16-byte boundary; so do the gains, and the table's rows
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

__device__ __forceinline__ void store4(float* p, bool vec, const float* x) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = x[i];
  }
}

// Two f32 operations in one instruction, each rounded as its own: the rows
// kernel is bound by how many instructions it issues. A sum of products is added
// by scalar operations: a paired product and a paired sum would be contracted to
// a fused multiply-add in spite of their .rn.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
  return *reinterpret_cast<const float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
  return *reinterpret_cast<const float2*>(&r);
}

// How a row lies in the D/8 lanes that hold it: lane l has columns 4 l .. 4 l + 3
// (x[0..3]) and D/2 + 4 l .. (x[4..7]), so 16-byte accesses of neighbouring lanes
// are contiguous, the pairs (i, i + d/2) of a full rotation meet in one lane, and
// a warp does 256 / d rows with one instruction.

// Quantise and store the rows that a warp holds; `on` lanes' rows are stored.
// Every step is one IEEE operation in f32, so the codes are those of the
// definition evaluated in f32 by any other program.
template <int D>
__device__ __forceinline__ void kv4_store_rows(const float (&x)[8], bool on, uint8_t* codes, uint32_t* sb,
                                               long long row) {
  constexpr int L = D / 8;
  const int l = threadIdx.x & (L - 1);
  #pragma unroll
  for (int h = 0; h < 2; ++h) {  // groups of 32 columns: 8 lanes of one half
    float c[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = min_nan(max_nan(x[4 * h + i], -kKv4Clamp), kKv4Clamp);
    float lo = min_nan(min_nan(c[0], c[1]), min_nan(c[2], c[3])), hi = max_nan(max_nan(c[0], c[1]), max_nan(c[2], c[3]));
    #pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float step = __half2float(__float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)));
    const float base = __half2float(__float2half_rn(__fsub_rn(lo, __fmul_rn(16.f, step))));
    const float inv = step > 0.f ? __frcp_rn(step) : 0.f;
    uint32_t bits = 0;
    const float2 less = make_float2(-base, -base), by = make_float2(inv, inv);
    const float2 r0 = mul2(add2(make_float2(c[0], c[1]), less), by), r1 = mul2(add2(make_float2(c[2], c[3]), less), by);
    const float r[4] = {r0.x, r0.y, r1.x, r1.y};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      // rint by adding 1.5 * 2^23 (|x| is far below 2^22): the integer lies in the low bits, and no conversion is needed
      const int n = __float_as_int(__fadd_rn(r[i], 12582912.f)) - 0x4B400000 - 16;
      bits |= static_cast<uint32_t>(min(max(n, 0), 15)) << (4 * i);
    }
    if (on) {
      *reinterpret_cast<uint16_t*>(codes + row * (D / 2) + h * (D / 4) + l * 2) = static_cast<uint16_t>(bits);
      if ((l & 7) == 0) sb[row * (D / kKv4Group) + h * (D / 64) + l / 8] = kv4_pack_sb(step, base);
    }
  }
}

// The sum of a row's squares, added in halves (columns c and c + d/2, then d/4,
// ...): the same tree, and so the same bits, whatever the lanes hold. While a
// lane has several values, each exchange sends one half of them and keeps the
// sums of the other: 7 shuffles for the two rows of d = 128 that a warp holds.
template <int D>
__device__ __forceinline__ float tree_sum(const float (&x)[8]) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x;
  float s[4];
  #pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float2 a = make_float2(x[i], x[i + 1]), b = make_float2(x[i + 4], x[i + 5]);
    const float2 y = mul2(a, a), z = mul2(b, b);
    s[i] = __fadd_rn(y.x, z.x), s[i + 1] = __fadd_rn(y.y, z.y);
  }
  #pragma unroll
  for (int h = 2, o = L / 2; h > 0; h /= 2, o /= 2) {
    const bool up = lane & o;
    #pragma unroll
    for (int i = 0; i < h; ++i) {
      const float mine = up ? s[i + h] : s[i], other = up ? s[i] : s[i + h];
      s[i] = __fadd_rn(mine, __shfl_xor_sync(0xffffffffu, other, o));
    }
  }
  #pragma unroll
  for (int o = L / 8; o > 0; o /= 2) s[0] = __fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], o));
  // lane bits L/2 and L/4 say which of the four values s[0] is the sum of
  s[0] = __fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], L / 2));
  return __fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], L / 4));
}

__device__ __forceinline__ void load4(const float* p, bool vec, float* x) {
  if (vec) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p[i];
  }
}

// Heads 0 .. n_q-1 of a token are queries, then n_kv keys, then (with a cache)
// n_kv values; a warp takes 256 / d rows of one token at a time, p.steps times.
//   y = x * (1 / sqrt(sum(x^2) / d + eps)) * gain        (gain given)
//   (a, b) -> (a cos - b sin, b cos + a sin)             (table given)
// on the pairs (i, i + rot/2) or (2i, 2i + 1) of the first rot columns. Products
// and sums are rounded one by one: a key's code must not depend on whether a
// compiler fused them. Queries and keys may be written in place: a row is read
// whole before it is written, by the same lanes.
// Bound by HBM (each value is read once and written once) and nearly as much by
// instructions: the root and the tree count for 256 / d rows, the token's table
// rows and addresses for all steps. While a step is computed the next one's rows
// are on their way. 2047 tokens of 40 heads of 128, half rotated: 19.4 us, 4.3 TB/s
// (47% of issue slots); 8191 tokens of 48 heads written to a cache: 77 us, 4.6 TB/s
// (62%). In both the warps wait for loads most often (2.4 of 8 to 11 warp-cycles an
// instruction), then for fixed latencies and shuffles.
template <int D, bool kCache>
__global__ void __launch_bounds__(256, 4) kv4_rows_kernel(const Kv4Rows p, const Kv4View c,
                                                                       int* __restrict__ err) {
  constexpr int L = D / 8, kRows = 32 / L;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, l = lane & (L - 1);
  const int heads = p.n_q + p.n_kv + (kCache ? p.n_kv : 0);
  const uint32_t at = blockIdx.x * 8 + (threadIdx.x >> 5), tok = at / p.sets;
  if (tok >= p.tokens) return;
  int h = static_cast<int>(at - tok * p.sets) * (p.steps * kRows) + lane / L;
  const int h1 = min(heads, h - lane / L + p.steps * kRows);
  const bool vec = p.vec;
  const float *q = p.q + tok * p.ldq + 4 * l, *k = p.k + tok * p.ldk + 4 * l - p.n_q * D,
              *v = p.v + tok * p.ldv + 4 * l - (p.n_q + p.n_kv) * D;  // of head 0: a row is h * D further
  auto fetch = [&](int at, float (&x)[8]) {
    if (at < heads) {
      const float* src = (at < p.n_q ? q : at < p.n_q + p.n_kv ? k : v) + at * D;
      load4(src, vec, x);
      load4(src + D / 2, vec, x + 4);
    } else {
      #pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
  };
  float x[8], ahead[8];
  fetch(h, x);
  // The token's cosines and sines of the lane's columns; columns behind rot: 1 and 0.
  float cs[8], sn[8];
  const int half = p.rot / 2;
  const bool whole = !p.interleaved && p.rot == D;
  if (p.cos_t) {
    const long long row = __ldg(p.pos + tok);
    if (row < 0 || row >= p.n_pos) {
      // an idle sequence has no position
      if (lane == 0 && !(kCache && __ldg(p.len + tok / static_cast<uint32_t>(p.m)) < 0)) atomicCAS(err, 0, kDevRopePos);
      return;
    }
    const float *ct = p.cos_t + row * half, *st = p.sin_t + row * half;
    #pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int c0 = z * (D / 2) + 4 * l;  // the lane's first column here
      if (whole && z == 1) {
        #pragma unroll
        for (int i = 4; i < 8; ++i) cs[i] = cs[i - 4], sn[i] = sn[i - 4];
      } else if (c0 >= p.rot) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) cs[4 * z + i] = 1.f, sn[4 * z + i] = 0.f;
      } else if (p.interleaved) {
        #pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float co = __ldg(ct + (c0 + i) / 2), si = __ldg(st + (c0 + i) / 2);
          cs[4 * z + i] = cs[4 * z + i + 1] = co, sn[4 * z + i] = sn[4 * z + i + 1] = si;
        }
      } else {
        const int e = c0 < half ? c0 : c0 - half;
        load4(ct + e, p.vec_t, cs + 4 * z);
        load4(st + e, p.vec_t, sn + 4 * z);
      }
    }
    // The sine with the sign that it has where it is added: a cos - b sin as a sum, the same bits.
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool first = p.interleaved ? (i & 1) == 0 : (i / 4) * (D / 2) + 4 * l < half;
      if (first) sn[i] = -sn[i];
    }
  }
  const uint32_t b = kCache ? tok / static_cast<uint32_t>(p.m) : 0;
  long long cache_row = -1;  // of kv head 0; negative: not written
  if constexpr (kCache) {
    const long long had = __ldg(p.len + b), slot = had + (tok - b * static_cast<uint32_t>(p.m));
    if (had >= 0 && slot >= c.cap && lane == 0) atomicCAS(err, 0, kDevKv4Slot);
    if (had >= 0 && slot < c.cap) cache_row = static_cast<long long>(b) * c.n_kv * c.cap + slot;  // had < 0: an idle sequence
  }

  #pragma unroll 1
  for (; h - lane / L < h1; h += kRows) {
    if (h - lane / L + kRows < h1) fetch(h + kRows, ahead);
    const bool in = h < heads, is_q = h < p.n_q, is_v = h >= p.n_q + p.n_kv;
    if (__any_sync(0xffffffffu, !is_v)) {  // a warp of values has nothing to do before they are stored
      const float* gain = is_q ? p.gq : p.gk;
      const float sum = tree_sum<D>(x);
      if (gain) {
        float g[8];
        load4(gain + 4 * l, p.vec_g, g);
        load4(gain + D / 2 + 4 * l, p.vec_g, g + 4);
        const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(sum, 1.f / D), p.eps)));
        if (!is_v) {
          #pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float2 z = mul2(mul2(make_float2(x[i], x[i + 1]), make_float2(inv, inv)), make_float2(g[i], g[i + 1]));
            x[i] = z.x, x[i + 1] = z.y;
          }
        }
      }
      if (p.cos_t) {
        float y[8];  // each column's partner
        if (whole) {
          #pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[i ^ 4];
        } else if (p.interleaved) {
          #pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
        } else {
          // the partner of a lane's four columns is another lane's four, of either half of the row
          #pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int c0 = w * (D / 2) + 4 * l, to = c0 < half ? c0 + half : c0 - half;
            const int from = lane - l + (to >= 0 ? to / 4 % L : l);
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float lower = __shfl_sync(0xffffffffu, x[i], from);
              const float upper = p.rot > D / 2 ? __shfl_sync(0xffffffffu, x[4 + i], from) : 0.f;
              y[4 * w + i] = to >= D / 2 ? upper : lower;
            }
          }
        }
        #pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (!is_v && (whole || w * (D / 2) + 4 * l < p.rot)) {
            #pragma unroll
            for (int i = 4 * w; i < 4 * w + 4; i += 2) {
              const float2 z = mul2(make_float2(x[i], x[i + 1]), make_float2(cs[i], cs[i + 1]));
              const float2 w2 = mul2(make_float2(y[i], y[i + 1]), make_float2(sn[i], sn[i + 1]));
              x[i] = __fadd_rn(z.x, w2.x), x[i + 1] = __fadd_rn(z.y, w2.y);
            }
          }
        }
      }
    }
    if (is_q || (!kCache && in)) {
      float* to = is_q ? p.qo + tok * p.ldqo + h * D + 4 * l : p.ko + tok * p.ldko + (h - p.n_q) * D + 4 * l;
      store4(to, vec, x);
      store4(to + D / 2, vec, x + 4);
    }
    if constexpr (kCache) {
      if (__any_sync(0xffffffffu, in && !is_q)) {
        const bool on = in && !is_q && cache_row >= 0;
        const int kvh = h - p.n_q - (is_v ? p.n_kv : 0);
        kv4_store_rows<D>(x, on, is_v ? c.v : c.k, is_v ? c.vs : c.ks, on ? cache_row + kvh * c.cap : 0);
      }
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ahead[i];
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

// Values as halves: a thread takes code words (8 columns) of K and of V. Rows
// start[b] + i, i < count; a row at or behind end[b] reads as zeros. Bound by
// the halves it writes (4 d bytes a slot against 1.25 d read): 64 heads of 4096 rows
// of 128 take 29 us, 6.0 TB/s. Grid: (words, n_seq * n_kv).
constexpr int kReadWords = 2;  // of K, and as many of V, that a thread has in flight

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4View c, const int32_t* __restrict__ start,
                                                       const int32_t* __restrict__ end, int count,
                                                       __half* __restrict__ ko, __half* __restrict__ vo,
                                                       int* __restrict__ err) {
  constexpr int W = D / 8;
  pdl_wait_prior();
  pdl_launch_dependents();
  for (long long bh = blockIdx.y; bh < static_cast<long long>(c.n_seq) * c.n_kv; bh += gridDim.y) {
    const int b = static_cast<int>(bh / c.n_kv);
    const long long s0 = __ldg(start + b), e = __ldg(end + b);
    uint32_t word[kReadWords][2], sb[kReadWords][2];
    #pragma unroll
    for (int i = 0; i < kReadWords; ++i) {
      const long long t = static_cast<long long>(blockIdx.x) * (256 * kReadWords) + i * 256 + threadIdx.x;
      const int r = static_cast<int>(t / W), w = threadIdx.x % W;
      const long long slot = s0 + r, at = bh * c.cap + slot;
      const bool on = r < count && slot < e;
      const bool in = slot >= 0 && slot < c.cap;
      if (on && !in) atomicCAS(err, 0, kDevKv4Slot);
      word[i][0] = word[i][1] = sb[i][0] = sb[i][1] = 0;
      if (on && in) {
        word[i][0] = __ldg(reinterpret_cast<const uint32_t*>(c.k) + at * W + w);
        word[i][1] = __ldg(reinterpret_cast<const uint32_t*>(c.v) + at * W + w);
        sb[i][0] = __ldg(c.ks + at * (D / kKv4Group) + w / 4);
        sb[i][1] = __ldg(c.vs + at * (D / kKv4Group) + w / 4);
      }
    }
    #pragma unroll
    for (int i = 0; i < kReadWords; ++i) {
      const long long t = static_cast<long long>(blockIdx.x) * (256 * kReadWords) + i * 256 + threadIdx.x;
      if (t / W >= count) break;
      #pragma unroll
      for (int z = 0; z < 2; ++z) {
        const __half2 sb2 = *reinterpret_cast<const __half2*>(&sb[i][z]);
        __half2 h[4];
        kv4_unpack(word[i][z], __low2half2(sb2), __high2half2(sb2), h);
        const __half2 p01 = __lows2half2(h[0], h[1]), p23 = __lows2half2(h[2], h[3]);
        const __half2 p45 = __highs2half2(h[0], h[1]), p67 = __highs2half2(h[2], h[3]);
        reinterpret_cast<uint4*>(z ? vo : ko)[bh * count * W + t] =
            make_uint4(*reinterpret_cast<const uint32_t*>(&p01), *reinterpret_cast<const uint32_t*>(&p23),
                       *reinterpret_cast<const uint32_t*>(&p45), *reinterpret_cast<const uint32_t*>(&p67));
      }
    }
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
constexpr int kEvictMaxCluster = 8;
constexpr int kEvictBins = 2048;   // 11 bits a pass of the radix select: 11, 11, 10
constexpr int kEvictKeys = 24 * 1024;  // keys that a CTA's shared memory holds, two CTAs on an SM
// Slots a CTA from which a cluster is made larger. 8 heads of 16384 slots take 24.1 us with 4096, 25.7 with 2048, 29.6 with
// 8192; 32 heads of 8192: 22.9, 24.3, 26.2; 16 heads of 6000: 16.2, 16.7, 15.3.
constexpr int kEvictShare = 4096;

// Shared memory: a histogram, the scans' words, the CTA's keys (and later its kept slots).
__host__ __device__ constexpr int evict_smem_bytes(int keys) { return kEvictBins * 4 + 256 + keys * 4; }

struct Kv4Evict {
  const float* w;
  const int32_t* len;
  int32_t* idx;
  float* w_out;
  int32_t* len_out;
  int keep, first, recent;
  int keys;  // keys of a share that lie in shared memory; the others are read again
};

// An exclusive sum over the block's threads and the total; scratch: 33 words.
__device__ __forceinline__ int block_scan(int v, int* scratch, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
  #pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = scratch[lane];
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    scratch[lane] = s;
  }
  __syncthreads();
  const int before = warp ? scratch[warp - 1] : 0;
  *total = scratch[31];
  __syncthreads();
  return before + x - v;
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One cluster per (sequence, kv head), each CTA an equal share of the slots.
// The first `first` and the last `recent` slots are kept; of the others the
// `keep - first - recent` largest weights, found by a radix select over order-
// preserving keys: T, the key of the last one kept, and how many keys equal to
// T are kept, lowest slots first. Each pass counts the keys that share the
// digits found so far by their next digit, in the CTA, then adds the cluster's
// counts; the keys are read from global memory once and stay in shared memory.
// Then every CTA knows what it keeps and where its first kept slot goes, and
// moves its rows. Bound by HBM for long caches (4 bytes a slot, 2.5 d a kept
// one), by the passes' barriers for short ones: 36 heads of 1100 slots of 64, 512
// kept, 9.9 us; 64 heads of up to 32768 slots of 128, 4096 kept, 49 us, where warps
// wait for loads and barriers in turn and DRAM is busy 24% of the time.
template <int D>
__global__ void __launch_bounds__(kEvictThreads, 2)
    kv4_evict_kernel(const Kv4Evict p, const Kv4View src, const Kv4View dst, int* __restrict__ err) {
  extern __shared__ __align__(128) unsigned char smem[];
  uint32_t* hist = reinterpret_cast<uint32_t*>(smem);            // [kEvictBins]
  int* scratch = reinterpret_cast<int*>(hist + kEvictBins);      // [33 + 31]
  uint32_t* keys = reinterpret_cast<uint32_t*>(scratch + 64);    // [p.keys]
  __shared__ int s_pick[3], s_count[2];
  const int tid = threadIdx.x;
  const uint32_t rank = cluster_ctarank();
  uint32_t size;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(size));
  const int bh = blockIdx.y, b = bh / src.n_kv;
  pdl_wait_prior();
  pdl_launch_dependents();
  long long n_all = __ldg(p.len + b);
  if (n_all > src.cap) {
    if (tid == 0 && rank == 0) atomicCAS(err, 0, kDevKv4Slot);
    n_all = src.cap;
  }
  const int n = n_all < 0 ? 0 : static_cast<int>(n_all), keep = p.keep;
  if (bh - b * src.n_kv == 0 && rank == 0 && tid == 0) p.len_out[b] = min(n, keep);
  if (keep == 0) return;  // w and idx may be null
  const int i0 = static_cast<int>(static_cast<long long>(n) * rank / size);
  const int i1 = static_cast<int>(static_cast<long long>(n) * (rank + 1) / size);
  const float* w = p.w + static_cast<long long>(bh) * src.cap;
  int32_t* io = p.idx + static_cast<long long>(bh) * keep;
  float* wo = p.w_out ? p.w_out + static_cast<long long>(bh) * keep : nullptr;
  const int lo = p.first, hi = n - p.recent;  // the slots that the weights decide about
  const bool all = n <= keep;
  uint32_t prefix = 0;
  int shift = 0;  // of a key's digits to prefix
  int want = all ? 0 : keep - p.first - p.recent;  // the want-th largest of the keys that begin with prefix
  auto key_at = [&](int i) { return i - i0 < p.keys ? keys[i - i0] : kv4_weight_key(__ldg(w + i)); };
  if (want > 0) {  // the same in the whole cluster
    for (int i = i0 + tid; i < min(i1, i0 + p.keys); i += kEvictThreads) keys[i - i0] = kv4_weight_key(__ldg(w + i));
    #pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass == 2 ? 10 : 11;
      shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      // equal neighbours in a thread's sequence are counted together: many slots may have the same weight
      int last = -1, run = 0;
      for (int i = max(i0, lo) + tid; i < min(i1, hi); i += kEvictThreads) {
        const uint32_t key = key_at(i);
        if (pass > 0 && (key >> (shift + bits)) != prefix) continue;
        const int bin = static_cast<int>(key >> shift & ((1u << bits) - 1u));
        if (bin != last) {
          if (run) atomicAdd(hist + last, static_cast<uint32_t>(run));
          last = bin, run = 0;
        }
        ++run;
      }
      if (run) atomicAdd(hist + last, static_cast<uint32_t>(run));
      __syncthreads();
      if (size > 1) cluster_sync();
      // thread t has bins kEvictBins - 1 - 2 t and the one below: a sum from the top
      uint32_t c[2] = {0, 0};
      const int top = kEvictBins - 1 - 2 * tid;
      #pragma unroll
      for (int z = 0; z < 2; ++z) {
        if (size == 1) {
          c[z] = hist[top - z];
        } else {
          const uint32_t addr = smem_u32(hist + top - z);
          for (uint32_t r = 0; r < size; ++r) c[z] += ld_cluster_u32(mapa_shared(addr, r));
        }
      }
      int total;
      const int above = block_scan(static_cast<int>(c[0] + c[1]), scratch, &total);
      if (above < want && above + static_cast<int>(c[0]) >= want)
        s_pick[0] = top, s_pick[1] = want - above, s_pick[2] = c[0];
      if (above + static_cast<int>(c[0]) < want && above + static_cast<int>(c[0] + c[1]) >= want)
        s_pick[0] = top - 1, s_pick[1] = want - above - static_cast<int>(c[0]), s_pick[2] = c[1];
      __syncthreads();
      prefix = prefix << bits | static_cast<uint32_t>(s_pick[0]);
      want = s_pick[1];
      const bool done = want == s_pick[2];  // all keys with these digits are kept: the others do not matter
      if (size > 1) cluster_sync();  // the counts have been read
      else __syncthreads();
      if (done) break;
    }
  }
  // prefix = T (or the digits of T that decide), want = how many of the keys equal to it are kept (all kept: 0, not
  // asked). A warp takes neighbouring slots, 32 at a time; the counts of keys above T (and of what is kept anyway) and
  // equal to T before it say where it writes.
  const int lane = tid & 31, warp = tid >> 5;
  const int each = (i1 - i0 + kEvictThreads - 1) / kEvictThreads * 32;
  const int t0 = min(i1, i0 + warp * each), t1 = min(i1, t0 + each);
  const bool pick = !all && keep - p.first - p.recent > 0;
  auto look = [&](int i, bool& sure, bool& equal) {
    sure = i < t1 && (all || i < lo || i >= hi), equal = false;
    if (i < t1 && !sure && pick) {
      const uint32_t key = key_at(i) >> shift;
      sure = key > prefix, equal = key == prefix;
    }
  };
  int sure_n = 0, equal_n = 0;
  for (int i = t0 + lane; i - lane < t1; i += 32) {
    bool sure, equal;
    look(i, sure, equal);
    sure_n += __popc(__ballot_sync(0xffffffffu, sure)), equal_n += __popc(__ballot_sync(0xffffffffu, equal));
  }
  __syncthreads();  // scratch is free
  if (lane == 0) scratch[warp] = sure_n, scratch[32 + warp] = equal_n;
  __syncthreads();
  const int sure_w = scratch[lane], equal_w = scratch[32 + lane];
  const int all_sure = __reduce_add_sync(0xffffffffu, sure_w), all_equal = __reduce_add_sync(0xffffffffu, equal_w);
  int s_seen = __reduce_add_sync(0xffffffffu, lane < warp ? sure_w : 0);
  int e_seen = __reduce_add_sync(0xffffffffu, lane < warp ? equal_w : 0);
  int cta_sure = 0, cta_equal = 0;  // of the CTAs before
  if (size > 1) {
    if (tid == 0) s_count[0] = all_sure, s_count[1] = all_equal;
    cluster_sync();
    for (uint32_t r = 0; r < rank; ++r) {
      cta_sure += static_cast<int>(ld_cluster_u32(mapa_shared(smem_u32(s_count), r)));
      cta_equal += static_cast<int>(ld_cluster_u32(mapa_shared(smem_u32(s_count + 1), r)));
    }
  }
  // where a slot goes: behind the sure ones before it, and the equal ones before it as far as they are kept
  const int base = cta_sure + min(want, cta_equal);  // the CTA's first
  s_seen += cta_sure, e_seen += cta_equal;
  const uint32_t below = (1u << lane) - 1u;
  for (int i = t0 + lane; i - lane < t1; i += 32) {
    bool sure, equal;
    look(i, sure, equal);
    const uint32_t ms = __ballot_sync(0xffffffffu, sure), me = __ballot_sync(0xffffffffu, equal);
    const int e_before = e_seen + __popc(me & below);
    if (sure || (equal && e_before < want)) {
      const int at = s_seen + __popc(ms & below) + min(want, e_before);
      io[at] = i;
      if (wo) wo[at] = __ldg(w + i);
    }
    s_seen += __popc(ms), e_seen += __popc(me);
  }
  const int mine = all_sure + min(max(want - cta_equal, 0), all_equal);
  if (rank + 1 == size)
    for (int i = base + mine + tid; i < keep; i += kEvictThreads) {
      io[i] = -1;
      if (wo) wo[i] = 0.f;
    }
  __syncthreads();  // io is read below by other threads of the CTA
  // The rows: units of 16 bytes, U of K's codes, U of V's, and their steps and bases (d = 64: 8 bytes each, by words).
  constexpr int U = D / 32;
  const long long from0 = static_cast<long long>(bh) * src.cap, to0 = static_cast<long long>(bh) * dst.cap;
  const uint4 *sk = reinterpret_cast<const uint4*>(src.k), *sv = reinterpret_cast<const uint4*>(src.v);
  uint4 *dk = reinterpret_cast<uint4*>(dst.k), *dv = reinterpret_cast<uint4*>(dst.v);
  constexpr int kBatch = 2;  // units in flight a thread; of its registers, 32, they take 20
  #pragma unroll 1
  for (int x0 = tid; x0 < mine * U; x0 += kBatch * kEvictThreads) {
    long long from[kBatch];
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int x = x0 + i * kEvictThreads;
      from[i] = x < mine * U ? (from0 + io[base + x / U]) * U + x % U : 0;
    }
    uint4 k[kBatch], v[kBatch];
    uint32_t ks[kBatch], vs[kBatch];
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (x0 + i * kEvictThreads >= mine * U) continue;
      k[i] = __ldg(sk + from[i]), v[i] = __ldg(sv + from[i]);
      ks[i] = __ldg(src.ks + from[i]), vs[i] = __ldg(src.vs + from[i]);
    }
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int x = x0 + i * kEvictThreads;
      if (x >= mine * U) continue;
      const long long to = (to0 + base) * U + x;
      dk[to] = k[i], dv[to] = v[i];
      dst.ks[to] = ks[i], dst.vs[to] = vs[i];
    }
  }
  if (size > 1) cluster_sync();  // no CTA leaves while another may read its counts
}

}  // namespace vmlm
