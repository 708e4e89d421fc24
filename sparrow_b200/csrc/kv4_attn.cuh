// kv4_attn.cuh -- attention of the newest tokens over a 4-bit cache.
//
// Token t of the m newest of sequence b sees the slots j < len[b] - (m - 1 - t):
//   s_j = scale * q . k_j,  p = softmax(s),  out = sum_j p_j v_j
// (no slot visible: out = 0), and, where asked for, the weight that each slot
// received: w_out[j] = w_in[j] + the sum of p_j over the m tokens and over the
// query heads that share the kv head (w_in counts as 0 for the m newest slots).
//
// Floor: 1.25 d bytes a slot and kv head. At 6.5 TB/s an SM has 6.5 cycles for
// a slot of d = 128, in which 256 nibbles become halves and are multiplied with
// every query row of the group: on CUDA cores the products alone would take
// that long for two rows, so they run on the tensor cores, straight from the
// registers in which the halves are made (mma.sync m16n8k16; tcgen05 would take
// its operands through shared memory, four times the bytes of the codes).
//
// Both products have the cached values as A, 16 rows each, and the query rows
// as the 8 columns of B: four rows, each split in two halves x = hi + lo, whose
// products with a cached half are exact, so both products are f32 to 22 bits.
//   scores  S^T[slot][row]  = K[slot][d] . q[d][row]     A rows: slots
//   output  O^T[d][row]     = V^T[d][slot] . P[slot][row] A rows: columns of V
// V^T comes without a transpose: A's register holds one column of two slots,
// and one PRMT pairs the halves of two slots' code words, after which a shift
// and a LOP3 give both slots' nibbles of one column. Which column of V is which
// row of A, and which column of K and q is which k, is free, and chosen so that
// each lane takes whole words. S^T leaves the tensor core with a row's hi and lo
// sums in one lane; P goes back through movmatrix, an 8 x 8 transpose.
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
  float* score;       // [n_seq][n_kv][rows][cap]: log2 of the unnormalised weights (w_out only)
  float* lse;         // [n_seq][n_kv][rows]: log2 of their sum
  float* part;        // two partial results a CTA: m, l, O of a chunk of rows
  int* arrived;       // [n_seq][n_kv][chunks]: partial results written, zero between calls
  float scale2;       // scale * log2(e)
  int m, n_q, group, rows, chunks;  // rows = m * group query rows a kv head, in chunks
  int min_units;      // work of a CTA, in units of kAttnUnit slots, below which fewer CTAs are used
  int vec;            // q rows start on 16-byte boundaries
};

constexpr int kAttnWarps = 8;
constexpr int kAttnUnit = 64;            // slots: the grain in which work is shared out
constexpr int kAttnStageBytes = 5120;    // 4096 values of K and of V with their steps and bases
constexpr float kAttnShift = 14.f;       // weights are held as 2^14 times their value, so that their halves keep 2^-25 of 2^-14
constexpr float kAttnSlack = 1.f;        // a running maximum may lag by this (log2): 2^15 is still a half

// Dynamic shared memory: the warps' rings, then the merge buffer.
__host__ __device__ constexpr int attn_merge_floats(int D, int NT) {
  return kAttnWarps * NT * 4 * (NT * D > 128 ? D / 2 : D);
}
__host__ __device__ constexpr int attn_smem_bytes(int D, int NT) {
  return kAttnWarps * 2 * kAttnStageBytes + attn_merge_floats(D, NT) * 4 + kAttnWarps * NT * 4 * 8;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: the destination is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool on) {
  const int n = on ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// Nibble I (0..3) of both 16-bit halves of u as the halves of their values.
template <int I>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t u, __half2 step, __half2 base) {
  const uint32_t t = I == 0 ? u << 6 : I == 1 ? u << 2 : I == 2 ? u >> 2 : u >> 6;
  return h2_bits(__hfma2(bits_h2((t & 0x03C003C0u) | 0x4C004C00u), step, base));
}
__device__ __forceinline__ uint32_t kv4_pair_at(int i, uint32_t u, __half2 step, __half2 base) {
  return i == 0 ? kv4_pair<0>(u, step, base) : i == 1 ? kv4_pair<1>(u, step, base)
       : i == 2 ? kv4_pair<2>(u, step, base) : kv4_pair<3>(u, step, base);
}

// Where a slot's 16-byte chunk c of codes lies in its row in shared memory: the
// K reads (two rows, all chunks) and the V reads (four even rows, two chunks) of
// a quarter or half warp then meet in no bank (d = 256) or in pairs.
template <int D>
__device__ __forceinline__ int attn_swizzle(int slot, int c) {
  if constexpr (D == 256) return c ^ (slot & 7);
  if constexpr (D == 128) return c ^ ((slot >> 1) & 3);
  return c;
}

// A run of slots [s0, s1) of one item (sequence, kv head, chunk of rows).
struct AttnSeg {
  int b, hc;          // sequence, kv head * chunks + chunk
  int s0, s1, n;      // n: the sequence's length
  long long first;    // the item's first unit
  int units;          // the item's units
  bool whole;         // the run is the whole item
};

// Walks the runs of one CTA: units [pos, end) of all items in order of
// sequence, kv head and chunk. Every warp walks alone and sees the same.
struct AttnWalk {
  const int32_t* len;
  int n_seq, hc_count;
  long long cap, pos, end, base;  // base: the first unit of sequence b
  int b;

  __device__ __forceinline__ int length(int i) const {
    const long long n = __ldg(len + i);
    return static_cast<int>(n > cap ? cap : n < 0 ? 0 : n);
  }
  __device__ __forceinline__ bool next(AttnSeg& s) {
    if (pos >= end) return false;
    int n, u;
    while (true) {
      n = length(b);
      u = (n + kAttnUnit - 1) / kAttnUnit;
      const long long all = static_cast<long long>(u) * hc_count;
      if (pos < base + all) break;
      base += all;
      ++b;
    }
    const long long at = pos - base;
    s.b = b;
    s.hc = static_cast<int>(at / u);
    const int off = static_cast<int>(at - static_cast<long long>(s.hc) * u);
    const long long left = end - pos;
    const int take = static_cast<int>(left < u - off ? left : u - off);
    s.n = n;
    s.s0 = off * kAttnUnit;
    s.s1 = min(n, (off + take) * kAttnUnit);
    s.first = pos - off;
    s.units = u;
    s.whole = take == u;
    pos += take;
    return true;
  }
};

// D: head size. NT: chunks hold 4 * NT rows. kW: scores are kept for w_out.
template <int D, int NT, bool kW>
__global__ void __launch_bounds__(kAttnWarps * 32, 2) kv4_attn_kernel(const Kv4Attn p, const Kv4View c,
                                                                       int* __restrict__ err) {
  constexpr int TS = 4096 / D;      // slots of a tile
  constexpr int ST = TS / 16;       // its 16-slot steps
  constexpr int KW = D / 32;        // code words of a K row that a lane takes
  constexpr int VW = D / 64;        // code words of a V row that a lane takes
  constexpr int RC = 4 * NT;        // rows of a chunk
  constexpr int OT = D / 16;        // 16-column tiles of the output
  constexpr int kCh = D / 32;       // 16-byte chunks of a row of codes
  constexpr int kHalves = NT * D > 128 ? 2 : 1;  // the merge buffer holds this part of the output at a time
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  unsigned char* ring = smem + warp * 2 * kAttnStageBytes;
  float* merge = reinterpret_cast<float*>(smem + kAttnWarps * 2 * kAttnStageBytes);
  float* ml = merge + attn_merge_floats(D, NT);  // [warp][row][m, l]
  __shared__ int s_last;

  // All units, and this CTA's share of them.
  AttnWalk walk;
  walk.len = p.len, walk.n_seq = c.n_seq, walk.hc_count = c.n_kv * p.chunks, walk.cap = c.cap;
  long long units = 0;
  for (int i = lane; i < c.n_seq; i += 32) {
    if (__ldg(p.len + i) > c.cap && tid == lane) atomicCAS(err, 0, kDevKv4Slot);
    units += (walk.length(i) + kAttnUnit - 1) / kAttnUnit;
  }
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
  units *= walk.hc_count;
  const long long want = units / p.min_units;
  const int ctas = static_cast<int>(want < 1 ? 1 : want < gridDim.x ? want : gridDim.x);
  const int cta = blockIdx.x;

  // Sequences without a slot: zeros.
  for (int i = cta; i < c.n_seq; i += gridDim.x) {
    if (walk.length(i) > 0) continue;
    for (long long x = tid; x < static_cast<long long>(p.m) * p.n_q * D; x += kAttnWarps * 32) {
      const long long t = x / (p.n_q * D);
      p.out[(static_cast<long long>(i) * p.m + t) * p.ldo + (x - t * p.n_q * D)] = 0.f;
    }
  }
  if (cta >= ctas) return;
  walk.pos = units * cta / ctas;
  walk.end = units * (cta + 1) / ctas;
  walk.b = 0, walk.base = 0;

  // The part of a run that this warp takes, and its first tile's loads.
  auto share = [&](const AttnSeg& s, int& w0, int& w1) {
    const int per = ((s.s1 - s.s0 + kAttnWarps - 1) / kAttnWarps + 15) & ~15;
    w0 = min(s.s1, s.s0 + warp * per);
    w1 = min(s.s1, w0 + per);
  };
  auto fetch = [&](const AttnSeg& s, int at, int end, int stage) {
    const int head = s.hc / p.chunks;
    const long long row = (static_cast<long long>(s.b) * c.n_kv + head) * c.cap + at;
    const uint32_t dst = smem_u32(ring + stage * kAttnStageBytes);
    const int left = end - at;  // rows of the tile that exist
    const uint8_t *k = c.k + row * (D / 2), *v = c.v + row * (D / 2);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = lane + 32 * i, slot = x / kCh, ch = x % kCh;
      const uint32_t to = slot * (D / 2) + attn_swizzle<D>(slot, ch) * 16;
      const long long from = slot < left ? x * 16 : 0;
      cp_async16(dst + to, k + from, slot < left);
      cp_async16(dst + 2048 + to, v + from, slot < left);
    }
    const uint8_t *ks = reinterpret_cast<const uint8_t*>(c.ks) + row * (D / 8);
    const uint8_t *vs = reinterpret_cast<const uint8_t*>(c.vs) + row * (D / 8);
    if constexpr (D == 64) {  // 8 bytes a row: no more alignment than that
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int x = lane + 32 * i;
        cp_async8(dst + 4096 + x * 8, ks + (x < left ? x * 8 : 0), x < left);
        cp_async8(dst + 4608 + x * 8, vs + (x < left ? x * 8 : 0), x < left);
      }
    } else {
      const int slot = lane * 16 / (D / 8);
      cp_async16(dst + 4096 + lane * 16, ks + (slot < left ? lane * 16 : 0), slot < left);
      cp_async16(dst + 4608 + lane * 16, vs + (slot < left ? lane * 16 : 0), slot < left);
    }
  };

  AttnSeg seg, nxt;
  if (!walk.next(seg)) return;
  int w0, w1;
  share(seg, w0, w1);
  if (w0 < w1) fetch(seg, w0, w1, 0);
  cp_async_commit();
  int stage = 0;

  while (true) {
    const bool more = walk.next(nxt);
    int x0 = 0, x1 = 0;
    if (more) share(nxt, x0, x1);
    const int head = seg.hc / p.chunks, r0 = (seg.hc - head * p.chunks) * RC;

    // The chunk's rows: B fragments of their halves, a power of two apart from
    // the row so that its largest value lies in [1, 2). Lane (gid, tig) has row
    // gid / 2 of each four, hi for even gid and lo for odd.
    uint32_t qb[NT][2 * KW][2];
    float sc[NT];  // what a score has to be multiplied by (log2 units), of row tig
    int vis[NT];   // slots that row tig sees
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + nt * 4 + (gid >> 1);
      float x[D / 4];
      if (r < p.rows) {
        const int t = r / p.group;
        const float* src = p.q + (static_cast<long long>(seg.b) * p.m + t) * p.ldq +
                           static_cast<long long>(head * p.group + r - t * p.group) * D + tig * (D / 4);
        load_row<D / 4>(src, p.vec, x);
      } else {
        #pragma unroll
        for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
      }
      float top = 0.f;
      #pragma unroll
      for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max(static_cast<int>((__float_as_uint(top) >> 23) & 255) - 127, -120), 120);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      sc[nt] = __shfl_sync(0xffffffffu, __uint_as_float(static_cast<uint32_t>(127 + e) << 23), 8 * tig) * p.scale2;
      #pragma unroll
      for (int w = 0; w < KW; ++w) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = x[8 * w + i] * down, b = x[8 * w + i + 4] * down;
          const __half2 hi = __floats2half2_rn(a, b);
          const __half2 lo = __floats2half2_rn(a - __low2float(hi), b - __high2float(hi));
          qb[nt][2 * w + (i >> 1)][i & 1] = (gid & 1) ? h2_bits(lo) : h2_bits(hi);
        }
      }
      const int rt = r0 + nt * 4 + tig;
      vis[nt] = rt < p.rows ? seg.n - (p.m - 1 - rt / p.group) : 0;
    }

    float top[NT], sum[NT], o[OT][2][NT];
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      top[nt] = -1e30f, sum[nt] = 0.f;
      #pragma unroll
      for (int i = 0; i < OT; ++i) o[i][0][nt] = 0.f, o[i][1][nt] = 0.f;
    }

    int at = w0;
    do {
      if (at + TS < w1) {
        fetch(seg, at + TS, w1, stage ^ 1);
      } else if (more && x0 < x1) {
        fetch(nxt, x0, x1, stage ^ 1);
      }
      cp_async_commit();
      cp_async_wait<1>();
      __syncwarp();
      const unsigned char* st = ring + stage * kAttnStageBytes;
      const int left = w1 - at;
      if (left > 0) {
        // scores, in log2 units
        float s[ST][2][NT];
        #pragma unroll
        for (int u = 0; u < ST; ++u) {
          float acc[NT][4];
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
          if (u * 16 < left) {
            const int ja = u * 16 + gid, jb = ja + 8;
            uint32_t wa[KW], wb[KW];
            if constexpr (D == 64) {
              const uint2 a = *reinterpret_cast<const uint2*>(st + ja * 32 + tig * 8);
              const uint2 b = *reinterpret_cast<const uint2*>(st + jb * 32 + tig * 8);
              wa[0] = a.x, wa[1] = a.y, wb[0] = b.x, wb[1] = b.y;
            } else {
              #pragma unroll
              for (int h = 0; h < KW / 4; ++h) {
                const int ch = tig * (KW / 4) + h;
                const uint4 a = *reinterpret_cast<const uint4*>(st + ja * (D / 2) + attn_swizzle<D>(ja, ch) * 16);
                const uint4 b = *reinterpret_cast<const uint4*>(st + jb * (D / 2) + attn_swizzle<D>(jb, ch) * 16);
                wa[4 * h] = a.x, wa[4 * h + 1] = a.y, wa[4 * h + 2] = a.z, wa[4 * h + 3] = a.w;
                wb[4 * h] = b.x, wb[4 * h + 1] = b.y, wb[4 * h + 2] = b.z, wb[4 * h + 3] = b.w;
              }
            }
            const uint32_t* sb = reinterpret_cast<const uint32_t*>(st + 4096);
            #pragma unroll
            for (int w = 0; w < KW; ++w) {
              const int g = D == 64 ? tig >> 1 : tig * (KW / 4) + w / 4;
              const __half2 sa = bits_h2(sb[ja * (D / 32) + g]), sbb = bits_h2(sb[jb * (D / 32) + g]);
              __half2 ha[4], hb[4];
              kv4_unpack(wa[w], __low2half2(sa), __high2half2(sa), ha);
              kv4_unpack(wb[w], __low2half2(sbb), __high2half2(sbb), hb);
              #pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16(acc[nt], h2_bits(ha[0]), h2_bits(hb[0]), h2_bits(ha[1]), h2_bits(hb[1]), qb[nt][2 * w][0],
                        qb[nt][2 * w][1]);
                mma_f16(acc[nt], h2_bits(ha[2]), h2_bits(hb[2]), h2_bits(ha[3]), h2_bits(hb[3]), qb[nt][2 * w + 1][0],
                        qb[nt][2 * w + 1][1]);
              }
            }
          }
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            s[u][0][nt] = (acc[nt][0] + acc[nt][1]) * sc[nt];
            s[u][1][nt] = (acc[nt][2] + acc[nt][3]) * sc[nt];
          }
        }
        if (kW) {
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int r = r0 + nt * 4 + tig;
            if (r < p.rows) {
              float* to = p.score + ((static_cast<long long>(seg.b) * c.n_kv + head) * p.rows + r) * c.cap + at;
              #pragma unroll
              for (int u = 0; u < ST; ++u) {
                if (u * 16 + gid < left) to[u * 16 + gid] = s[u][0][nt];
                if (u * 16 + gid + 8 < left) to[u * 16 + gid + 8] = s[u][1][nt];
              }
            }
          }
        }
        // slots that a row does not see; then the running maximum
        uint32_t pb[ST][NT][2];
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int see = min(left, vis[nt] - at);
          if (__any_sync(0xffffffffu, see < TS)) {
            #pragma unroll
            for (int u = 0; u < ST; ++u) {
              if (u * 16 + gid >= see) s[u][0][nt] = -INFINITY;
              if (u * 16 + gid + 8 >= see) s[u][1][nt] = -INFINITY;
            }
          }
          float best = s[0][0][nt];
          #pragma unroll
          for (int u = 0; u < ST; ++u) best = fmaxf(best, fmaxf(s[u][0][nt], s[u][1][nt]));
          if (__any_sync(0xffffffffu, best > top[nt] + kAttnSlack)) {
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 8));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 16));
            best = fmaxf(best, top[nt]);
            const float f = ex2(top[nt] - best);
            top[nt] = best;
            sum[nt] *= f;
            #pragma unroll
            for (int i = 0; i < OT; ++i) o[i][0][nt] *= f, o[i][1][nt] *= f;
          }
          const float off = kAttnShift - top[nt];
          #pragma unroll
          for (int u = 0; u < ST; ++u) {
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float e = ex2(s[u][h][nt] + off);
              sum[nt] += e;
              const float hi = __uint_as_float(__float_as_uint(e) & 0xFFFFE000u);
              pb[u][nt][h] = transpose8x8(h2_bits(__floats2half2_rn(hi, e - hi)));
            }
          }
        }
        // output: nibble by nibble of the V words
        const unsigned char* sv = st + 2048;
        const uint32_t* sb = reinterpret_cast<const uint32_t*>(st + 4608);
        uint32_t ul[ST][2][VW], uh[ST][2][VW];  // low and high 16 bits of two slots' words
        __half2 stp[ST][2], bas[ST][2];
        #pragma unroll
        for (int u = 0; u < ST; ++u) {
          #pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ja = u * 16 + 8 * h + 2 * tig, jb = ja + 1;
            uint32_t wa[VW], wb[VW];
            const int byte = gid * VW * 4, ch = byte / 16, in = byte % 16;
            const unsigned char* pa = sv + ja * (D / 2) + attn_swizzle<D>(ja, ch) * 16 + in;
            const unsigned char* pq = sv + jb * (D / 2) + attn_swizzle<D>(jb, ch) * 16 + in;
            if constexpr (VW == 1) {
              wa[0] = *reinterpret_cast<const uint32_t*>(pa), wb[0] = *reinterpret_cast<const uint32_t*>(pq);
            } else if constexpr (VW == 2) {
              const uint2 a = *reinterpret_cast<const uint2*>(pa), b = *reinterpret_cast<const uint2*>(pq);
              wa[0] = a.x, wa[1] = a.y, wb[0] = b.x, wb[1] = b.y;
            } else {
              const uint4 a = *reinterpret_cast<const uint4*>(pa), b = *reinterpret_cast<const uint4*>(pq);
              wa[0] = a.x, wa[1] = a.y, wa[2] = a.z, wa[3] = a.w;
              wb[0] = b.x, wb[1] = b.y, wb[2] = b.z, wb[3] = b.w;
            }
            #pragma unroll
            for (int w = 0; w < VW; ++w) {
              ul[u][h][w] = __byte_perm(wa[w], wb[w], 0x5410);
              uh[u][h][w] = __byte_perm(wa[w], wb[w], 0x7632);
            }
            const int g = gid * VW / 4;
            const uint32_t x = sb[ja * (D / 32) + g], y = sb[jb * (D / 32) + g];
            stp[u][h] = bits_h2(__byte_perm(x, y, 0x5410));
            bas[u][h] = bits_h2(__byte_perm(x, y, 0x7632));
          }
        }
        #pragma unroll
        for (int i = 0; i < OT; ++i) {
          float acc[NT][4];
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
          #pragma unroll
          for (int u = 0; u < ST; ++u) {
            if (u * 16 < left) {
              uint32_t a[4];
              #pragma unroll
              for (int h = 0; h < 2; ++h) {
                if constexpr (VW == 1) {  // tile i: columns 8 gid + i and 8 gid + 4 + i
                  a[2 * h] = kv4_pair_at(i, ul[u][h][0], stp[u][h], bas[u][h]);
                  a[2 * h + 1] = kv4_pair_at(i, uh[u][h][0], stp[u][h], bas[u][h]);
                } else {  // tile (pair, n): columns n of words 2 pair and 2 pair + 1 of the lane's words
                  const int w = i / 8 * 2, n = i % 8;
                  a[2 * h] = kv4_pair_at(n & 3, n < 4 ? ul[u][h][w] : uh[u][h][w], stp[u][h], bas[u][h]);
                  a[2 * h + 1] = kv4_pair_at(n & 3, n < 4 ? ul[u][h][w + 1] : uh[u][h][w + 1], stp[u][h], bas[u][h]);
                }
              }
              #pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt], a[0], a[1], a[2], a[3], pb[u][nt][0], pb[u][nt][1]);
            }
          }
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            o[i][0][nt] += acc[nt][0] + acc[nt][1];
            o[i][1][nt] += acc[nt][2] + acc[nt][3];
          }
        }
      }
      __syncwarp();
      stage ^= 1;
      at += TS;
    } while (at < w1);

    // The warps' results become one: largest maximum, then scaled sums.
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      #pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum[nt] += __shfl_xor_sync(0xffffffffu, sum[nt], x);
      if (gid == 0) {
        ml[(warp * RC + nt * 4 + tig) * 2] = top[nt];
        ml[(warp * RC + nt * 4 + tig) * 2 + 1] = sum[nt];
      }
    }
    const long long item = static_cast<long long>(seg.b) * walk.hc_count + seg.hc;
    const bool starts = seg.s0 == 0;
    float* part = p.part + (static_cast<long long>(cta) * 2 + (starts ? 1 : 0)) * (RC * (D + 2));
    #pragma unroll
    for (int hv = 0; hv < kHalves; ++hv) {
      constexpr int OH = OT / kHalves;
      __syncthreads();
      #pragma unroll
      for (int i = 0; i < OH; ++i)
        #pragma unroll
        for (int h = 0; h < 2; ++h)
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            merge[((warp * OH + i) * 2 + h) * NT * 32 + nt * 32 + lane] = o[hv * OH + i][h][nt];
      __syncthreads();
      for (int x = tid; x < RC * D / kHalves; x += kAttnWarps * 32) {
        // x -> (row, a column of this part): lanes take neighbouring columns
        const int r = x / (D / kHalves), y = x % (D / kHalves);
        int col, ti, h, g;
        if constexpr (D == 64) {
          constexpr int per = 8 / kHalves;  // columns of a lane's word in this part
          g = y / per;
          const int z = y % per;            // (h, i within the part)
          h = z / OH, ti = z % OH;
          col = 8 * g + 4 * h + hv * OH + ti;
        } else {
          constexpr int words = VW / kHalves > 1 ? VW / kHalves : 1;  // words of a lane in this part
          if constexpr (VW / kHalves >= 2) {
            const int w = y / 8, n = y % 8;
            g = w / words;
            const int ww = w % words;
            h = ww & 1, ti = ww / 2 * 8 + n;
            col = 8 * (g * VW + hv * words + ww) + n;
          } else {  // d = 128 in two parts: nibbles 4 hv .. 4 hv + 3 of both words
            const int w = y / 4, n = y % 4;
            g = w / 2, h = w & 1, ti = n;
            col = 8 * (g * VW + h) + 4 * hv + n;
          }
        }
        float m = -1e30f;
        #pragma unroll
        for (int k = 0; k < kAttnWarps; ++k) m = fmaxf(m, ml[(k * RC + r) * 2]);
        float v = 0.f, l = 0.f;
        #pragma unroll
        for (int k = 0; k < kAttnWarps; ++k) {
          const float f = ex2(ml[(k * RC + r) * 2] - m);
          l = fmaf(f, ml[(k * RC + r) * 2 + 1], l);
          v = fmaf(f, merge[((k * OH + ti) * 2 + h) * NT * 32 + (r >> 2) * 32 + g * 4 + (r & 3)], v);
        }
        const int row = r0 + r;
        if (seg.whole) {
          if (row < p.rows) {
            const int t = row / p.group;
            p.out[(static_cast<long long>(seg.b) * p.m + t) * p.ldo +
                  static_cast<long long>(head * p.group + row - t * p.group) * D + col] = l != 0.f ? v / l : 0.f;
            if (kW && col == 0)
              p.lse[(static_cast<long long>(seg.b) * c.n_kv + head) * p.rows + row] = m - kAttnShift + log2f(l);
          }
        } else {
          part[2 * RC + r * D + col] = v;
          if (col == 0) part[r] = m, part[RC + r] = l;
        }
      }
    }
    if (!seg.whole) {
      // The CTA that finds every other part of the item written joins them.
      __threadfence();
      __syncthreads();
      const long long last_unit = seg.first + seg.units - 1;
      const int c0 = static_cast<int>(((seg.first + 1) * ctas - 1) / units);
      const int c1 = static_cast<int>(((last_unit + 1) * ctas - 1) / units);
      if (tid == 0) s_last = atom_add_acq_rel_gpu(p.arrived + item, 1) == c1 - c0;
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int x = tid; x < RC * D; x += kAttnWarps * 32) {
          const int r = x / D, col = x % D, row = r0 + r;
          if (row >= p.rows) continue;
          float m = -1e30f, v = 0.f, l = 0.f;
          for (int k = c0; k <= c1; ++k) {
            const float* from = p.part + (static_cast<long long>(k) * 2 + (k == c0 ? 1 : 0)) * (RC * (D + 2));
            const float mk = __ldcg(from + r), lk = __ldcg(from + RC + r), vk = __ldcg(from + 2 * RC + r * D + col);
            const float mm = fmaxf(m, mk), f = ex2(m - mm), fk = ex2(mk - mm);
            l = fmaf(l, f, lk * fk), v = fmaf(v, f, vk * fk), m = mm;
          }
          const int t = row / p.group;
          p.out[(static_cast<long long>(seg.b) * p.m + t) * p.ldo +
                static_cast<long long>(head * p.group + row - t * p.group) * D + col] = l != 0.f ? v / l : 0.f;
          if (kW && col == 0)
            p.lse[(static_cast<long long>(seg.b) * c.n_kv + head) * p.rows + row] = m - kAttnShift + log2f(l);
        }
        if (tid == 0) p.arrived[item] = 0;
      }
    }
    if (!more) break;
    __syncthreads();  // ml and merge are read before the next run writes them
    seg = nxt, w0 = x0, w1 = x1;
  }
  cp_async_wait<0>();
}

// The weights from the kept scores: one thread per (sequence, kv head, slot).
__global__ void __launch_bounds__(256) kv4_weights_kernel(const Kv4Attn p, const Kv4View c) {
  const long long j = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long bh = blockIdx.y;
  const long long b = bh / c.n_kv;
  long long n = __ldg(p.len + b);
  if (n > c.cap) n = c.cap;
  if (j >= n) return;
  float w = 0.f;
  const float* s = p.score + bh * p.rows * c.cap + j;
  for (int r = 0; r < p.rows; ++r)
    if (j < n - (p.m - 1 - r / p.group)) w += ex2(__ldg(s + r * c.cap) - __ldg(p.lse + bh * p.rows + r));
  const long long at = bh * c.cap + j;
  p.w_out[at] = (p.w_in && j < n - p.m ? p.w_in[at] : 0.f) + w;
}

}  // namespace vmlm
