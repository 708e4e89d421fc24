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
// and one PRMT pairs the bytes of two slots' code words, after which a LOP3 and
// a multiply-add give both slots' nibbles of one column. Which column of V is which
// row of A, and which column of K and q is which k, is free, and chosen so that
// each lane takes whole words. S^T leaves the tensor core with a row's hi and lo
// sums in one lane; P goes back through movmatrix, an 8 x 8 transpose.
//
// Measured: 8 kv heads of 4 rows, d = 128, 131071 slots: 41.3 us = 4.1 TB/s of codes; 48 ragged sequences of up to 8192
// slots: 56.2 us = 4.5 TB/s; 36 heads of one row, d = 64, 777 slots: 8.3 us, of which 2 are the launch and the loads'
// latency most of the rest. With few rows the loads in flight bound it (two tiles a warp), with many the instructions of
// the softmax: about 25 for two scores a lane.
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
  float* score;       // [n_seq][n_kv][chunks][kept_rows][cap]: log2 of the unnormalised weights (w_out only)
  float2* norm;       // [n_seq][n_kv][rows]: what is added to a score to be the exponent of a weight, 1 / the weights' sum
  float* part;        // two partial results a CTA: m, l, O of a chunk of rows
  int2* split;        // [n_seq][n_kv][chunks]: the first CTA of an item and how many have a part of it (one: the output is there)
  float scale_m;      // scale * log2(e) = scale_m * 2^scale_e, 1 <= |scale_m| < 2 (or 0, or not finite)
  int scale_e;
  int m, n_q, group, rows;  // rows = m * group query rows a kv head
  int chunks, chunk_rows;   // in chunks of a multiple of 4
  int kept_rows;            // of a chunk among the kept scores: chunk_rows and what a kernel rounds them up to
  int alone;          // few and short items get a CTA each: up to how many tiles
  int vec;            // q rows start on 16-byte boundaries
  uint32_t mul4, mul64;  // 4 and 64, as values that the compiler does not know: see kv4_pair
};

constexpr int kAttnStageBytes = 5120;    // 4096 values of K and of V with their steps and bases
// A row's weights are 2^(score - top), in log2 units. top is the integer from 13 to 14 below the running maximum, so the largest
// weight lies between 2^13 and 2^14 and halves keep 2^-38 of it, or up to 2^15, still a half, before top is moved. Integers,
// so that differences of tops, and what one part's weights are multiplied by to join another's, are exact; and where
// scores are so large (2^24) that f32 has no such integer, top is rounded up: a weight then is smaller, never above 2^15.
constexpr float kAttnBelow = 14.f, kAttnRoom = 15.f;
constexpr float kAttnNone = -3.402823466e38f;  // of no scores: finite, so that what joins parts is a number
__device__ __forceinline__ float attn_top(float best) { return __fadd_ru(ceilf(best), -kAttnBelow); }
__device__ __forceinline__ float attn_limit(float top) { return __fadd_rd(top, kAttnRoom); }  // scores above it move top
constexpr int kAttnAlone = 4;            // tiles a warp up to which a CTA may take an item alone

// Warps of the one CTA on an SM. A chunk of rows takes D/8 registers a four rows
// for its queries and as many for its output: 4 rows of d = 64 or 128 fit 128
// registers (16 warps), of d = 256 168 (12 warps; 8: 139 us against 134 for 8 rows
// over 16 x 8 heads of 8192 slots). More rows run best with 8 warps of 255
// registers, whose instructions overlap instead of the warps (d = 64, 33 rows, weights
// kept: 56 us against 60 with 12 warps).
__host__ __device__ constexpr int attn_warps(int D, int NT) { return NT > 1 ? 8 : D == 256 ? 12 : 16; }
// Fours of rows that a chunk holds at most.
__host__ __device__ constexpr int attn_most(int D) { return D == 64 ? 4 : D == 128 ? 2 : 1; }
constexpr int kAttnManyRows = 25;  // d = 256: rows from which a CTA shares what it unpacks
// Dynamic shared memory: the warps' rings, a partial result and two (m, l) lists a warp.
__host__ __device__ constexpr int attn_smem_bytes(int D, int NT) {
  return attn_warps(D, NT) * (2 * kAttnStageBytes + 4 * NT * D * 4 + 2 * 4 * NT * 8);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
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
// The same with a zero accumulator: no registers to clear.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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

// The low (kHigh = false) or high nibbles of bits 0..7 of both halves of u as the halves of their values. The mask keeps
// the nibble where it is and a multiply-add moves it to the mantissa's top and puts 16.0 under it: one LOP3 and two
// operations of the FMA pipe for two values. With a shift and a LOP3 instead, three of four operations are the ALU
// pipe's, and it was the first to fill up (58% busy at 131071 slots, 32/8 heads of 128, where the FMA pipe had 20%).
// The factors come from the caller: a constant power of two would be turned into a shift on the ALU pipe.
template <bool kHigh>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t u, uint32_t mul, __half2 step, __half2 base) {
  const uint32_t t = (u & (kHigh ? 0x00F000F0u : 0x000F000Fu)) * mul + 0x4C004C00u;  // mul: 4 (high) or 64
  return h2_bits(__hfma2(bits_h2(t), step, base));
}

// Values of slots that some rows of a chunk see and others do not. A hidden slot's weight is 0, but 0 times a NaN or an
// infinity is NaN, and a product takes a slot's values for all rows: where values of one slot and group of 32 columns are
// not finite (as the smallest and the largest code have it), their step and base become zeros in shared memory, and the
// rows that see them get them by scalar operations once the tile is done. This is looked for only in tiles that a row of
// the chunk sees in part, and there first by a test that all usual values pass: a step below 1024, a base below 32768.
__device__ __forceinline__ bool kv4_large(uint32_t sb) { return (((sb & 0x7FFF7FFFu) + 0x08001C00u) & 0x80008000u) != 0; }
__device__ __forceinline__ bool kv4_infinite(uint32_t sb) {
  const __half2 step = __low2half2(bits_h2(sb)), base = __high2half2(bits_h2(sb));
  const uint32_t x = h2_bits(__hfma2(__floats2half2_rn(16.f, 31.f), step, base)) & 0x7C007C00u;
  return (x & 0x7C00u) == 0x7C00u || x >> 16 == 0x7C00u;
}
__device__ __forceinline__ float kv4_value(uint32_t word, int nibble, uint32_t sb) {
  const __half2 x = bits_h2(sb);
  return __half2float(__hfma(__float2half_rn(16.f + static_cast<float>(word >> 4 * nibble & 15u)), __low2half(x), __high2half(x)));
}
// A weight from its halves: slot `odd` of two in the fragments of a row's hi and lo.
__device__ __forceinline__ float kv4_weight(uint32_t hi, uint32_t lo, int odd) {
  return odd ? __high2float(bits_h2(hi)) + __high2float(bits_h2(lo)) : __low2float(bits_h2(hi)) + __low2float(bits_h2(lo));
}

// A query row as B fragments of its halves: the row times the scale, a power of two apart from that so that its largest value
// lies in [1, 4). Lane (gid, tig) has columns tig * D/4 .. of row gid / 2 of four: hi for even gid, lo for odd. Returns the
// power of two that a score has to be multiplied by to be in log2 units, exactly.
template <int D>
__device__ __forceinline__ float attn_query(const float* src, bool vec, float scale_m, int scale_e, uint32_t (&qb)[D / 16][2]) {
  const int gid = (threadIdx.x & 31) >> 2, tig = threadIdx.x & 3;
  float x[D / 4];
  if (src) {
    load_row<D / 4>(src + tig * (D / 4), vec, x);
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
  const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * scale_m;
  #pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[8 * w + i] * down, b = x[8 * w + i + 4] * down;
      const __half2 hi = __floats2half2_rn(a, b);
      const __half2 lo = __floats2half2_rn(a - __low2float(hi), b - __high2float(hi));
      qb[2 * w + (i >> 1)][i & 1] = (gid & 1) ? h2_bits(lo) : h2_bits(hi);
    }
  }
  // not 0, or a hidden slot's -inf would become a NaN
  return __uint_as_float(static_cast<uint32_t>(min(max(e + scale_e, -126), 127) + 127) << 23);
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

// The work is the tiles of TS = 4096 / d slots of every item (sequence, kv head,
// chunk of rows), in that order, in equal contiguous shares for the CTAs and,
// within a CTA, for its warps, whatever the lengths are: a warp's share is a few
// runs, each a part of an item or all of it. Few and short items (at most one a
// CTA, of at most p.alone tiles) get a CTA each instead, where sharing would save
// no more than a tile a warp: the join of parts across CTAs costs as much. d = 64,
// one row: 144 items of 4096 slots take 18.0 us alone and 19.3 shared, 36 items of
// 4096 slots 16.3 alone and 11.5 shared.
struct AttnRun {
  int b, hc;          // sequence, kv head * chunks + chunk
  int head, r0;       // kv head, the chunk's first row
  int s0, s1, n;      // slots [s0, s1) of the n of the sequence
  int first, units;   // where the item's tiles begin among all units, and how many they are
  bool enter, leave;  // the item has tiles before, behind this run
};

// The shares are counted in units: an item is its tiles, and before them `cost` units for what a run costs besides
// (its queries and its result), so that short items do not gather in one share.
// Of a warp here. 16 ragged sequences of up to 4000 slots, 8 x 8 heads of 128: 28.5 us with 1, 23.9 with 2, 23.4 with 3; 64 of
// up to 1000, 2 x 4 heads of 256: 19.6, 18.0, 17.8; 200 of up to 600, 8 heads of 64: 23.6, 23.9, 25.2.
constexpr int kAttnRunCost = 2;

template <int TS, int kCost>
struct AttnWalk {
  const int32_t* len;
  int n_seq, hc_count, chunks, chunk_rows;
  long long cap;
  int pos, end, base;  // units [pos, end); base: the first unit of sequence b
  int b;

  __device__ __forceinline__ int length(int i) const {
    const long long n = __ldg(len + i);
    return static_cast<int>(n > cap ? cap : n < 0 ? 0 : n);
  }
  __device__ __forceinline__ int units_of(int n) const { return n > 0 ? (n + TS - 1) / TS + kCost : 0; }
  // Moves (b, base) to the sequence that holds unit `at`; with kItems, to the one that holds the at-th item. Returns how
  // many come before that sequence.
  template <bool kItems>
  __device__ __forceinline__ int seek(int at) {
    const int lane = threadIdx.x & 31;
    int before = 0, unit = 0;
    #pragma unroll 1
    for (int i0 = 0; i0 < n_seq; i0 += 32) {
      const int t = i0 + lane < n_seq ? units_of(length(i0 + lane)) * hc_count : 0;
      const int w = kItems ? (t > 0 ? hc_count : 0) : t;
      int sum = w, sum_t = t;
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o), y = __shfl_up_sync(0xffffffffu, sum_t, o);
        if (lane >= o) sum += x, sum_t += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > at);
      if (past) {
        const int l = __ffs(past) - 1;
        b = i0 + l;
        base = unit + __shfl_sync(0xffffffffu, sum_t - t, l);
        return before + __shfl_sync(0xffffffffu, sum - w, l);
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
      unit += __shfl_sync(0xffffffffu, sum_t, 31);
    }
    return before;
  }
  __device__ __forceinline__ bool next(AttnRun& s) {
    while (pos < end) {
      const int n = length(b), u = units_of(n);
      if (pos >= base + u * hc_count) {
        base += u * hc_count;
        ++b;
        continue;
      }
      const int at = pos - base;
      s.hc = hc_count == 1 ? 0 : at / u;
      const int off = at - s.hc * u, take = min(end - pos, u - off);
      const int t0 = max(0, off - kCost), t1 = off + take - kCost;  // its tiles
      s.first = pos - off + kCost;
      pos += take;
      if (t1 <= t0) continue;
      s.b = b;
      s.head = chunks == 1 ? s.hc : s.hc / chunks;
      s.r0 = (s.hc - s.head * chunks) * chunk_rows;
      s.n = n;
      s.s0 = t0 * TS;
      s.s1 = min(n, t1 * TS);
      s.units = u - kCost;
      s.enter = t0 > 0;
      s.leave = t1 < s.units;
      return true;
    }
    return false;
  }
};

// The output's fragments: element x of a chunk is tile x / (64 NT), half, four of rows, lane (gid, row of the four).
// Its column:
template <int D, int NT>
__device__ __forceinline__ int attn_col(int x) {
  const int g = (x & 31) >> 2, h = x / (32 * NT) & 1, ti = x / (64 * NT);
  if constexpr (D == 64) return 8 * g + 4 * h + ti;
  return 8 * (g * (D / 64) + ti / 8 * 2 + h) + ti % 8;
}
template <int NT>
__device__ __forceinline__ int attn_row(int x) { return x / 32 % NT * 4 + (x & 3); }
// Where a column lies: tile, half, lane group.
template <int D>
__device__ __forceinline__ void attn_place(int col, int& ti, int& h, int& g) {
  if constexpr (D == 64) {
    g = col >> 3, h = (col >> 2) & 1, ti = col & 3;
  } else {
    constexpr int VW = D / 64;
    const int w = col >> 3, in = w % VW;
    g = w / VW, h = in & 1, ti = in / 2 * 8 + (col & 7);
  }
}

// (m, l, v) joined with another part's: the larger maximum, scaled sums.
__device__ __forceinline__ void attn_join(float& m, float& l, float& v, float pm, float pl, float pv) {
  const float mm = fmaxf(m, pm), f = ex2(m - mm), fp = ex2(pm - mm);
  l = fmaf(l, f, pl * fp), v = fmaf(v, f, pv * fp), m = mm;
}

// A query row's token; its place in q and in the output; where its maximum and sum go.
__device__ __forceinline__ int attn_token(const Kv4Attn& p, int row) { return p.m == 1 ? 0 : row / p.group; }
template <int D>
__device__ __forceinline__ long long attn_row_at(const Kv4Attn& p, const AttnRun& s, int row, long long ld) {
  const int t = attn_token(p, row);
  return (static_cast<long long>(s.b) * p.m + t) * ld + static_cast<long long>(s.head * p.group + row - t * p.group) * D;
}
__device__ __forceinline__ void attn_put_norm(const Kv4Attn& p, const Kv4View& c, const AttnRun& s, int row, float m, float inv) {
  // not the log of the sum: a row without a weight gives every slot 0, and weights are what the output was made with
  p.norm[(static_cast<long long>(s.b) * c.n_kv + s.head) * p.rows + row] = make_float2(-m, inv);
}

// An item's first run says which CTAs have parts of it: shares of `each` tiles, one more for the first `extra` CTAs.
__device__ __forceinline__ void attn_put_split(const Kv4Attn& p, const AttnRun& s, int hc_count, int cta, int each, int extra) {
  const int last = s.first + s.units - 1, big = (each + 1) * extra;
  const int end = last < big ? last / (each + 1) : extra + (last - big) / each;
  p.split[s.b * hc_count + s.hc] = make_int2(cta, end - cta + 1);
}

// D: head size. NT: chunks hold 4 * NT rows. kW: scores are kept for w_out. kSeveral: m may be above 1, so that rows of a
// chunk may see different slots (one token needs no look at the values: 60.7 against 59.8 us for the 48 ragged sequences).
template <int D, int NT, bool kW, bool kSeveral>
__global__ void __launch_bounds__(attn_warps(D, NT) * 32, 1) kv4_attn_kernel(const Kv4Attn p, const Kv4View c,
                                                                             int* __restrict__ err) {
  constexpr int kWarps = attn_warps(D, NT), kThreads = kWarps * 32;
  constexpr int TS = 4096 / D;      // slots of a tile
  constexpr int ST = TS / 16;       // its 16-slot steps
  constexpr int KW = D / 32;        // code words of a K row that a lane takes
  constexpr int VW = D / 64;        // code words of a V row that a lane takes
  constexpr int RC = 4 * NT;        // rows of a chunk
  constexpr int OT = D / 16;        // 16-column tiles of the output
  constexpr int kCh = D / 32;       // 16-byte chunks of a row of codes
  constexpr int kPart = RC * (D + 2);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) float s_mul[kWarps * 32 * RC];  // a warp's factors for the parts that it joins, and where they lie
  __shared__ int s_at[kWarps * 32];
  // Parts of items that the warps leave for each other, in the order of the work: 2 w of warp w is the end of an item
  // that other warps began, 2 w + 1 the beginning of one that others end.
  __shared__ int s_state[2 * kWarps];  // 0: none, 1: the item ends here, 2: it goes on
  __shared__ int s_from[2 * kWarps];   // the output part: bytes into smem
  __shared__ AttnRun s_run[2 * kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  unsigned char* ring = smem + warp * 2 * kAttnStageBytes;
  float* heads = reinterpret_cast<float*>(smem + kWarps * 2 * kAttnStageBytes);  // [warp][RC * D]
  float* ml = heads + kWarps * RC * D;                                           // [warp][head, tail][row][m, l]

  pdl_wait_prior();
  pdl_launch_dependents();
  // All tiles, this CTA's share of them, and this warp's share of those.
  AttnWalk<TS, kAttnRunCost> walk;
  walk.len = p.len, walk.n_seq = c.n_seq, walk.hc_count = c.n_kv * p.chunks, walk.cap = c.cap;
  walk.chunks = p.chunks, walk.chunk_rows = p.chunk_rows;
  int units = 0, longest = 0, used = 0;
  #pragma unroll 1
  for (int i = lane; i < c.n_seq; i += 32) {
    if (__ldg(p.len + i) > c.cap && tid == lane) atomicCAS(err, 0, kDevKv4Slot);
    const int u = walk.units_of(walk.length(i));
    units += u, longest = max(longest, u), used += u > 0;
  }
  units = __reduce_add_sync(0xffffffffu, units) * walk.hc_count;
  longest = __reduce_max_sync(0xffffffffu, longest);
  used = __reduce_add_sync(0xffffffffu, used) * walk.hc_count;
  const int cta = blockIdx.x, grid = gridDim.x;
  const bool alone = used <= grid && longest <= p.alone + kAttnRunCost;
  const int ctas = alone ? used : max(1, min(grid, units / kWarps));
  const int each = units / max(1, ctas), extra = units - each * ctas;  // the first `extra` CTAs have one unit more

  // Sequences without a slot: zeros.
  #pragma unroll 1
  for (int i = cta; i < c.n_seq; i += grid) {
    if (walk.length(i) > 0) continue;
    #pragma unroll 1
    for (long long x = tid; x < static_cast<long long>(p.m) * p.n_q * D; x += kThreads) {
      const long long t = x / (p.n_q * D);
      p.out[(static_cast<long long>(i) * p.m + t) * p.ldo + (x - t * p.n_q * D)] = 0.f;
    }
  }
  if (cta >= ctas) return;
  int lo, hi;
  if (alone) {
    const int before = walk.template seek<true>(cta);
    const int u = walk.units_of(walk.length(walk.b));
    lo = walk.base + (cta - before) * u, hi = lo + u;
  } else {
    lo = cta * each + min(cta, extra), hi = lo + each + (cta < extra);
  }
  walk.pos = lo + (hi - lo) * warp / kWarps;
  walk.end = lo + (hi - lo) * (warp + 1) / kWarps;
  if (!alone) walk.template seek<false>(walk.pos);

  // Lane-constant places in a stage: the lane's chunks as they arrive (source bytes lane * 16 + 512 i of the tile) ...
  uint32_t put[4];
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = lane + 32 * i, slot = x / kCh;
    put[i] = smem_u32(ring) + slot * (D / 2) + attn_swizzle<D>(slot, x % kCh) * 16;
  }
  const uint32_t put_sb = smem_u32(ring) + 4096 + lane * (D == 64 ? 8 : 16);
  // ... and what it reads: its words of K slot gid, of V slots 2 tig and 2 tig + 1, and their steps and bases.
  const int k_at = gid * (D / 2) + (D == 64 ? tig * 8 : D == 128 ? attn_swizzle<D>(gid, tig) * 16 : 0);
  const int v_in = gid * VW * 4;
  const int va_at = 2048 + 2 * tig * (D / 2) + attn_swizzle<D>(2 * tig, v_in / 16) * 16 + v_in % 16;
  const int vb_at = 2048 + (2 * tig + 1) * (D / 2) + attn_swizzle<D>(2 * tig + 1, v_in / 16) * 16 + v_in % 16;
  const int ks_at = 4096 + gid * (D / 8) + (D == 64 ? (tig >> 1) * 4 : tig * (D / 32));
  const int vs_at = 4608 + 2 * tig * (D / 8) + gid * VW / 4 * 4;

  auto fetch = [&](long long row, int left, int stage) {  // row: of the tile's first slot; left: rows that exist
    const uint32_t off = stage * kAttnStageBytes;
    const uint8_t *k = c.k + row * (D / 2) + lane * 16, *v = c.v + row * (D / 2) + lane * 16;
    constexpr int kSb = D == 64 ? 8 : 16;  // a d = 64 row has 8 bytes of steps and bases, and no more alignment
    const uint8_t* ks = reinterpret_cast<const uint8_t*>(c.ks) + row * (D / 8) + lane * kSb;
    const uint8_t* vs = reinterpret_cast<const uint8_t*>(c.vs) + row * (D / 8) + lane * kSb;
    if (left >= TS) {
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        cp_async16(put[i] + off, k + 512 * i);
        cp_async16(put[i] + off + 2048, v + 512 * i);
      }
      if constexpr (D == 64) {
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          cp_async8(put_sb + off + 256 * i, ks + 256 * i);
          cp_async8(put_sb + off + 512 + 256 * i, vs + 256 * i);
        }
      } else {
        cp_async16(put_sb + off, ks);
        cp_async16(put_sb + off + 512, vs);
      }
      return;
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) {  // rows that do not exist become zeros: finite values, whatever lies there
      const bool on = (lane + 32 * i) / kCh < left;
      cp_async16(put[i] + off, on ? k + 512 * i : c.k, on);
      cp_async16(put[i] + off + 2048, on ? v + 512 * i : c.v, on);
    }
    if constexpr (D == 64) {
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool on = lane + 32 * i < left;
        cp_async8(put_sb + off + 256 * i, on ? static_cast<const void*>(ks + 256 * i) : c.ks, on);
        cp_async8(put_sb + off + 512 + 256 * i, on ? static_cast<const void*>(vs + 256 * i) : c.vs, on);
      }
    } else {
      const bool on = lane * 16 / (D / 8) < left;
      cp_async16(put_sb + off, on ? static_cast<const void*>(ks) : c.ks, on);
      cp_async16(put_sb + off + 512, on ? static_cast<const void*>(vs) : c.vs, on);
    }
  };
  auto first_row = [&](const AttnRun& s) { return (static_cast<long long>(s.b) * c.n_kv + s.head) * c.cap; };
  auto token = [&](int row) { return attn_token(p, row); };
  auto row_at = [&](const AttnRun& s, int row, long long ld) { return attn_row_at<D>(p, s, row, ld); };
  auto put_norm = [&](const AttnRun& s, int row, float m, float inv) { attn_put_norm(p, c, s, row, m, inv); };

  if (lane < 2) s_state[2 * warp + lane] = 0;
  __syncwarp();
  // A run's queries on their way to L1, before they are needed.
  auto touch = [&](const AttnRun& s) {
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = s.r0 + nt * 4 + (gid >> 1);
      if (r < p.rows) {
        const float* at = p.q + row_at(s, r, p.ldq) + tig * (D / 4);
        asm volatile("prefetch.global.L1 [%0];" ::"l"(at));
        if constexpr (D == 256) asm volatile("prefetch.global.L1 [%0];" ::"l"(at + 32));
      }
    }
  };
  AttnRun run, nxt;
  bool have = walk.next(run);
  long long row0 = 0;
  if (have) {
    touch(run);
    row0 = first_row(run);
    fetch(row0 + run.s0, run.s1 - run.s0, 0);
  }
  cp_async_commit();
  int stage = 0;

  while (have) {
    const bool more = walk.next(nxt);
    long long row1 = 0;  // the next run's first slot, and its slots
    int left1 = 0;
    if (more) row1 = first_row(nxt) + nxt.s0, left1 = nxt.s1 - nxt.s0;
    const int r0 = run.r0;

    // The chunk's rows.
    uint32_t qb[NT][2 * KW][2];
    float sc[NT];  // what a score has to be multiplied by to be in log2 units, of row tig; not negative
    int vis[NT];   // slots that row tig sees
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + nt * 4 + (gid >> 1), rt = r0 + nt * 4 + tig;
      const float up = attn_query<D>(r < p.rows ? p.q + row_at(run, r, p.ldq) : nullptr, p.vec, p.scale_m, p.scale_e, qb[nt]);
      sc[nt] = __shfl_sync(0xffffffffu, up, 8 * tig);
      vis[nt] = rt < p.rows ? run.n - (p.m - 1 - token(rt)) : 0;
    }
    const int all_see = run.n - (p.m - 1 - token(r0));  // slots that every row sees (rows that are not there: any)

    float top[NT], sum[NT], o[OT][2][NT];
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      top[nt] = kAttnNone, sum[nt] = 0.f;
      #pragma unroll
      for (int i = 0; i < OT; ++i) o[i][0][nt] = 0.f, o[i][1][nt] = 0.f;
    }

    #pragma unroll 1
    for (int at = run.s0; at < run.s1; at += TS) {
      const bool same = at + TS < run.s1;
      if (same || more) fetch(same ? row0 + at + TS : row1, same ? run.s1 - at - TS : left1, stage ^ 1);
      cp_async_commit();
      cp_async_wait<1>();
      __syncwarp();
      const unsigned char* st = ring + stage * kAttnStageBytes;
      const int left = run.s1 - at;
      bool unsafe = false;
      if (kSeveral && all_see < run.n && at + TS > all_see) {  // a row may not see slots that others do
        uint32_t* sb = reinterpret_cast<uint32_t*>(ring + stage * kAttnStageBytes + 4608 + lane * 16);
        const uint4 x = *reinterpret_cast<const uint4*>(sb);
        unsafe = __any_sync(0xffffffffu, kv4_large(x.x) || kv4_large(x.y) || kv4_large(x.z) || kv4_large(x.w));
        if (unsafe) {
          #pragma unroll 1
          for (int i = 0; i < 4; ++i)
            if ((lane * 4 + i) / (D / 32) >= all_see - at && kv4_infinite(sb[i])) sb[i] = 0;
          __syncwarp();
        }
      }
      // scores (times sc: in log2 units)
      float s[ST][2][NT];
      #pragma unroll
      for (int u = 0; u < ST; ++u) {
        float acc[NT][4];
        {
          const unsigned char* pk = st + k_at + u * 16 * (D / 2);
          uint32_t wa[KW], wb[KW];
          if constexpr (D == 64) {
            const uint2 a = *reinterpret_cast<const uint2*>(pk), b = *reinterpret_cast<const uint2*>(pk + 8 * (D / 2));
            wa[0] = a.x, wa[1] = a.y, wb[0] = b.x, wb[1] = b.y;
          } else {
            #pragma unroll
            for (int h = 0; h < KW / 4; ++h) {
              const int ch = D == 128 ? 0 : attn_swizzle<D>(gid, tig * 2 + h) * 16;
              const uint4 a = *reinterpret_cast<const uint4*>(pk + ch), b = *reinterpret_cast<const uint4*>(pk + 8 * (D / 2) + ch);
              wa[4 * h] = a.x, wa[4 * h + 1] = a.y, wa[4 * h + 2] = a.z, wa[4 * h + 3] = a.w;
              wb[4 * h] = b.x, wb[4 * h + 1] = b.y, wb[4 * h + 2] = b.z, wb[4 * h + 3] = b.w;
            }
          }
          const unsigned char* ps = st + ks_at + u * 16 * (D / 8);
          #pragma unroll
          for (int w = 0; w < KW; ++w) {
            const __half2 sa = *reinterpret_cast<const __half2*>(ps + w / 4 * 4);
            const __half2 sb = *reinterpret_cast<const __half2*>(ps + 8 * (D / 8) + w / 4 * 4);
            const __half2 sta = __low2half2(sa), bsa = __high2half2(sa), stb = __low2half2(sb), bsb = __high2half2(sb);
            const uint32_t a0 = kv4_pair<false>(wa[w], p.mul64, sta, bsa), b0 = kv4_pair<false>(wb[w], p.mul64, stb, bsb);
            const uint32_t a1 = kv4_pair<true>(wa[w], p.mul4, sta, bsa), b1 = kv4_pair<true>(wb[w], p.mul4, stb, bsb);
            const uint32_t xa = wa[w] >> 8, xb = wb[w] >> 8;
            const uint32_t a2 = kv4_pair<false>(xa, p.mul64, sta, bsa), b2 = kv4_pair<false>(xb, p.mul64, stb, bsb);
            const uint32_t a3 = kv4_pair<true>(xa, p.mul4, sta, bsa), b3 = kv4_pair<true>(xb, p.mul4, stb, bsb);
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (w == 0)
                mma_f16_first(acc[nt], a0, b0, a1, b1, qb[nt][0][0], qb[nt][0][1]);
              else
                mma_f16(acc[nt], a0, b0, a1, b1, qb[nt][2 * w][0], qb[nt][2 * w][1]);
              mma_f16(acc[nt], a2, b2, a3, b3, qb[nt][2 * w + 1][0], qb[nt][2 * w + 1][1]);
            }
          }
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            s[u][0][nt] = acc[nt][0] + acc[nt][1];
            s[u][1][nt] = acc[nt][2] + acc[nt][3];
          }
        }
      }
      if (kW) {
        // rows of the chunk that are not there have a place too: only slots are checked, in a tile that is not whole
        float* to = p.score + ((static_cast<long long>(run.b) * walk.hc_count + run.hc) * RC + tig) * c.cap + at + gid;
        const long long next = 4 * c.cap;
        if (left >= TS) {
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt, to += next) {
            #pragma unroll
            for (int u = 0; u < ST; ++u) to[u * 16] = s[u][0][nt] * sc[nt], to[u * 16 + 8] = s[u][1][nt] * sc[nt];
          }
        } else {
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt, to += next) {
            #pragma unroll
            for (int u = 0; u < ST; ++u) {
              if (u * 16 + gid < left) to[u * 16] = s[u][0][nt] * sc[nt];
              if (u * 16 + gid + 8 < left) to[u * 16 + 8] = s[u][1][nt] * sc[nt];
            }
          }
        }
      }
      // slots that a row does not see; then the running maximum, and the weights as split halves
      const bool some_hidden = left < TS || at + TS > all_see;
      uint32_t pb[ST][NT][2];
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (some_hidden) {
          const int see = min(left, vis[nt] - at);
          #pragma unroll
          for (int u = 0; u < ST; ++u) {
            if (u * 16 + gid >= see) s[u][0][nt] = -INFINITY;
            if (u * 16 + gid + 8 >= see) s[u][1][nt] = -INFINITY;
          }
        }
        float best = s[0][0][nt];
        #pragma unroll
        for (int u = 0; u < ST; ++u) best = fmaxf(best, fmaxf(s[u][0][nt], s[u][1][nt]));
        best *= sc[nt];
        if (__any_sync(0xffffffffu, best > attn_limit(top[nt]))) {
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 8));
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 16));
          best = fmaxf(attn_top(best), top[nt]);
          const float f = ex2(top[nt] - best);
          top[nt] = best;
          sum[nt] *= f;
          #pragma unroll
          for (int i = 0; i < OT; ++i) o[i][0][nt] *= f, o[i][1][nt] *= f;
        }
        #pragma unroll
        for (int u = 0; u < ST; ++u) {
          #pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float e = ex2(fmaf(s[u][h][nt], sc[nt], -top[nt]));
            sum[nt] += e;
            const float big = __uint_as_float(__float_as_uint(e) & 0xFFFFE000u);
            pb[u][nt][h] = transpose8x8(h2_bits(__floats2half2_rn(big, e - big)));
          }
        }
      }
      // output: byte by byte of the V words
      uint32_t wa[ST][2][VW], wb[ST][2][VW];  // two slots' words
      __half2 stp[ST][2], bas[ST][2];
      #pragma unroll
      for (int u = 0; u < ST; ++u) {
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char* pa = st + va_at + (u * 16 + h * 8) * (D / 2);
          const unsigned char* pq = st + vb_at + (u * 16 + h * 8) * (D / 2);
          if constexpr (VW == 1) {
            wa[u][h][0] = *reinterpret_cast<const uint32_t*>(pa), wb[u][h][0] = *reinterpret_cast<const uint32_t*>(pq);
          } else if constexpr (VW == 2) {
            const uint2 a = *reinterpret_cast<const uint2*>(pa), b = *reinterpret_cast<const uint2*>(pq);
            wa[u][h][0] = a.x, wa[u][h][1] = a.y, wb[u][h][0] = b.x, wb[u][h][1] = b.y;
          } else {
            const uint4 a = *reinterpret_cast<const uint4*>(pa), b = *reinterpret_cast<const uint4*>(pq);
            wa[u][h][0] = a.x, wa[u][h][1] = a.y, wa[u][h][2] = a.z, wa[u][h][3] = a.w;
            wb[u][h][0] = b.x, wb[u][h][1] = b.y, wb[u][h][2] = b.z, wb[u][h][3] = b.w;
          }
          const unsigned char* ps = st + vs_at + (u * 16 + h * 8) * (D / 8);
          const uint32_t x = *reinterpret_cast<const uint32_t*>(ps), y = *reinterpret_cast<const uint32_t*>(ps + D / 8);
          stp[u][h] = bits_h2(__byte_perm(x, y, 0x5410));
          bas[u][h] = bits_h2(__byte_perm(x, y, 0x7632));
        }
      }
      // Tiles 2 y and 2 y + 1 are the low and the high nibbles of one byte of the words: d = 64, columns 8 gid + n and
      // 8 gid + 4 + n of the lane's word (n = tile); else columns n of words 2 w and 2 w + 1 of the lane's words
      // (tile = 8 w + n).
      #pragma unroll
      for (int y = 0; y < OT / 2; ++y) {
        float acc[2][NT][4];
        #pragma unroll
        for (int u = 0; u < ST; ++u) {
          {
            uint32_t ln[4], hn[4];
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
              #pragma unroll
              for (int z = 0; z < 2; ++z) {
                const int w = VW == 1 ? 0 : y / 4 * 2 + z, byte = VW == 1 ? y + 2 * z : y % 4;
                const uint32_t both = __byte_perm(wa[u][h][w], wb[u][h][w], byte | (byte + 4) << 8);
                ln[2 * h + z] = kv4_pair<false>(both, p.mul64, stp[u][h], bas[u][h]);
                hn[2 * h + z] = kv4_pair<true>(both, p.mul4, stp[u][h], bas[u][h]);
              }
            }
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (u == 0) {
                mma_f16_first(acc[0][nt], ln[0], ln[1], ln[2], ln[3], pb[u][nt][0], pb[u][nt][1]);
                mma_f16_first(acc[1][nt], hn[0], hn[1], hn[2], hn[3], pb[u][nt][0], pb[u][nt][1]);
              } else {
                mma_f16(acc[0][nt], ln[0], ln[1], ln[2], ln[3], pb[u][nt][0], pb[u][nt][1]);
                mma_f16(acc[1][nt], hn[0], hn[1], hn[2], hn[3], pb[u][nt][0], pb[u][nt][1]);
              }
            }
          }
        }
        #pragma unroll
        for (int z = 0; z < 2; ++z) {
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            o[2 * y + z][0][nt] += acc[z][nt][0] + acc[z][nt][1];
            o[2 * y + z][1][nt] += acc[z][nt][2] + acc[z][nt][3];
          }
        }
      }
      if (unsafe) {  // what was taken out of the products
        #pragma unroll 1
        for (int slot = max(all_see - at, 0); slot < min(left, TS); ++slot) {
          const uint32_t sb = __ldg(c.vs + (row0 + at + slot) * (D / kKv4Group) + gid * VW / 4);
          const bool mine = kv4_infinite(sb);
          if (!__any_sync(0xffffffffu, mine)) continue;
          const uint32_t* words = reinterpret_cast<const uint32_t*>(
              st + 2048 + slot * (D / 2) + attn_swizzle<D>(slot, v_in / 16) * 16 + v_in % 16);
          #pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t both = 0;  // not pb[slot ..]: an index would put it into memory
            #pragma unroll
            for (int x = 0; x < 2 * ST; ++x) both |= pb[x / 2][nt][x % 2] & -static_cast<uint32_t>(slot / 8 == x);
            const int from = 8 * tig + slot % 8 / 2;
            const uint32_t hi = __shfl_sync(0xffffffffu, both, from), lo = __shfl_sync(0xffffffffu, both, from + 4);
            if (!mine || at + slot >= vis[nt]) continue;
            const float w = kv4_weight(hi, lo, slot & 1);
            #pragma unroll
            for (int t = 0; t < OT; ++t)
              #pragma unroll
              for (int h = 0; h < 2; ++h)
                o[t][h][nt] += w * kv4_value(words[VW == 1 ? 0 : t / 8 * 2 + h], VW == 1 ? 4 * h + t : t % 8, sb);
          }
        }
      }
      __syncwarp();
      stage ^= 1;
    }

    // The run's result. All of an item: the output, through the stage that was just used up. A part of one: left in
    // shared memory for the CTA; the end of an item that others began comes first in the share and lies apart from the
    // ring, which goes on; the beginning of one that others end comes last and stays in the used-up stage.
    float* fr = run.enter ? heads + warp * RC * D : reinterpret_cast<float*>(ring + (stage ^ 1) * kAttnStageBytes);
    const int which = 2 * warp + (run.enter ? 0 : 1);
    #pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      #pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum[nt] += __shfl_xor_sync(0xffffffffu, sum[nt], x);
      if (gid == 0 && (run.enter || run.leave)) {
        float* to = ml + (which * RC + nt * 4 + tig) * 2;
        to[0] = top[nt], to[1] = sum[nt];
      }
      #pragma unroll
      for (int i = 0; i < OT; ++i)
        #pragma unroll
        for (int h = 0; h < 2; ++h) fr[((i * 2 + h) * NT + nt) * 32 + lane] = o[i][h][nt];
    }
    if (!run.enter && !run.leave) {
      __syncwarp();
      #pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float inv = sum[nt] != 0.f ? 1.f / sum[nt] : 0.f;
        #pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int r = nt * 4 + r4;
          const float f = __shfl_sync(0xffffffffu, inv, r4), tp = __shfl_sync(0xffffffffu, top[nt], r4);
          if (r0 + r >= p.rows) continue;
          float* to = p.out + row_at(run, r0 + r, p.ldo);
          #pragma unroll
          for (int x = 0; x < D; x += 32) {
            int ti, h, g;
            attn_place<D>(x + lane, ti, h, g);
            to[x + lane] = fr[((ti * 2 + h) * NT + nt) * 32 + g * 4 + r4] * f;
          }
          if (kW && lane == 0) put_norm(run, r0 + r, tp, f);
        }
      }
      if (lane == 0) p.split[run.b * walk.hc_count + run.hc] = make_int2(cta, 1);
      __syncwarp();
    } else if (lane == 0) {
      s_state[which] = run.leave ? 2 : 1;
      s_from[which] = static_cast<int>(reinterpret_cast<unsigned char*>(fr) - smem);
      s_run[which] = run;
    }
    have = more;
    row0 = row1 - nxt.s0;
    run = nxt;
  }
  cp_async_wait<0>();
  __syncthreads();

  // Parts of one item left by neighbouring warps become one result: all of the item, or this CTA's part of it, of which
  // there are at most two (kind 0: it began in an earlier CTA; kind 1: it began here and goes on). Lane k knows part k. A
  // list begins with every beginning of an item (odd parts), and with the first part if that is the end of one; each warp
  // takes a slice of a list.
  const uint32_t valid = __ballot_sync(0xffffffffu, lane < 2 * kWarps && s_state[lane] != 0);
  if (!valid) return;
  const uint32_t begins = (valid & 0xAAAAAAAAu) | (valid & -valid);
  const int lists = __popc(begins);
  for (int mine = warp; mine < max(lists, kWarps / lists * lists); mine += kWarps) {
    const int list = mine % lists, slice = mine / lists, slices = lists < kWarps ? kWarps / lists : 1;
    uint32_t left = begins;
    for (int i = 0; i < list; ++i) left &= left - 1;
    const int first = __ffs(left) - 1;
    left &= left - 1;
    const uint32_t parts = valid & ~((1u << first) - 1u) & (left ? (1u << (__ffs(left) - 1)) - 1u : 0xffffffffu);
    const int kind = first & 1, last = 31 - __clz(parts);
    const bool final_here = kind == 1 && s_state[last] == 1;
    const AttnRun& it = s_run[first];
    float* part = p.part + (static_cast<long long>(cta) * 2 + kind) * kPart;
    // Lane (row, group): the row's maximum and sum over the parts, which the groups take in turn; then the factors.
    constexpr int kRowLanes = RC > 8 ? 16 : RC, kGroups = 32 / kRowLanes;  // a power of two; lanes of rows that are not there repeat row 0
    const int count = __popc(parts), lane_row = lane % kRowLanes, group = lane / kRowLanes;
    const bool has_row = lane_row < RC;
    const int row = has_row ? lane_row : 0;
    float* mul = s_mul + warp * 32 * RC;  // [part][row]
    int* from = s_at + warp * 32;         // [part]
    if (parts >> lane & 1) from[__popc(parts & ((1u << lane) - 1u))] = lane;
    __syncwarp();
    float m = kAttnNone, l = 0.f;
    for (int i = group; i < count; i += kGroups) m = fmaxf(m, ml[(from[i] * RC + row) * 2]);
    #pragma unroll
    for (int x = kRowLanes; x < 32; x *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    for (int i = group; i < count; i += kGroups) {
      const float f = ex2(ml[(from[i] * RC + row) * 2] - m);
      l = fmaf(f, ml[(from[i] * RC + row) * 2 + 1], l);
      if (has_row) mul[i * RC + row] = f;
    }
    #pragma unroll
    for (int x = kRowLanes; x < 32; x *= 2) l += __shfl_xor_sync(0xffffffffu, l, x);
    const float inv = final_here ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
    if (slice == 0 && group == 0 && has_row) {
      if (!final_here)
        part[row] = m, part[RC + row] = l;
      else if (kW && it.r0 + row < p.rows)
        put_norm(it, it.r0 + row, m, inv);
    }
    __syncwarp();
    if ((parts >> lane & 1) != 0) from[__popc(parts & ((1u << lane) - 1u))] = s_from[lane];
    __syncwarp();
    for (int x = (slice * 32 + lane) * 4; x < RC * D; x += slices * 128) {  // the four rows of a column
      const int r = attn_row<NT>(x);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      #pragma unroll 4
      for (int i = 0; i < count; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(mul + i * RC + r);
        const float4 y = *reinterpret_cast<const float4*>(smem + from[i] + x * 4);
        v.x = fmaf(f.x, y.x, v.x), v.y = fmaf(f.y, y.y, v.y), v.z = fmaf(f.z, y.z, v.z), v.w = fmaf(f.w, y.w, v.w);
      }
      if (!final_here) *reinterpret_cast<float4*>(part + 2 * RC + x) = v;
      const float w[4] = {v.x, v.y, v.z, v.w};
      #pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float scale = __shfl_sync(0xffffffffu, inv, r + j);  // lane r + j has row r + j
        if (final_here && it.r0 + r + j < p.rows)
          p.out[row_at(it, it.r0 + r + j, p.ldo) + attn_col<D, NT>(x)] = w[j] * scale;
      }
    }
    if (kind == 1 && slice == 0 && lane == 0) {
      if (final_here)
        p.split[it.b * walk.hc_count + it.hc] = make_int2(cta, 1);
      else
        attn_put_split(p, it, walk.hc_count, cta, each, extra);
    }
    __syncwarp();
  }
}

// The parts of split items, once every CTA's are written: a block has 32 times four values of an item's chunk (the four
// rows of a column), its warps take turns with the parts, and their maxima, sums and values are joined in shared memory.
constexpr int kJoinWarps = 4;

template <int D, int NT, bool kW>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_join_kernel(const Kv4Attn p, const Kv4View c) {
  constexpr int RC = 4 * NT, kPart = RC * (D + 2), kSlices = RC * D / 128;
  __shared__ float4 s_join[kJoinWarps - 1][3][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int item = blockIdx.x / kSlices, slice = blockIdx.x - item * kSlices;
  const int hc = item % (c.n_kv * p.chunks), b = item / (c.n_kv * p.chunks);
  const int n = __ldg(p.len + b);
  const int2 s = p.split[item];  // of a sequence without slots: left over
  if (n <= 0 || s.y <= 1) return;
  const int x = (slice * 32 + lane) * 4, r = attn_row<NT>(x);
  AttnRun it;
  it.b = b, it.head = hc / p.chunks, it.r0 = (hc - it.head * p.chunks) * p.chunk_rows;
  const int rows = min(p.chunk_rows, p.rows - it.r0);
  float m[4] = {kAttnNone, kAttnNone, kAttnNone, kAttnNone}, l[4] = {}, v[4] = {};
  constexpr int kAhead = 5;
  #pragma unroll 1
  for (int k0 = warp; k0 < s.y; k0 += kAhead * kJoinWarps) {
    float4 pm[kAhead], pl[kAhead], pv[kAhead];
    #pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int k = k0 + i * kJoinWarps;
      if (k >= s.y || r >= rows) continue;
      const float* at = p.part + (static_cast<long long>(s.x + k) * 2 + (k == 0 ? 1 : 0)) * kPart;
      pm[i] = *reinterpret_cast<const float4*>(at + r);
      pl[i] = *reinterpret_cast<const float4*>(at + RC + r);
      pv[i] = *reinterpret_cast<const float4*>(at + 2 * RC + x);
    }
    #pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (k0 + i * kJoinWarps >= s.y || r >= rows) continue;
      attn_join(m[0], l[0], v[0], pm[i].x, pl[i].x, pv[i].x);
      attn_join(m[1], l[1], v[1], pm[i].y, pl[i].y, pv[i].y);
      attn_join(m[2], l[2], v[2], pm[i].z, pl[i].z, pv[i].z);
      attn_join(m[3], l[3], v[3], pm[i].w, pl[i].w, pv[i].w);
    }
  }
  if (warp > 0) {
    s_join[warp - 1][0][lane] = make_float4(m[0], m[1], m[2], m[3]);
    s_join[warp - 1][1][lane] = make_float4(l[0], l[1], l[2], l[3]);
    s_join[warp - 1][2][lane] = make_float4(v[0], v[1], v[2], v[3]);
  }
  __syncthreads();
  if (warp > 0) return;
  #pragma unroll
  for (int g = 0; g < kJoinWarps - 1; ++g) {
    const float4 pm = s_join[g][0][lane], pl = s_join[g][1][lane], pv = s_join[g][2][lane];
    attn_join(m[0], l[0], v[0], pm.x, pl.x, pv.x);
    attn_join(m[1], l[1], v[1], pm.y, pl.y, pv.y);
    attn_join(m[2], l[2], v[2], pm.z, pl.z, pv.z);
    attn_join(m[3], l[3], v[3], pm.w, pl.w, pv.w);
  }
  const int col = attn_col<D, NT>(x);
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (r + j >= rows) continue;
    p.out[attn_row_at<D>(p, it, it.r0 + r + j, p.ldo) + col] = l[j] != 0.f ? v[j] / l[j] : 0.f;
    if (kW && col == 0) attn_put_norm(p, c, it, it.r0 + r + j, m[j], l[j] != 0.f ? 1.f / l[j] : 0.f);
  }
}

// The weights that slots received, from the kept scores and the rows' sums: a thread has kWeightSlots slots, 256 apart, of
// a kv head. Bound by the scores' reads (4 bytes a row and slot): four slots keep enough of them in flight for few rows (8 x
// 8 heads of 4 rows, up to 16384 slots: the call takes 32.8 us, with one slot 35.1), one slot makes enough blocks where many
// rows do that (8 x 8 heads of 16 rows, up to 4096 slots: 23.3 us, with four 25.3). At 8 rows they are close: 28.8 with four
// and 28.7 with one for 8 x 8 heads of up to 8192 slots, 26.4 and 25.8 for 16 x 8 of up to 2000; at 12, 37.6 and 35.9.
constexpr int kWeightThreads = 256, kWeightFewRows = 8;

template <int kWeightSlots>
__global__ void __launch_bounds__(kWeightThreads) kv4_weights_kernel(const Kv4Attn p, const Kv4View c, int blocks) {
  __shared__ float2 s_norm[kWeightThreads];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int tid = threadIdx.x, bh = blockIdx.x / blocks, b = bh / c.n_kv;
  const long long j0 = static_cast<long long>(blockIdx.x - bh * blocks) * (kWeightThreads * kWeightSlots);
  long long n = __ldg(p.len + b);
  if (n > c.cap) n = c.cap;
  if (j0 >= n) return;
  const long long at = static_cast<long long>(bh) * c.cap + j0 + tid;
  // slots of this thread, and rows that come too early to see each of them
  const int have = static_cast<int>(n - j0 - tid), old = static_cast<int>(n - p.m - j0 - tid);
  float w[kWeightSlots], got[kWeightSlots];  // what was received is added up by itself, then to the old weight: one rounding of that
  int skip[kWeightSlots];
  #pragma unroll
  for (int i = 0; i < kWeightSlots; ++i) {
    const int late = i * kWeightThreads - old;
    w[i] = late < 0 && p.w_in ? p.w_in[at + i * kWeightThreads] : 0.f, got[i] = 0.f;
    skip[i] = i * kWeightThreads >= have ? p.rows : late > 0 ? late * p.group : 0;
  }
  for (int chunk = 0, r0 = 0; chunk < p.chunks; ++chunk, r0 += p.chunk_rows) {  // at most 80 rows
    const int rows = min(p.chunk_rows, p.rows - r0);
    __syncthreads();
    if (tid < rows) s_norm[tid] = p.norm[static_cast<long long>(bh) * p.rows + r0 + tid];
    __syncthreads();
    const float* s = p.score + (static_cast<long long>(bh) * p.chunks + chunk) * p.kept_rows * c.cap + j0 + tid;
    constexpr int kAhead = kWeightSlots == 1 ? 4 : 8;  // rows in flight; the other way round the two calls take 59.8 and 35.1 us
    #pragma unroll kAhead
    for (int r = 0; r < rows; ++r) {
      const float2 norm = s_norm[r];
      #pragma unroll
      for (int i = 0; i < kWeightSlots; ++i) {
        const bool sees = r0 + r >= skip[i];
        const float score = sees ? __ldg(s + i * kWeightThreads) : 0.f, sum = fmaf(ex2(score + norm.x), norm.y, got[i]);
        got[i] = sees ? sum : got[i];  // not 0 times what may be a NaN
      }
      s += c.cap;
    }
  }
  #pragma unroll
  for (int i = 0; i < kWeightSlots; ++i)
    if (i * kWeightThreads < have) p.w_out[at + i * kWeightThreads] = w[i] + got[i];
}

}  // namespace vmlm
