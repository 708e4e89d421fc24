// kv4_attn_rows.cuh -- attention over a 4-bit cache for many query rows a kv head of
// d = 256 (several new tokens, or many heads that share keys and values).
//
// The products and their layouts are those of kv4_attn.cuh. There every warp
// unpacks its own slots and multiplies them with all rows, whose output it holds:
// 4 rows at d = 256, and the cache is unpacked again for every 4. Here a CTA of 16
// warps shares a tile of 64 slots, and up to 80 rows (16 heads of 5 tokens) are one
// chunk:
//   scores   warp (slots 16 s .., part g of the rows): K unpacked once a part
//   weights  to shared memory as B fragments, with a maximum shared by the tile
//   output   each warp its 16 columns of V, V unpacked once, all slots, all rows
// Three barriers a tile. What bounds it is the latency between them, with four
// warps a scheduler (35% of issue slots, mma.sync 21% active; 80 rows over 16 ragged
// caches of up to 3001 slots take 46 us), then mma.sync (one m16n8k16 in two cycles an SM: 64 slots take
// d * rows / 8 of them) and the B fragments' reads from shared memory (256 bytes
// for one).
#pragma once
#include "kv4_attn.cuh"

namespace vmlm {

constexpr int kRowsHead = 256;
constexpr int kRowsSlots = 64;        // of a tile
constexpr int kRowsWarps = 16;
constexpr int kRowsMost = 20;         // fours of rows that a chunk holds at most: what 128 registers a thread hold
constexpr int kRowsRunCost = 3;       // what a run costs besides its tiles, in tiles (its queries' fragments and its result)
constexpr int kRowsStageBytes = kRowsSlots * kRowsHead / 4 * 5;
// Shared memory: two tiles, the queries' and the weights' fragments, per row 4 maxima, factor, 4 sums, scale and sight.
__host__ __device__ constexpr int rows_smem_bytes(int NT) {
  return 2 * kRowsStageBytes + NT * (kRowsHead / 32) * 512 + 4 * NT * 256 + NT * 4 * 11 * 4;
}

// NT: fours of rows of a chunk, a multiple of the 4 parts; rows that are not there are zeros that see nothing.
template <int NT, bool kW>
__global__ void __launch_bounds__(kRowsWarps * 32, 1) kv4_attn_rows_kernel(const Kv4Attn p, const Kv4View c, int* __restrict__ err) {
  constexpr int D = kRowsHead, TS = kRowsSlots, kRowsThreads = kRowsWarps * 32;
  constexpr int PARTS = kRowsWarps / 4, NG = NT / PARTS;  // parts of the rows, fours of rows of each
  static_assert(NT % PARTS == 0 && TS * D / 32 == kRowsThreads, "");
  constexpr int RC = 4 * NT, kPart = RC * (D + 2);
  constexpr int KW = D / 32, VW = D / 64, kCh = D / 32;
  constexpr int kStage = kRowsStageBytes;
  constexpr int kVAt = TS * D / 2, kKsAt = TS * D, kVsAt = TS * D + TS * D / 8;  // in a stage: K, V, K's and V's scales
  extern __shared__ __align__(128) unsigned char smem[];
  uint4* qs = reinterpret_cast<uint4*>(smem + 2 * kStage);                          // [NT][KW][lane]
  uint2* ps = reinterpret_cast<uint2*>(smem + 2 * kStage + NT * KW * 512);          // [4][NT][lane]
  float* s_max = reinterpret_cast<float*>(ps + 4 * NT * 32);                              // [4][RC]
  float* s_fac = s_max + 4 * RC;                                                    // [RC]
  float* s_sum = s_fac + RC;                                                        // [4][RC]
  float* s_scale = s_sum + 4 * RC;                                                  // [RC]
  int* s_see = reinterpret_cast<int*>(s_scale + RC);                                // [RC]: slots that a row sees
  __shared__ int s_grown[2][5];  // by a tile's parity: a part's maxima grew; values were taken out of the products (4)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  const int st = warp & 3, share = warp >> 2;           // scores: slots 16 st .., fours share * NG ..
  const int ot = warp;                                  // output: its tile

  pdl_wait_prior();
  pdl_launch_dependents();
  AttnWalk<TS, kRowsRunCost> walk;
  walk.len = p.len, walk.n_seq = c.n_seq, walk.hc_count = c.n_kv * p.chunks, walk.cap = c.cap;
  walk.chunks = p.chunks, walk.chunk_rows = p.chunk_rows;
  int units = 0;
  #pragma unroll 1
  for (int i = lane; i < c.n_seq; i += 32) {
    if (__ldg(p.len + i) > c.cap && tid == lane) atomicCAS(err, 0, kDevKv4Slot);
    units += walk.units_of(walk.length(i));
  }
  units = __reduce_add_sync(0xffffffffu, units) * walk.hc_count;
  const int cta = blockIdx.x, grid = gridDim.x;
  #pragma unroll 1
  for (int i = cta; i < c.n_seq; i += grid) {  // sequences without a slot: zeros
    if (walk.length(i) > 0) continue;
    #pragma unroll 1
    for (long long x = tid; x < static_cast<long long>(p.m) * p.n_q * D; x += kRowsThreads) {
      const long long t = x / (p.n_q * D);
      p.out[(static_cast<long long>(i) * p.m + t) * p.ldo + (x - t * p.n_q * D)] = 0.f;
    }
  }
  const int ctas = min(grid, units);
  if (cta >= ctas) return;
  const int each = units / ctas, extra = units - each * ctas;
  walk.pos = cta * each + min(cta, extra), walk.end = walk.pos + each + (cta < extra);
  walk.template seek<false>(walk.pos);

  // A thread's part of a tile: one 16-byte chunk of K's codes and of V's, and the first threads one chunk of the steps
  // and bases of each.
  const bool has_sb = tid < TS * D / 8 / 16;
  const int code_slot = tid / kCh, sb_slot = tid * 16 / (D / 8);
  const uint32_t code_to = smem_u32(smem) + code_slot * (D / 2) + attn_swizzle<D>(code_slot, tid % kCh) * 16;
  const uint32_t sb_to = smem_u32(smem) + kKsAt + tid * 16;
  const uint8_t *k_from = c.k + tid * 16, *v_from = c.v + tid * 16;
  const uint8_t* ks_from = reinterpret_cast<const uint8_t*>(c.ks) + tid * 16;
  const uint8_t* vs_from = reinterpret_cast<const uint8_t*>(c.vs) + tid * 16;
  auto fetch = [&](long long row, int left, int stage) {  // rows that do not exist become zeros
    const uint32_t to = stage * kStage;
    bool on = code_slot < left;
    long long at = on ? row * (D / 2) : -tid * 16ll;
    cp_async16(code_to + to, k_from + at, on);
    cp_async16(code_to + to + kVAt, v_from + at, on);
    if (has_sb) {
      on = sb_slot < left;
      at = on ? row * (D / 8) : -tid * 16ll;
      cp_async16(sb_to + to, ks_from + at, on);
      cp_async16(sb_to + to + kVsAt - kKsAt, vs_from + at, on);
    }
  };
  auto first_row = [&](const AttnRun& s) { return (static_cast<long long>(s.b) * c.n_kv + s.head) * c.cap; };

  const int k_at = (st * 16 + gid) * (D / 2);
  const int ks_at = kKsAt + (st * 16 + gid) * (D / 8) + tig * (D / 32);
  const int v_in = gid * VW * 4;
  const int va_at = kVAt + 2 * tig * (D / 2) + attn_swizzle<D>(2 * tig, v_in / 16) * 16 + v_in % 16;
  const int vb_at = kVAt + (2 * tig + 1) * (D / 2) + attn_swizzle<D>(2 * tig + 1, v_in / 16) * 16 + v_in % 16;
  const int vs_at = kVsAt + 2 * tig * (D / 8) + gid * VW / 4 * 4;
  const uint32_t nibbles = ot & 1 ? 0x00F000F0u : 0x000F000Fu, to_top = ot & 1 ? p.mul4 : p.mul64;

  AttnRun run, nxt;
  if (!walk.next(run)) return;  // a share may be an item's run cost alone
  // the first run's queries on their way to L1
  for (int nt = warp; nt < NT; nt += kRowsWarps) {
    const int r = nt * 4 + (gid >> 1);
    if (r < min(p.chunk_rows, p.rows - run.r0)) {
      const float* at = p.q + attn_row_at<D>(p, run, run.r0 + r, p.ldq) + tig * (D / 4);
      asm volatile("prefetch.global.L1 [%0];" ::"l"(at));
      asm volatile("prefetch.global.L1 [%0];" ::"l"(at + 32));
    }
  }
  long long row0 = first_row(run);
  fetch(row0 + run.s0, run.s1 - run.s0, 0);
  cp_async_commit();
  int stage = 0, parity = 0;
  if (tid < 10) s_grown[tid / 5][tid % 5] = 0;

  while (true) {
    const bool more = walk.next(nxt);
    long long row1 = 0;
    int left1 = 0;
    if (more) row1 = first_row(nxt) + nxt.s0, left1 = nxt.s1 - nxt.s0;
    const int rows = min(p.chunk_rows, p.rows - run.r0);  // of this chunk
    __syncthreads();  // the last run's fragments have been read
    for (int nt = warp; nt < NT; nt += kRowsWarps) {
      const int r = nt * 4 + (gid >> 1);
      uint32_t qb[2 * KW][2];
      const float up = attn_query<D>(r < rows ? p.q + attn_row_at<D>(p, run, run.r0 + r, p.ldq) : nullptr, p.vec, p.scale_m, p.scale_e, qb);
      #pragma unroll
      for (int w = 0; w < KW; ++w)
        qs[(nt * KW + w) * 32 + lane] = make_uint4(qb[2 * w][0], qb[2 * w][1], qb[2 * w + 1][0], qb[2 * w + 1][1]);
      if (tig == 0 && !(gid & 1)) {
        s_scale[r] = up;
        s_see[r] = r < rows ? run.n - (p.m - 1 - attn_token(p, run.r0 + r)) : 0;
      }
    }
    const int n0 = share * NG;  // the first four of rows of this warp's scores
    // of a row: what a score is multiplied by, its top so far, the score from which that moves
    float sc[NG], top[NG], grow[NG], sum[NG];
    const int all_see = run.n - (p.m - 1 - attn_token(p, run.r0));  // slots that every row sees (rows that are not there: any)
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < NG; ++i)
      sc[i] = s_scale[(n0 + i) * 4 + tig], top[i] = kAttnNone, grow[i] = -INFINITY, sum[i] = 0.f;
    float o[2][NT];
    #pragma unroll
    for (int i = 0; i < NT; ++i) o[0][i] = o[1][i] = 0.f;

    #pragma unroll 1
    for (int at = run.s0; at < run.s1; at += TS) {
      cp_async_wait<0>();
      __syncthreads();  // the tile is there; the other stage and the weights of the last tile have been read
      const bool same = at + TS < run.s1;
      if (same || more) fetch(same ? row0 + at + TS : row1, same ? run.s1 - at - TS : left1, stage ^ 1);
      cp_async_commit();
      const unsigned char* tile = smem + stage * kStage;
      const int left = run.s1 - at;
      const bool partly = all_see < run.n && at + TS > all_see;  // a row may not see slots that others do
      if (partly) {
        uint32_t* sb = reinterpret_cast<uint32_t*>(smem + stage * kStage + kVsAt) + tid;
        if (kv4_large(*sb) && tid / (D / 32) >= all_see - at && kv4_infinite(*sb)) *sb = 0, s_grown[parity][4] = 1;
      }

      // scores of 16 slots and a part of the rows
      float acc[NG][4];
      #pragma unroll
      for (int w = 0; w < KW; ++w) {
        const unsigned char *pk = tile + k_at + attn_swizzle<D>(gid, tig * 2 + w / 4) * 16 + w % 4 * 4, *pc = tile + ks_at;
        const uint32_t wa = *reinterpret_cast<const uint32_t*>(pk), wb = *reinterpret_cast<const uint32_t*>(pk + 8 * (D / 2));
        const __half2 sa = *reinterpret_cast<const __half2*>(pc + w / 4 * 4);
        const __half2 sb = *reinterpret_cast<const __half2*>(pc + 8 * (D / 8) + w / 4 * 4);
        const __half2 sta = __low2half2(sa), bsa = __high2half2(sa), stb = __low2half2(sb), bsb = __high2half2(sb);
        uint32_t a[2][4];
        #pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t xa = wa >> 8 * y, xb = wb >> 8 * y;
          a[y][0] = kv4_pair<false>(xa, p.mul64, sta, bsa), a[y][1] = kv4_pair<false>(xb, p.mul64, stb, bsb);
          a[y][2] = kv4_pair<true>(xa, p.mul4, sta, bsa), a[y][3] = kv4_pair<true>(xb, p.mul4, stb, bsb);
        }
        #pragma unroll
        for (int i = 0; i < NG; ++i) {
          const uint4 q = qs[((n0 + i) * KW + w) * 32 + lane];
          if (w == 0)
            mma_f16_first(acc[i], a[0][0], a[0][1], a[0][2], a[0][3], q.x, q.y);
          else
            mma_f16(acc[i], a[0][0], a[0][1], a[0][2], a[0][3], q.x, q.y);
          mma_f16(acc[i], a[1][0], a[1][1], a[1][2], a[1][3], q.z, q.w);
        }
      }
      const bool some_hidden = left < TS || at + TS > all_see;
      if (kW) {  // rows of the chunk that are not there have a place too: only slots are checked, in a tile that is not whole
        float* to = p.score + ((static_cast<long long>(run.b) * walk.hc_count + run.hc) * RC + n0 * 4 + tig) * c.cap + at + st * 16 + gid;
        const long long next = 4 * c.cap;
        const int have = left - st * 16 - gid;
        if (left >= TS) {
          #pragma unroll
          for (int i = 0; i < NG; ++i, to += next) {
            to[0] = (acc[i][0] + acc[i][1]) * sc[i];
            to[8] = (acc[i][2] + acc[i][3]) * sc[i];
          }
        } else {
          #pragma unroll
          for (int i = 0; i < NG; ++i, to += next) {
            if (have > 0) to[0] = (acc[i][0] + acc[i][1]) * sc[i];
            if (have > 8) to[8] = (acc[i][2] + acc[i][3]) * sc[i];
          }
        }
      }
      // hidden slots, and whether a maximum has grown
      bool grown = false;
      float s[2][NG];
      #pragma unroll
      for (int i = 0; i < NG; ++i) {
        float s0 = acc[i][0] + acc[i][1], s1 = acc[i][2] + acc[i][3];
        if (some_hidden) {
          const int see = min(left, s_see[(n0 + i) * 4 + tig] - at) - st * 16;
          if (gid >= see) s0 = -INFINITY;
          if (gid + 8 >= see) s1 = -INFINITY;
        }
        s[0][i] = s0, s[1][i] = s1;
        const float best = fmaxf(s0, s1);
        grown |= best > grow[i];
      }
      if (named_bar_or(1 + share, 128, grown)) {  // the four warps that share these rows
        #pragma unroll
        for (int i = 0; i < NG; ++i) {
          float best = fmaxf(s[0][i], s[1][i]) * sc[i];
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 8));
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 16));
          if (gid == 0) s_max[st * RC + (n0 + i) * 4 + tig] = best;
        }
        named_bar_sync(1 + share, 128);
        #pragma unroll
        for (int i = 0; i < NG; ++i) {
          const int r = (n0 + i) * 4 + tig;
          const float best = fmaxf(fmaxf(s_max[r], s_max[RC + r]), fmaxf(s_max[2 * RC + r], s_max[3 * RC + r]));
          const float now = fmaxf(attn_top(best), top[i]), f = ex2(top[i] - now);
          top[i] = now, grow[i] = now > kAttnNone ? attn_limit(now) / sc[i] : -INFINITY, sum[i] *= f;
          if (st == 0 && gid == 0) s_fac[r] = f;
        }
        if (st == 0 && lane == 0) s_grown[parity][share] = 1;
      }
      #pragma unroll
      for (int i = 0; i < NG; ++i) {
        uint32_t pb[2];
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float e = ex2(fmaf(s[h][i], sc[i], -top[i]));
          sum[i] += e;
          const float big = __uint_as_float(__float_as_uint(e) & 0xFFFFE000u);
          pb[h] = transpose8x8(h2_bits(__floats2half2_rn(big, e - big)));
        }
        ps[(st * NT + n0 + i) * 32 + lane] = make_uint2(pb[0], pb[1]);
      }
      __syncthreads();  // the weights are there

      // output: this warp's columns, all slots
      #pragma unroll
      for (int g = 0; g < NT / NG; ++g) {
        if (s_grown[parity][g]) {
          #pragma unroll
          for (int i = 0; i < NG; ++i) {
            const float f = s_fac[(g * NG + i) * 4 + tig];
            o[0][g * NG + i] *= f, o[1][g * NG + i] *= f;
          }
        }
      }
      if (tid < 5) s_grown[parity ^ 1][tid] = 0;  // read last before this tile's first barrier
      // Tile 8 w + n is columns n of words 2 w and 2 w + 1 of the lane's; odd tiles are high nibbles.
      uint32_t a[4][4];
      #pragma unroll
      for (int u = 0; u < 4; ++u) {
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char* pc = tile + vs_at + (u * 16 + h * 8) * (D / 8);
          const uint32_t x = *reinterpret_cast<const uint32_t*>(pc), y = *reinterpret_cast<const uint32_t*>(pc + D / 8);
          const __half2 step = bits_h2(__byte_perm(x, y, 0x5410)), base = bits_h2(__byte_perm(x, y, 0x7632));
          #pragma unroll
          for (int z = 0; z < 2; ++z) {
            const int byte = ot % 8 / 2, off = (u * 16 + h * 8) * (D / 2) + (ot / 8 * 2 + z) * 4;
            const uint32_t wa = *reinterpret_cast<const uint32_t*>(tile + va_at + off);
            const uint32_t wb = *reinterpret_cast<const uint32_t*>(tile + vb_at + off);
            const uint32_t both = __byte_perm(wa, wb, byte | (byte + 4) << 8);
            a[u][2 * h + z] = h2_bits(__hfma2(bits_h2((both & nibbles) * to_top + 0x4C004C00u), step, base));  // kv4_pair
          }
        }
      }
      #pragma unroll
      for (int i = 0; i < NT; ++i) {
        float d[4];
        #pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint2 b = ps[(u * NT + i) * 32 + lane];
          if (u == 0)
            mma_f16_first(d, a[u][0], a[u][1], a[u][2], a[u][3], b.x, b.y);
          else
            mma_f16(d, a[u][0], a[u][1], a[u][2], a[u][3], b.x, b.y);
        }
        o[0][i] += d[0] + d[1], o[1][i] += d[2] + d[3];
      }
      if (partly && s_grown[parity][4]) {
        #pragma unroll 1
        for (int slot = max(all_see - at, 0); slot < min(left, TS); ++slot) {
          const uint32_t sb = __ldg(c.vs + (row0 + at + slot) * (D / kKv4Group) + gid * VW / 4);
          if (!kv4_infinite(sb)) continue;
          const uint32_t* words = reinterpret_cast<const uint32_t*>(
              tile + kVAt + slot * (D / 2) + attn_swizzle<D>(slot, v_in / 16) * 16 + v_in % 16) + ot / 8 * 2;
          const float v0 = kv4_value(words[0], ot % 8, sb), v1 = kv4_value(words[1], ot % 8, sb);
          const uint32_t* from = reinterpret_cast<const uint32_t*>(ps + slot / 16 * NT * 32 + 8 * tig + slot % 8 / 2) + slot / 8 % 2;
          #pragma unroll
          for (int i = 0; i < NT; ++i) {
            if (at + slot >= s_see[i * 4 + tig]) continue;
            const float w = kv4_weight(from[i * 64], from[i * 64 + 8], slot & 1);
            o[0][i] += w * v0, o[1][i] += w * v1;
          }
        }
      }
      stage ^= 1, parity ^= 1;
    }

    // the rows' sums and maxima, then the output or this CTA's part of it
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < NG; ++i) {
      #pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], x);
      const int r = (n0 + i) * 4 + tig;
      if (gid == 0) {
        s_sum[st * RC + r] = sum[i];
        if (st == 0) s_max[r] = top[i];
      }
    }
    __syncthreads();
    const bool whole = !run.enter && !run.leave;
    const int kind = run.enter ? 0 : 1;
    float* part = p.part + (static_cast<long long>(cta) * 2 + kind) * kPart;
    for (int r = tid; r < RC; r += kRowsThreads) {
      const float l = s_sum[r] + s_sum[RC + r] + s_sum[2 * RC + r] + s_sum[3 * RC + r];
      if (!whole) {
        part[r] = s_max[r], part[RC + r] = l;
      } else {
        s_fac[r] = l != 0.f ? 1.f / l : 0.f;
        if (kW && r < rows) attn_put_norm(p, c, run, run.r0 + r, s_max[r], s_fac[r]);
      }
    }
    if (!whole) {
      #pragma unroll
      for (int i = 0; i < NT; ++i)
        #pragma unroll
        for (int h = 0; h < 2; ++h) part[2 * RC + ((ot * 2 + h) * NT + i) * 32 + lane] = o[h][i];
    } else {
      // Through shared memory, where the queries were, as rows: a lane's columns lie 16 or 32 apart, and 32 stores to 32
      // sectors each took 18 us for 80 rows of 256. Columns are moved so that few lanes share a bank.
      float* out = reinterpret_cast<float*>(qs);  // [RC][D], the queries' size
      auto place = [&](int r, int col) { return r * D + (col ^ ((col >> 5) | (r & 3) << 3)); };
      #pragma unroll
      for (int i = 0; i < NT; ++i)
        #pragma unroll
        for (int h = 0; h < 2; ++h)
          out[place(i * 4 + tig, attn_col<D, NT>(((ot * 2 + h) * NT + i) * 32 + lane))] = o[h][i];
      __syncthreads();
      for (int r = warp; r < rows; r += kRowsWarps) {
        float* to = p.out + attn_row_at<D>(p, run, run.r0 + r, p.ldo);
        const float inv = s_fac[r];
        #pragma unroll
        for (int x = 0; x < D; x += 32) to[x + lane] = out[place(r, x + lane)] * inv;
      }
    }
    if (tid == 0 && !run.enter) {
      if (whole)
        p.split[run.b * walk.hc_count + run.hc] = make_int2(cta, 1);
      else
        attn_put_split(p, run, walk.hc_count, cta, each, extra);
    }
    if (!more) break;
    row0 = row1 - nxt.s0;
    run = nxt;
  }
  cp_async_wait<0>();
}

}  // namespace vmlm
