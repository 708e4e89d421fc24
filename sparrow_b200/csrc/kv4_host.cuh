// kv4_host.cuh -- host side of the 4-bit cache's entry points: argument checks,
// kernel choice and launches. Included by vmlm_cuda.cu behind the contexts and
// launch helpers.
#pragma once

namespace {

constexpr size_t kKv4MaxDim = static_cast<size_t>(1) << 31;
constexpr size_t kKv4MaxSlots = kKv4MaxDim - 8192;  // slots are ints, and a kernel's walk goes up to a block's step past them

int kv4_check(const char* what, const vmlm_kv4* c) {
  if (!c) return fail(VMLM_ERR_ARG, "%s: null cache", what);
  if (c->d != 64 && c->d != 128 && c->d != 256)
    return fail(VMLM_ERR_SHAPE, "%s: head size %zu (64, 128 and 256 are built)", what, c->d);
  if (c->n_kv == 0) return fail(VMLM_ERR_ARG, "%s: no kv heads", what);
  if (c->n_seq >= kKv4MaxDim || c->n_kv >= kKv4MaxDim || c->n_seq * c->n_kv >= kKv4MaxDim)
    return fail(VMLM_ERR_SHAPE, "%s: n_seq * n_kv must be < 2^31", what);
  if (c->cap > kKv4MaxSlots) return fail(VMLM_ERR_SHAPE, "%s: cap must be at most 2^31 - 8192", what);
  if (c->n_seq > 0 && c->cap > 0) {
    if (!c->k || !c->v || !c->ks || !c->vs) return fail(VMLM_ERR_ARG, "%s: null pointer in the cache", what);
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->ks) || !aligned16(c->vs))
      return fail(VMLM_ERR_ARG, "%s: the cache's buffers must start on a 16-byte boundary", what);
  }
  return VMLM_OK;
}

Kv4View kv4_view(const vmlm_kv4* c) {
  Kv4View v;
  v.k = static_cast<uint8_t*>(c->k);
  v.v = static_cast<uint8_t*>(c->v);
  v.ks = static_cast<uint32_t*>(c->ks);
  v.vs = static_cast<uint32_t*>(c->vs);
  v.cap = static_cast<long long>(c->cap);
  v.n_seq = static_cast<int>(c->n_seq);
  v.n_kv = static_cast<int>(c->n_kv);
  return v;
}

// A [tokens] x [heads * d] activation argument with row stride ld.
int kv4_check_rows(const char* what, const char* name, const float* x, size_t ld, size_t heads, size_t d) {
  if (!x) return fail(VMLM_ERR_ARG, "%s: %s is null", what, name);
  if (ld < heads * d) return fail(VMLM_ERR_ARG, "%s: row stride of %s is %zu, below %zu", what, name, ld, heads * d);
  return VMLM_OK;
}

bool kv4_vec(const float* x, size_t ld) { return !x || (aligned16(x) && ld % 4 == 0); }

bool kv4_overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + nb && y < x + na;
}

// Whether `rows` rows of wa values at a (lda apart) and of wb values at b share a byte. Slices of one wider matrix may lie
// between each other's rows; with different strides, spans that meet count as shared.
bool kv4_rows_overlap(const float* a, size_t lda, size_t wa, const float* b, size_t ldb, size_t wb, size_t rows) {
  if (rows == 0 || wa == 0 || wb == 0) return false;
  if (rows == 1 || lda != ldb) return kv4_overlap(a, ((rows - 1) * lda + wa) * 4, b, ((rows - 1) * ldb + wb) * 4);
  if (b < a) std::swap(a, b), std::swap(wa, wb);
  const size_t off = reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a), ld = lda * 4;
  const size_t down = off / ld, in = off % ld;  // b's first row begins `in` bytes into a's row `down`
  return (down < rows && in < wa * 4) || (down + 1 < rows && in + wb * 4 > ld);
}

// The written rows `to` of heads that are read from `from`: in place, or apart.
int kv4_check_out(const char* what, const char* name, const float* to, size_t ldt, const float* from, size_t ldf, size_t width,
                  size_t rows) {
  if (to == from && (ldt == ldf || rows == 1)) return VMLM_OK;
  if (kv4_rows_overlap(to, ldt, width, from, ldf, width, rows))
    return fail(VMLM_ERR_ARG, "%s: %so and %s overlap and are not the same rows", what, name, name);
  return VMLM_OK;
}

int kv4_check_rope(const char* what, const vmlm_rope* r, size_t d) {
  if (!r) return VMLM_OK;
  if (!r->cos_t || !r->sin_t || !r->pos) return fail(VMLM_ERR_ARG, "%s: null pointer in the rotation", what);
  if (r->rot == 0 || r->rot % 16 != 0 || r->rot > d)
    return fail(VMLM_ERR_ARG, "%s: rot is %zu: a multiple of 16 up to %zu is wanted", what, r->rot, d);
  if (r->n_pos == 0 || r->n_pos >= kKv4MaxDim) return fail(VMLM_ERR_ARG, "%s: n_pos is %zu", what, r->n_pos);
  return VMLM_OK;
}

template <int D, bool kCache>
int kv4_launch_rows_d(Ctx* ctx, Kv4Rows p, const Kv4View& v, cudaStream_t st) {
  const long long heads = p.n_q + p.n_kv + (kCache ? p.n_kv : 0);
  // Steps of 256 / d rows a warp: as many as leave every SM 64 warps, so that a token's table rows and addresses are
  // shared by more rows (2047 tokens of 40 heads of 128: 19.5 us with 64, 20.2 with 128, 20.2 to 22 with 32).
  const long long all = cdiv(heads, 256 / D);
  p.steps = static_cast<int>(std::max<long long>(1, std::min<long long>(all, p.tokens * all / (ctx->sms * 64ll))));
  p.sets = static_cast<uint32_t>(cdiv(all, p.steps));
  p.steps = static_cast<int>(cdiv(all, p.sets));  // evenly
  const long long warps = p.tokens * p.sets;
  if (warps == 0) return VMLM_OK;
  if (warps >= static_cast<long long>(kKv4MaxDim))
    return fail(VMLM_ERR_SHAPE, "tokens x heads is too large (%lld rows)", p.tokens * heads);
  p.vec_g = (!p.gq || aligned16(p.gq)) && (!p.gk || aligned16(p.gk));
  p.vec_t = aligned16(p.cos_t) && aligned16(p.sin_t);  // rot is a multiple of 16, so rows of the table are too
  return launch(kv4_rows_kernel<D, kCache>, dim3(static_cast<unsigned>(cdiv(warps, 8))), dim3(256), 0, st, true, p, v,
                ctx->err);
}

template <bool kCache>
int kv4_launch_rows(Ctx* ctx, const Kv4Rows& p, const Kv4View& v, size_t d, cudaStream_t st) {
  if (d == 64) return kv4_launch_rows_d<64, kCache>(ctx, p, v, st);
  if (d == 128) return kv4_launch_rows_d<128, kCache>(ctx, p, v, st);
  return kv4_launch_rows_d<256, kCache>(ctx, p, v, st);
}

template <int D>
int kv4_launch_evict(Ctx* ctx, Kv4Evict p, const Kv4View& s, const Kv4View& d, cudaStream_t st) {
  static bool set[64] = {};
  if (ctx->dev < 64 && !set[ctx->dev]) {
    VMLM_CUDA(cudaFuncSetAttribute(kv4_evict_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   evict_smem_bytes(kEvictKeys)));
    set[ctx->dev] = true;
  }
  // CTAs a head: as many as two an SM have room for, while each still has kEvictShare slots: below, the barriers of a
  // cluster cost more than the work that it divides.
  const long long heads = static_cast<long long>(s.n_seq) * s.n_kv;
  int size = 1;
  while (size < kEvictMaxCluster && heads * size <= ctx->sms && s.cap > kEvictShare * size) size *= 2;
  p.keys = static_cast<int>(std::min<long long>(kEvictKeys, cdiv(s.cap, size)));
  return launch_ex(kv4_evict_kernel<D>, dim3(size, static_cast<unsigned>(heads)), dim3(kEvictThreads),
                   evict_smem_bytes(p.keys), st, true, size, p, s, d, ctx->err);
}

void kv4_set_rope(Kv4Rows* p, const vmlm_rope* r) {
  if (!r) return;
  p->cos_t = r->cos_t;
  p->sin_t = r->sin_t;
  p->pos = r->pos;
  p->n_pos = static_cast<long long>(r->n_pos);
  p->rot = static_cast<int>(r->rot);
  p->interleaved = r->interleaved;
}

// The launches behind the attention kernel: the join of items that several CTAs had parts of (`whole`: there can be none,
// whatever the lengths are), and the weights of a call with w_out.
template <int D, int NT, bool kW>
int kv4_launch_finish(const Kv4Attn& p, const Kv4View& v, bool whole, cudaStream_t st) {
  const long long heads = static_cast<long long>(v.n_seq) * v.n_kv;
  const long long joins = heads * p.chunks * (4 * NT * D / 128), blocks = cdiv(v.cap, kWeightThreads * (p.rows <= kWeightFewRows ? 4 : 1));
  if (joins >= static_cast<long long>(kKv4MaxDim) || heads * blocks >= static_cast<long long>(kKv4MaxDim))
    return fail(VMLM_ERR_SHAPE, "kv4_attn_dev: n_seq * n_q * m * cap is too large");
  if (!whole && joins > 0)
    VMLM_TRY(launch(kv4_join_kernel<D, NT, kW>, dim3(static_cast<unsigned>(joins)), dim3(kJoinWarps * 32), 0, st, true, p, v));
  if (!kW || heads * blocks == 0) return VMLM_OK;
  return launch(p.rows <= kWeightFewRows ? kv4_weights_kernel<4> : kv4_weights_kernel<1>,
                dim3(static_cast<unsigned>(heads * blocks)), dim3(kWeightThreads), 0, st, true, p, v, static_cast<int>(blocks));
}

// Workspace and limits that both kernels share: nt fours of rows a chunk at most, `grid` CTAs, tiles of `tile` slots.
int kv4_prepare_attn(Ctx* ctx, Kv4Attn* p, const Kv4View& v, int nt, int d, int grid, int tile) {
  const size_t heads = static_cast<size_t>(v.n_seq) * v.n_kv;
  p->chunks = static_cast<int>(cdiv(p->rows, 4 * nt));
  p->chunk_rows = static_cast<int>(cdiv(cdiv(p->rows, p->chunks), 4)) * 4;  // even chunks
  p->kept_rows = 4 * nt;
  p->mul4 = 4, p->mul64 = 64;
  if (heads * p->chunks * static_cast<size_t>(cdiv(v.cap, tile) + 4) >= kKv4MaxDim)  // units, with a run's cost
    return fail(VMLM_ERR_SHAPE, "kv4_attn_dev: n_seq * n_q * m * cap is too large");
  VMLM_TRY(ensure(ctx->kv4_part, static_cast<size_t>(grid) * 2 * 4 * nt * (d + 2) * 4));
  VMLM_TRY(ensure(ctx->kv4_split, heads * p->chunks * sizeof(int2)));
  p->part = static_cast<float*>(ctx->kv4_part.p);
  p->split = static_cast<int2*>(ctx->kv4_split.p);
  if (p->w_out) {
    if (static_cast<double>(heads) * p->chunks * p->kept_rows * static_cast<double>(v.cap) > 2.5e11)
      return fail(VMLM_ERR_SHAPE, "kv4_attn_dev: the scores of a call with w_out take %.3g bytes",
                  4.0 * static_cast<double>(heads) * p->chunks * p->kept_rows * static_cast<double>(v.cap));
    VMLM_TRY(ensure(ctx->kv4_norm, heads * p->rows * sizeof(float2)));
    VMLM_TRY(ensure(ctx->kv4_score, heads * p->chunks * p->kept_rows * static_cast<size_t>(v.cap) * 4));
    p->norm = static_cast<float2*>(ctx->kv4_norm.p);
    p->score = static_cast<float*>(ctx->kv4_score.p);
  }
  return VMLM_OK;
}

template <int D, int NT, bool kW, bool kSeveral = true>
int kv4_launch_attn(Ctx* ctx, Kv4Attn p, const Kv4View& v, cudaStream_t st) {
  if constexpr (NT == 1 && kSeveral)
    if (p.m == 1) return kv4_launch_attn<D, NT, kW, false>(ctx, p, v, st);
  constexpr int kSmem = attn_smem_bytes(D, NT);
  static bool set[64] = {};
  if (ctx->dev < 64 && !set[ctx->dev]) {
    VMLM_CUDA(cudaFuncSetAttribute(kv4_attn_kernel<D, NT, kW, kSeveral>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    set[ctx->dev] = true;
  }
  const int grid = ctx->sms;
  VMLM_TRY(kv4_prepare_attn(ctx, &p, v, NT, D, grid, 4096 / D));
  // An item of t tiles takes a CTA t / kWarps alone and items / grid times that shared: alone while that saves no tile.
  const long long items = static_cast<long long>(v.n_seq) * v.n_kv * p.chunks, spare = grid - items;
  constexpr int kWarps = attn_warps(D, NT);
  p.alone = static_cast<int>(spare < 0 ? 0 : spare * kAttnAlone <= grid ? kWarps * kAttnAlone : kWarps * grid / spare);
  VMLM_TRY(launch(kv4_attn_kernel<D, NT, kW, kSeveral>, dim3(grid), dim3(kWarps * 32), kSmem, st, true, p, v, ctx->err));
  const bool whole = spare >= 0 && v.cap <= static_cast<long long>(p.alone) * (4096 / D);
  return kv4_launch_finish<D, NT, kW>(p, v, whole, st);
}

template <int NT, bool kW>
int kv4_launch_attn_rows(Ctx* ctx, Kv4Attn p, const Kv4View& v, cudaStream_t st) {
  constexpr int D = kRowsHead, kSmem = rows_smem_bytes(NT);
  static bool set[64] = {};
  if (ctx->dev < 64 && !set[ctx->dev]) {
    VMLM_CUDA(cudaFuncSetAttribute(kv4_attn_rows_kernel<NT, kW>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    set[ctx->dev] = true;
  }
  const int grid = ctx->sms;
  VMLM_TRY(kv4_prepare_attn(ctx, &p, v, NT, D, grid, kRowsSlots));
  VMLM_TRY(launch(kv4_attn_rows_kernel<NT, kW>, dim3(grid), dim3(kRowsWarps * 32), kSmem, st, true, p, v, ctx->err));
  return kv4_launch_finish<D, NT, kW>(p, v, v.cap <= kRowsSlots, st);
}

// A warp takes 4 to 4 * attn_most rows at a time: as few as leave no warp more than a tile, so that short caches spread
// their rows over the SMs (d = 64, 4 x 8 heads of 512 slots, 12 rows: 7.6 us as 4 + 4 + 4, 11.3 as 12), else as many as
// its registers hold, in even chunks (16 x 8 heads of 8192 slots, 12 rows: 42 us as 12, 53 as 8 + 4). d = 256 holds 4
// rows; there a CTA shares what it unpacks if rows and tiles a CTA are many: with 8 heads of 8192 slots and 16 sequences,
// 28 rows take 412 us so and 435 by fours, 80 rows 743 and 1333, 20 rows 405 and 313; 80 rows over 16 ragged caches of
// up to 3001 slots take 46 us and 53, over 32 of 1024 (3.5 tiles a CTA) 67 and 58, over 64 ragged ones of up to 1024 79 and
// 80 (all full 108 and 105). The tiles are those of cap, which the host knows, not of the lengths: over 8 ragged caches of up
// to 3001 slots (2.5 tiles a CTA) it would win by 29 against 34, over 8 full ones it ties (43). Its chunks of 80 rows leave too few
// CTAs work below twice as many tiles (the ragged caches: 47.6 us as one chunk).
template <int D, bool kW>
int kv4_pick_attn(Ctx* ctx, const Kv4Attn& p, const Kv4View& v, cudaStream_t st) {
  if constexpr (D == 256) {
    const long long tiles = static_cast<long long>(v.n_seq) * v.n_kv * cdiv(v.cap, kRowsSlots);
    if (p.rows >= kAttnManyRows && tiles >= 5ll * ctx->sms) {
      const long long chunks = cdiv(p.rows, 4 * (tiles >= 10ll * ctx->sms ? kRowsMost : 16)), fours = cdiv(cdiv(p.rows, chunks), 4);
      if (fours <= 8) return kv4_launch_attn_rows<8, kW>(ctx, p, v, st);
      if (fours <= 12) return kv4_launch_attn_rows<12, kW>(ctx, p, v, st);
      if (fours <= 16) return kv4_launch_attn_rows<16, kW>(ctx, p, v, st);
      return kv4_launch_attn_rows<20, kW>(ctx, p, v, st);
    }
    return kv4_launch_attn<D, 1, kW>(ctx, p, v, st);
  } else {
    const long long heads = static_cast<long long>(v.n_seq) * v.n_kv, tiles = cdiv(v.cap, 4096 / D);
    const long long chunks = cdiv(p.rows, 4 * attn_most(D));
    int nt = static_cast<int>(cdiv(cdiv(p.rows, chunks), 4));
    for (int n = 1; n < nt; ++n) {
      const long long items = heads * cdiv(p.rows, 4 * n);
      if (items <= ctx->sms && items * tiles <= static_cast<long long>(ctx->sms) * attn_warps(D, n)) nt = n;
    }
    if (nt <= 1) return kv4_launch_attn<D, 1, kW>(ctx, p, v, st);
    if (nt == 2 || D == 128) return kv4_launch_attn<D, 2, kW>(ctx, p, v, st);
    if constexpr (D == 64) {
      if (nt == 3) return kv4_launch_attn<D, 3, kW>(ctx, p, v, st);
      return kv4_launch_attn<D, 4, kW>(ctx, p, v, st);
    }
    return VMLM_OK;
  }
}
}  // namespace

extern "C" {

int vmlm_qk_norm_rope_dev(const float* q, size_t ldq, const float* k, size_t ldk, const float* gq, const float* gk,
                          float eps, const vmlm_rope* rope, float* qo, size_t ldqo, float* ko, size_t ldko,
                          size_t tokens, size_t n_q, size_t n_kv, size_t d, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  const char* what = "qk_norm_rope_dev";
  if (d != 64 && d != 128 && d != 256)
    return fail(VMLM_ERR_SHAPE, "%s: head size %zu (64, 128 and 256 are built)", what, d);
  if (tokens >= kKv4MaxDim || n_q >= 65536 || n_kv >= 65536)
    return fail(VMLM_ERR_SHAPE, "%s: tokens must be < 2^31 and heads < 65536", what);
  VMLM_TRY(kv4_check_rope(what, rope, d));
  if (tokens == 0 || n_q + n_kv == 0) return VMLM_OK;
  if (n_q > 0) {
    VMLM_TRY(kv4_check_rows(what, "q", q, ldq, n_q, d));
    VMLM_TRY(kv4_check_rows(what, "qo", qo, ldqo, n_q, d));
  }
  if (n_kv > 0) {
    VMLM_TRY(kv4_check_rows(what, "k", k, ldk, n_kv, d));
    VMLM_TRY(kv4_check_rows(what, "ko", ko, ldko, n_kv, d));
  }
  if (n_q > 0) VMLM_TRY(kv4_check_out(what, "q", qo, ldqo, q, ldq, n_q * d, tokens));
  if (n_kv > 0) VMLM_TRY(kv4_check_out(what, "k", ko, ldko, k, ldk, n_kv * d, tokens));
  if (n_q > 0 && n_kv > 0 &&
      (kv4_rows_overlap(qo, ldqo, n_q * d, k, ldk, n_kv * d, tokens) || kv4_rows_overlap(ko, ldko, n_kv * d, q, ldq, n_q * d, tokens) ||
       kv4_rows_overlap(qo, ldqo, n_q * d, ko, ldko, n_kv * d, tokens)))
    return fail(VMLM_ERR_ARG, "%s: queries and keys overlap", what);
  Ctx* ctx = nullptr;
  VMLM_TRY(current_ctx(&ctx));
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  Kv4Rows p = {};
  p.q = q, p.k = k, p.qo = qo, p.ko = ko, p.gq = gq, p.gk = gk, p.eps = eps;
  p.ldq = ldq, p.ldk = ldk, p.ldqo = ldqo, p.ldko = ldko;
  p.tokens = tokens, p.m = tokens;
  p.n_q = static_cast<int>(n_q), p.n_kv = static_cast<int>(n_kv);
  kv4_set_rope(&p, rope);
  p.vec = (n_q == 0 || (kv4_vec(q, ldq) && kv4_vec(qo, ldqo))) && (n_kv == 0 || (kv4_vec(k, ldk) && kv4_vec(ko, ldko)));
  return kv4_launch_rows<false>(ctx, p, Kv4View{}, d, st);
}

int vmlm_kv4_append_dev(const vmlm_kv4* cache, const float* q, size_t ldq, float* qo, size_t ldqo, size_t n_q,
                        const float* k, size_t ldk, const float* v, size_t ldv, const float* gq, const float* gk,
                        float eps, const vmlm_rope* rope, const int32_t* len, size_t m, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  const char* what = "kv4_append_dev";
  VMLM_TRY(kv4_check(what, cache));
  VMLM_TRY(kv4_check_rope(what, rope, cache->d));
  if (m >= kKv4MaxDim || cache->n_seq * m >= kKv4MaxDim || n_q >= 65536 || cache->n_kv >= 65536)
    return fail(VMLM_ERR_SHAPE, "%s: tokens must be < 2^31 and heads < 65536", what);
  if (m == 0 || cache->n_seq == 0) return VMLM_OK;
  if (cache->cap == 0) return fail(VMLM_ERR_ARG, "%s: the cache has no slots", what);
  if (!len) return fail(VMLM_ERR_ARG, "%s: len is null", what);
  VMLM_TRY(kv4_check_rows(what, "k", k, ldk, cache->n_kv, cache->d));
  VMLM_TRY(kv4_check_rows(what, "v", v, ldv, cache->n_kv, cache->d));
  if (n_q > 0) {
    VMLM_TRY(kv4_check_rows(what, "q", q, ldq, n_q, cache->d));
    VMLM_TRY(kv4_check_rows(what, "qo", qo, ldqo, n_q, cache->d));
    const size_t tokens = cache->n_seq * m, wq = n_q * cache->d, wk = cache->n_kv * cache->d;
    VMLM_TRY(kv4_check_out(what, "q", qo, ldqo, q, ldq, wq, tokens));
    if (kv4_rows_overlap(qo, ldqo, wq, k, ldk, wk, tokens) || kv4_rows_overlap(qo, ldqo, wq, v, ldv, wk, tokens))
      return fail(VMLM_ERR_ARG, "%s: qo overlaps k or v", what);
  }
  Ctx* ctx = nullptr;
  VMLM_TRY(current_ctx(&ctx));
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  Kv4Rows p = {};
  p.q = q, p.k = k, p.v = v, p.qo = qo, p.gq = gq, p.gk = gk, p.eps = eps;
  p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldqo = ldqo;
  p.tokens = cache->n_seq * m, p.m = m, p.len = len;
  p.n_q = static_cast<int>(n_q), p.n_kv = static_cast<int>(cache->n_kv);
  kv4_set_rope(&p, rope);
  p.vec = (n_q == 0 || (kv4_vec(q, ldq) && kv4_vec(qo, ldqo))) && kv4_vec(k, ldk) && kv4_vec(v, ldv);
  return kv4_launch_rows<true>(ctx, p, kv4_view(cache), cache->d, st);
}

int vmlm_kv4_read_dev(const vmlm_kv4* cache, const int32_t* start, const int32_t* end, size_t count, uint16_t* k,
                      uint16_t* v, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  const char* what = "kv4_read_dev";
  VMLM_TRY(kv4_check(what, cache));
  if (count > kKv4MaxSlots) return fail(VMLM_ERR_SHAPE, "%s: count must be at most 2^31 - 8192", what);
  if (count == 0 || cache->n_seq == 0) return VMLM_OK;
  if (!start || !end || !k || !v) return fail(VMLM_ERR_ARG, "%s: null pointer", what);
  if (!aligned16(k) || !aligned16(v)) return fail(VMLM_ERR_ARG, "%s: k and v must start on a 16-byte boundary", what);
  Ctx* ctx = nullptr;
  VMLM_TRY(current_ctx(&ctx));
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const Kv4View c = kv4_view(cache);
  const long long words = static_cast<long long>(count) * static_cast<long long>(cache->d / 8);
  const long long blocks = cdiv(words, 256 * kReadWords);
  if (blocks >= static_cast<long long>(kKv4MaxDim)) return fail(VMLM_ERR_SHAPE, "%s: count is too large", what);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min<long long>(static_cast<long long>(c.n_seq) * c.n_kv, 65535)));
  const int n = static_cast<int>(count);
  __half *ko = reinterpret_cast<__half*>(k), *vo = reinterpret_cast<__half*>(v);
  if (cache->d == 64) return launch(kv4_read_kernel<64>, grid, dim3(256), 0, st, true, c, start, end, n, ko, vo, ctx->err);
  if (cache->d == 128) return launch(kv4_read_kernel<128>, grid, dim3(256), 0, st, true, c, start, end, n, ko, vo, ctx->err);
  return launch(kv4_read_kernel<256>, grid, dim3(256), 0, st, true, c, start, end, n, ko, vo, ctx->err);
}

int vmlm_kv4_attn_dev(const vmlm_kv4* cache, const float* q, size_t ldq, const int32_t* len, float* out, size_t ldo,
                      size_t m, size_t n_q, float scale, const float* w_in, float* w_out, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  const char* what = "kv4_attn_dev";
  VMLM_TRY(kv4_check(what, cache));
  if (n_q % cache->n_kv != 0)
    return fail(VMLM_ERR_SHAPE, "%s: %zu query heads do not share %zu kv heads evenly", what, n_q, cache->n_kv);
  if (n_q >= 65536 || m >= kKv4MaxDim || cache->n_seq * m >= kKv4MaxDim ||  // in steps: three factors can wrap
      cache->n_seq * m * n_q >= kKv4MaxDim)
    return fail(VMLM_ERR_SHAPE, "%s: n_seq * m * n_q must be < 2^31 and n_q < 65536", what);
  if (m == 0 || n_q == 0 || cache->n_seq == 0) return VMLM_OK;
  if (!len) return fail(VMLM_ERR_ARG, "%s: len is null", what);
  if (w_in && !w_out) return fail(VMLM_ERR_ARG, "%s: w_in without w_out", what);
  VMLM_TRY(kv4_check_rows(what, "q", q, ldq, n_q, cache->d));
  VMLM_TRY(kv4_check_rows(what, "out", out, ldo, n_q, cache->d));
  // A part of an item may read its queries when another part's result is written, and weights before they are replaced.
  if (kv4_rows_overlap(out, ldo, n_q * cache->d, q, ldq, n_q * cache->d, cache->n_seq * m))
    return fail(VMLM_ERR_ARG, "%s: out overlaps q", what);
  const size_t w_bytes = cache->n_seq * cache->n_kv * cache->cap * 4;
  if (w_in && w_in != w_out && kv4_overlap(w_in, w_bytes, w_out, w_bytes))
    return fail(VMLM_ERR_ARG, "%s: w_in and w_out overlap and are not the same", what);
  Ctx* ctx = nullptr;
  VMLM_TRY(current_ctx(&ctx));
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  Kv4Attn p = {};
  p.q = q, p.out = out, p.ldq = ldq, p.ldo = ldo, p.len = len, p.w_in = w_in, p.w_out = w_out;
  int e = 0;
  p.scale_m = static_cast<float>(2 * std::frexp(scale * 1.44269504088896340736, &e));
  p.scale_e = std::isfinite(scale) ? e - 1 : 0;
  p.m = static_cast<int>(m), p.n_q = static_cast<int>(n_q);
  p.group = static_cast<int>(n_q / cache->n_kv);
  p.rows = p.m * p.group;
  p.vec = kv4_vec(q, ldq);
  const Kv4View v = kv4_view(cache);
  if (cache->d == 64) return w_out ? kv4_pick_attn<64, true>(ctx, p, v, st) : kv4_pick_attn<64, false>(ctx, p, v, st);
  if (cache->d == 128) return w_out ? kv4_pick_attn<128, true>(ctx, p, v, st) : kv4_pick_attn<128, false>(ctx, p, v, st);
  return w_out ? kv4_pick_attn<256, true>(ctx, p, v, st) : kv4_pick_attn<256, false>(ctx, p, v, st);
}

int vmlm_kv4_evict_dev(const vmlm_kv4* src, const vmlm_kv4* dst, const float* w, const int32_t* len, size_t keep,
                       size_t first, size_t recent, int32_t* idx, float* w_out, int32_t* len_out, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  const char* what = "kv4_evict_dev";
  VMLM_TRY(kv4_check(what, src));
  VMLM_TRY(kv4_check(what, dst));
  if (src->n_seq != dst->n_seq || src->n_kv != dst->n_kv || src->d != dst->d)
    return fail(VMLM_ERR_SHAPE, "%s: the two caches differ in n_seq, n_kv or d", what);
  if (keep > dst->cap) return fail(VMLM_ERR_SHAPE, "%s: keep is %zu, dst holds %zu slots", what, keep, dst->cap);
  if (keep * (src->d / 32) > kKv4MaxSlots)
    return fail(VMLM_ERR_SHAPE, "%s: keep * d / 32 must be at most 2^31 - 8192", what);
  if (first > keep || recent > keep - first)
    return fail(VMLM_ERR_ARG, "%s: first + recent is above keep (%zu + %zu, %zu)", what, first, recent, keep);
  if (src->n_seq == 0) return VMLM_OK;
  if (!len || !len_out || (keep > 0 && (!w || !idx))) return fail(VMLM_ERR_ARG, "%s: null pointer", what);
  // CTAs of other heads read lengths, weights and rows while one writes: nothing is done in place.
  struct Span {
    const void* at;
    size_t bytes;
  };
  const size_t heads = src->n_seq * src->n_kv, rs = heads * src->cap, rd = heads * dst->cap, codes = src->d / 2, sb = src->d / 8;
  const Span read[6] = {{src->k, rs * codes}, {src->v, rs * codes}, {src->ks, rs * sb}, {src->vs, rs * sb}, {w, keep ? rs * 4 : 0},
                        {len, src->n_seq * 4}};
  const Span written[7] = {{dst->k, rd * codes}, {dst->v, rd * codes}, {dst->ks, rd * sb}, {dst->vs, rd * sb},
                           {idx, heads * keep * 4}, {w_out, w_out ? heads * keep * 4 : 0}, {len_out, src->n_seq * 4}};
  for (int i = 0; i < 7; ++i) {
    for (int j = 0; j < 6; ++j)
      if (kv4_overlap(written[i].at, written[i].bytes, read[j].at, read[j].bytes))
        return fail(VMLM_ERR_ARG, i < 4 && j < 4 ? "%s: src and dst overlap" : "%s: an output overlaps an input", what);
    for (int j = 0; j < i; ++j)
      if (kv4_overlap(written[i].at, written[i].bytes, written[j].at, written[j].bytes))
        return fail(VMLM_ERR_ARG, "%s: two outputs overlap", what);
  }
  Ctx* ctx = nullptr;
  VMLM_TRY(current_ctx(&ctx));
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const Kv4View s = kv4_view(src), d = kv4_view(dst);
  if (static_cast<long long>(s.n_seq) * s.n_kv >= 65536)
    return fail(VMLM_ERR_SHAPE, "%s: n_seq * n_kv must be < 65536", what);
  Kv4Evict p = {};
  p.w = w, p.len = len, p.idx = idx, p.w_out = w_out, p.len_out = len_out;
  p.keep = static_cast<int>(keep), p.first = static_cast<int>(first), p.recent = static_cast<int>(recent);
  if (src->d == 64) return kv4_launch_evict<64>(ctx, p, s, d, st);
  if (src->d == 128) return kv4_launch_evict<128>(ctx, p, s, d, st);
  return kv4_launch_evict<256>(ctx, p, s, d, st);
}

}  // extern "C"
