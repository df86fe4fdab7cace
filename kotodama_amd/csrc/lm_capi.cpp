// Host side of the language-model operators of libattnres_hip.so: argument
// checks, launch shapes and launches of the kernels in attention_kernels.hip
// and lm_kernels.hip.  As in attnres_capi.cpp: no allocation, no
// synchronisation, every argument checked before any HIP call.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>

#include "attnres.h"
#include "attnres_internal.h"
#include "lm_host.h"
#include "lm_params.h"

namespace {

// Code-object parts and kernel slots.
constexpr int kLmPart = 12, kAttnBf16Part = 13, kAttnF32Part = 14;
enum Slot {
  kAttnFwd = 0,                // + 12 * (fp32) + 3 * ((head_dim - 1) / 32) + log2 of the waves that share rows
  kAttnDq = kAttnFwd + 24,
  kAttnDkv = kAttnDq + 24,
  kAttnJoin = kAttnDkv + 24,   // + (fp32)
  kRopeFwd = kAttnJoin + 2,    // + 4 * (fp32) + 2 * (scalar) + (4 heads per lane group)
  kRopeBwd = kRopeFwd + 8,     // + 2 * (fp32) + (scalar)
  kRopeDw = kRopeBwd + 4,      // + (fp32)
  kEmbedFwd = kRopeDw + 2,     // + 2 * (fp32) + (scalar)
  kEmbedSum = kEmbedFwd + 4,
  kEmbedJoin = kEmbedSum + 4,  // + (fp32)
  kEmbedSort = kEmbedJoin + 2,
  kSlots
};
static_assert(kSlots <= kServingSlots, "kernel slots");

constexpr int64_t kMaxLen = (int64_t)1 << 30;  // tokens of one sequence
constexpr int kSplitPerCu = 2;                 // workgroups per CU to split the key axis into
constexpr int64_t kMaxTokenStride = (int64_t)32 << 20;  // bytes
constexpr int kMaxGroup = 4096;                // query heads per key head

// A tensor argument's strides; dimensions of one element have none.
int take_strides(const char* what, const void* p, const int64_t* st, int64_t nb, int64_t nh, int64_t nt, int es,
                 int align, lm_strides* out) {
  if (p == nullptr || st == nullptr) return fail(ATTNRES_ERR_ARG, "%s or its strides are NULL", what);
  out->b = nb > 1 ? st[0] : 0;
  out->h = nh > 1 ? st[1] : 0;
  out->t = nt > 1 ? st[2] : 0;
  const int64_t m = align / es;
  if (!aligned(p, align) || (m > 1 && (out->b % m || out->h % m || out->t % m)))
    return fail(ATTNRES_ERR_ALIGN, "%s: pointer and strides must be multiples of %d bytes", what, align);
  return ATTNRES_OK;
}

// ------------------------------------------------------------- attention --

int check_attention(int batch, int heads, int kv_heads, int64_t q_len, int64_t kv_slots, int head_dim, int dtype) {
  if (!valid_dtype(dtype)) return fail(ATTNRES_ERR_ARG, "attention: bad dtype %d", dtype);
  if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || q_len < 0 || kv_slots < 0)
    return fail(ATTNRES_ERR_ARG, "attention: bad sizes (batch %d, heads %d, kv_heads %d, q_len %lld, kv_slots %lld)",
                batch, heads, kv_heads, (long long)q_len, (long long)kv_slots);
  if (head_dim < 8 || head_dim > LM_ATTN_MAX_DIM || head_dim % 8 != 0)
    return fail(ATTNRES_ERR_UNSUPPORTED, "attention: head_dim %d is not a multiple of 8 up to %d", head_dim,
                LM_ATTN_MAX_DIM);
  if (q_len > kMaxLen || kv_slots > kMaxLen)
    return fail(ATTNRES_ERR_UNSUPPORTED, "attention: sequences over 2^30 tokens");
  if (heads / kv_heads > kMaxGroup || q_len * (heads / kv_heads) > kMaxLen)
    return fail(ATTNRES_ERR_UNSUPPORTED, "attention: over 4096 query heads per key head, or over 2^30 rows of them");
  const int64_t rows = q_len * (heads / kv_heads), lines = rows > kv_slots ? rows : kv_slots;
  if ((lines + 31) / 32 * batch * kv_heads > kMaxLen)
    return fail(ATTNRES_ERR_UNSUPPORTED, "attention: too many rows for one call");
  return ATTNRES_OK;
}

int fill_attention(lm_attn_params* P, int batch, int heads, int kv_heads, int64_t q_len, int64_t kv_slots,
                   int head_dim, int causal, float scale, const void* kv_lens, const void* q_start, int index_dtype,
                   int64_t q_start_value) {
  if (causal != 0 && causal != 1) return fail(ATTNRES_ERR_ARG, "attention: causal is 0 or 1");
  // masked scores are -inf before they are scaled, and the largest score has to be the largest scaled one
  if (!(scale > 0.f) || !std::isfinite(scale * 1.44269504088896340736f))
    return fail(ATTNRES_ERR_ARG, "attention: scale is not positive and finite");
  if (!valid_index(index_dtype)) return fail(ATTNRES_ERR_ARG, "attention: bad index_dtype %d", index_dtype);
  const int is = index_dtype == ATTNRES_INDEX_I64 ? 8 : 4;
  if (!aligned(kv_lens, is) || !aligned(q_start, is))
    return fail(ATTNRES_ERR_ALIGN, "attention: kv_lens and q_start must be aligned to their type");
  P->batch = batch;
  P->heads = heads;
  P->kv_heads = kv_heads;
  P->q_len = (int32_t)q_len;
  P->kv_len = (int32_t)kv_slots;
  P->dim = head_dim;
  P->causal = causal;
  P->scale = scale;
  P->scale_log2 = scale * 1.44269504088896340736f;
  P->kv_lens = kv_lens;
  P->q_start = q_start;
  P->lens64 = P->start64 = index_dtype == ATTNRES_INDEX_I64;
  P->start_from_end = q_start == nullptr && q_start_value == ATTNRES_START_FROM_END;
  P->q_start_const = P->start_from_end ? 0 : q_start_value;
  return ATTNRES_OK;
}

// Offsets within a tile (up to 128 rows) are 32 bits wide.
int check_span(const char* what, const lm_strides& s, int es) {
  if (s.b < 0 || s.h < 0 || s.t < 0) return fail(ATTNRES_ERR_ARG, "%s: a stride is negative", what);
  if (s.t * es >= kMaxTokenStride)
    return fail(ATTNRES_ERR_UNSUPPORTED, "%s: tokens are 32 MiB apart or more", what);
  return ATTNRES_OK;
}

// How the `lines` rows (or keys) of each key head are dealt out, 32 to a wave.
struct AttnPlan {
  int log = 0;     // 2^log waves share their rows
  int splits = 1;  // parts of the key axis (forward)
};

// Waves share rows (and split the key tiles) where there are too few of them
// for two or more on every SIMD: fwd and dq at the proxy training shape (1024
// waves) take 38 + 46 us with two sharing against 54 + 65 us with none, at the
// 8B one (8192) sharing costs 10-20%; dk and dv at the 8B shape (2048 waves)
// 608 us with two sharing, 725 with none and 761 with four, as workgroups of
// fewer keys balance the causal rows better.  Where even four sharing leave
// CUs without work, the forward splits the key axis over workgroups too.
AttnPlan attention_plan(int base, int64_t heads, int64_t lines, int64_t kv_slots, int cus) {
  AttnPlan p;
  const int64_t waves = heads * ((lines + 31) / 32), full = (int64_t)cus * (base == kAttnDkv ? 16 : 8);
  p.log = waves >= full ? 0 : waves * 2 >= full ? 1 : 2;
  if (base == kAttnFwd && p.log == 2) {
    // Tiles of 128 keys.  A part of one is short of work but not of time where
    // few rows join: one token over 1024, 2048 or 4096 keys (8/4 heads) takes
    // 7.0 + 3.8 us (kernel + join) against 10.7 + 3.8 with four tiles at least a
    // part, 512 keys 7.1 + 3.9 against 10.2 whole.  With many rows the join
    // costs more than the split gains: 4 x 512 causal tokens (4/2 heads) 10.7 us
    // whole against 12.9 + 22.2 in parts of two tiles, 2 x 613 in fp32 (6 heads
    // of 80) 30.0 against 35.4 + 20.6.  Past 4096 keys both ask for the same.
    const int64_t least = heads * lines <= (int64_t)cus * 4 ? 1 : 4;
    const int64_t most = (kv_slots + 127) / 128 / least, want = (int64_t)cus * kSplitPerCu / (waves > 0 ? waves : 1);
    const int64_t n = want < most ? want : most;
    p.splits = n < 2 ? 1 : n < LM_ATTN_MAX_SPLITS ? (int)n : LM_ATTN_MAX_SPLITS;
  }
  return p;
}

int launch_attention(int base, const char* kind, lm_attn_params& P, int dtype, int64_t lines, void* stream) {
  int cus = 0;
  int rc = attnres_internal_num_cus(&cus);
  if (rc != ATTNRES_OK) return rc;
  const int64_t heads = (int64_t)P.batch * P.kv_heads;
  const AttnPlan plan = attention_plan(base, heads, lines, P.kv_len, cus);
  const int per = 32 * LM_ATTN_WAVES >> plan.log;
  P.splits = plan.splits;
  P.n_tiles = (int32_t)((lines + per - 1) / per * plan.splits);
  P.cus_per_xcd = cus / 8 > 0 ? cus / 8 : 1;
  const int64_t items = P.n_tiles * heads;
  if (items > INT32_MAX - 8) return fail(ATTNRES_ERR_UNSUPPORTED, "attention: too many rows for one call");
  const bool f32 = dtype == ATTNRES_DTYPE_F32;
  const int blocks = (P.dim - 1) / 32;
  char name[64];
  snprintf(name, sizeof(name), "attnres_attention_%s_%s_d%d_s%d", kind, f32 ? "f32" : "bf16", 32 * (blocks + 1),
           1 << plan.log);
  return launch(base + (f32 ? 12 : 0) + 3 * blocks + plan.log, f32 ? kAttnF32Part : kAttnBf16Part, name,
                (unsigned)((items + 7) / 8 * 8), 1, 64 * LM_ATTN_WAVES, 0, P, stream);
}

// Bytes of the forward's partial rows, and where their maxima and sums begin.
int forward_workspace(int batch, int heads, int kv_heads, int64_t q_len, int64_t kv_slots, int head_dim, int64_t* ml,
                      int64_t* bytes) {
  int cus = 0;
  int rc = attnres_internal_num_cus(&cus);
  if (rc != ATTNRES_OK) return rc;
  const int splits =
      attention_plan(kAttnFwd, (int64_t)batch * kv_heads, q_len * (heads / kv_heads), kv_slots, cus).splits;
  const int64_t parts = splits > 1 ? (int64_t)batch * heads * q_len * splits : 0;
  *ml = parts * head_dim * 4;
  *bytes = *ml + parts * 8;
  return ATTNRES_OK;
}

// ------------------------------------------------------------------ rope --

constexpr int kRopeMaxDim = 256;
constexpr int kRopeThreads = 256;
constexpr int kRopeBwdPerCu = 4;    // workgroups of the backward
constexpr int kRopeMaxChunks = 64;  // head rows of its grid, for queries and for keys

int rope_lanes(int half, int v) {
  int n = (half + v - 1) / v, g = 1;
  while (g < n && g < 64) g <<= 1;
  return g;
}

// Checks and fills what forward and backward share; *vec: whether the 16-byte kernels apply.
int fill_rope(lm_rope_params* P, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
              int batch, int q_heads, int k_heads, int64_t tokens, int head_dim, int dtype, const void* q_weight,
              const void* k_weight, const void* cos, int64_t cos_ld, const void* sin, int64_t sin_ld,
              int64_t table_rows, int table_dtype, const void* positions, int index_dtype, int64_t pos_batch_stride,
              int64_t pos_token_stride, float eps, bool* vec) {
  if (!valid_dtype(dtype)) return fail(ATTNRES_ERR_ARG, "qk_norm_rope: bad dtype %d", dtype);
  if (table_dtype != dtype && table_dtype != ATTNRES_DTYPE_F32)
    return fail(ATTNRES_ERR_ARG, "qk_norm_rope: the tables' dtype must be the rows' or fp32");
  if (batch < 0 || q_heads < 0 || k_heads < 0 || tokens < 0) return fail(ATTNRES_ERR_ARG, "qk_norm_rope: bad sizes");
  if (tokens > kMaxLen || tokens * batch > kMaxLen || q_heads > (1 << 14) || k_heads > (1 << 14))
    return fail(ATTNRES_ERR_UNSUPPORTED, "qk_norm_rope: over 2^30 tokens, or over 2^14 heads");
  if (head_dim < 2 || head_dim > kRopeMaxDim || head_dim % 2 != 0)
    return fail(ATTNRES_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %d is not even and at most %d", head_dim, kRopeMaxDim);
  if (!std::isfinite(eps) || eps < 0) return fail(ATTNRES_ERR_ARG, "qk_norm_rope: bad eps");
  if (!valid_index(index_dtype)) return fail(ATTNRES_ERR_ARG, "qk_norm_rope: bad index_dtype %d", index_dtype);
  if (batch == 0 || tokens == 0 || q_heads + k_heads == 0) return ATTNRES_OK;
  const int es = esize(dtype), te = esize(table_dtype);
  if (cos == nullptr || sin == nullptr || table_rows < 0 || (table_rows > 1 && (cos_ld < head_dim || sin_ld < head_dim)))
    return fail(ATTNRES_ERR_ARG, "qk_norm_rope: bad tables");
  if (positions != nullptr && !aligned(positions, index_dtype == ATTNRES_INDEX_I64 ? 8 : 4))
    return fail(ATTNRES_ERR_ALIGN, "qk_norm_rope: positions must be aligned to their type");
  if (!aligned(cos, te) || !aligned(sin, te))
    return fail(ATTNRES_ERR_ALIGN, "qk_norm_rope: tables must be aligned to their type");
  const int v = 16 / es;
  bool ok = (head_dim / 2) % v == 0;
  const void* xs[2] = {q, k};
  const void* ws[2] = {q_weight, k_weight};
  const int64_t* sts[2] = {q_strides, k_strides};
  const int hs[2] = {q_heads, k_heads};
  const char* names[2] = {"qk_norm_rope: q", "qk_norm_rope: k"};
  for (int i = 0; i < 2; ++i) {
    P->heads[i] = hs[i];
    if (hs[i] == 0) continue;
    int rc = take_strides(names[i], xs[i], sts[i], batch, hs[i], tokens, es, es, &P->sx[i]);
    if (rc != ATTNRES_OK) return rc;
    if (ws[i] == nullptr) return fail(ATTNRES_ERR_ARG, "%s weight is NULL", names[i]);
    if (!aligned(ws[i], es)) return fail(ATTNRES_ERR_ALIGN, "%s weight must be aligned to its type", names[i]);
    P->x[i] = xs[i];
    P->w[i] = ws[i];
    ok = ok && aligned(xs[i], 16) && aligned(ws[i], 16) && P->sx[i].b % v == 0 && P->sx[i].h % v == 0 &&
         P->sx[i].t % v == 0;
  }
  ok = ok && (table_dtype == ATTNRES_DTYPE_F32 && dtype != ATTNRES_DTYPE_F32
                  ? true
                  : aligned(cos, 16) && aligned(sin, 16) && (table_rows <= 1 || (cos_ld % v == 0 && sin_ld % v == 0)));
  P->cos = cos;
  P->sin = sin;
  P->cos_ld = table_rows > 1 ? cos_ld : 0;
  P->sin_ld = table_rows > 1 ? sin_ld : 0;
  P->table_rows = table_rows;
  P->table_f32 = table_dtype == ATTNRES_DTYPE_F32 && dtype != ATTNRES_DTYPE_F32;
  P->positions = positions;
  P->pos64 = index_dtype == ATTNRES_INDEX_I64;
  P->pos_b = pos_batch_stride;
  P->pos_t = pos_token_stride;
  P->batch = batch;
  P->tokens = tokens;
  P->dim = head_dim;
  P->eps = eps;
  P->inv_dim = 1.0f / (float)head_dim;
  *vec = ok;
  return ATTNRES_OK;
}

int rope_extra(const char* what, const void* p, const int64_t* st, const lm_rope_params& P, int i, int es,
               lm_strides* out, bool* vec) {
  if (P.heads[i] == 0) return ATTNRES_OK;
  int rc = take_strides(what, p, st, P.batch, P.heads[i], P.tokens, es, es, out);
  if (rc != ATTNRES_OK) return rc;
  const int v = 16 / es;
  *vec = *vec && aligned(p, 16) && out->b % v == 0 && out->h % v == 0 && out->t % v == 0;
  return ATTNRES_OK;
}

const char* rope_kind(bool f32, bool vec) { return f32 ? (vec ? "f32_v4" : "f32_v1") : (vec ? "bf16_v8" : "bf16_v1"); }

// ------------------------------------------------------------- embedding --

struct EmbedPlan {
  int range, ranges, seg;
  int64_t stretches;
  int64_t at_rows, at_start, at_token, at_row, at_part, bytes;
};

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

EmbedPlan embed_plan(int64_t n, int64_t rows, int hidden) {
  EmbedPlan p;
  int64_t range = (rows + 255) / 256;  // a workgroup per CU
  if (range < 32) range = 32;
  if (range > LM_EMBED_MAX_RANGE) range = LM_EMBED_MAX_RANGE;
  p.range = (int)range;
  p.ranges = (int)((rows + range - 1) / range);
  int64_t seg = 8;
  while (seg < LM_EMBED_MAX_SEG && seg * 256 < n) seg <<= 1;
  p.seg = (int)seg;
  p.stretches = (n + seg - 1) / seg;
  p.at_rows = 256;
  p.at_start = p.at_rows + round256(rows * 4);
  p.at_token = p.at_start + round256(rows * 4);
  p.at_row = p.at_token + round256(n * 4);
  p.at_part = p.at_row + round256(n * 4);
  p.bytes = p.at_part + p.stretches * 2 * hidden * 4;
  return p;
}

int check_embedding_sizes(int64_t num_ids, int64_t rows, int hidden) {
  if (num_ids < 0 || rows < 0 || hidden < 1) return fail(ATTNRES_ERR_ARG, "embedding: bad sizes");
  if (num_ids > INT32_MAX - 64 || rows > INT32_MAX - LM_EMBED_MAX_RANGE || hidden > (1 << 23))
    return fail(ATTNRES_ERR_UNSUPPORTED, "embedding: more than 2^31 ids or rows, or a row over 2^23");
  return ATTNRES_OK;
}

int check_embedding(const void* ids, int index_dtype, int64_t num_ids, int64_t rows, int hidden, int dtype,
                    float scale) {
  if (!valid_dtype(dtype)) return fail(ATTNRES_ERR_ARG, "embedding: bad dtype %d", dtype);
  if (!valid_index(index_dtype)) return fail(ATTNRES_ERR_ARG, "embedding: bad index_dtype %d", index_dtype);
  int rc = check_embedding_sizes(num_ids, rows, hidden);
  if (rc != ATTNRES_OK) return rc;
  if (!std::isfinite(scale)) return fail(ATTNRES_ERR_ARG, "embedding: scale is not finite");
  if (num_ids > 0 && ids == nullptr) return fail(ATTNRES_ERR_ARG, "embedding: ids is NULL");
  if (!aligned(ids, index_dtype == ATTNRES_INDEX_I64 ? 8 : 4))
    return fail(ATTNRES_ERR_ALIGN, "embedding: ids must be aligned to their type");
  return ATTNRES_OK;
}

const char* embed_kind(bool f32, bool vec) { return rope_kind(f32, vec); }

}  // namespace

extern "C" {

int attnres_attention_workspace_size(int batch, int heads, int kv_heads, int64_t q_len, int64_t kv_slots, int head_dim,
                                     int dtype, int backward, int64_t* bytes) {
  if (bytes == nullptr) return fail(ATTNRES_ERR_ARG, "attention: bytes is NULL");
  int rc = check_attention(batch, heads, kv_heads, q_len, kv_slots, head_dim, dtype);
  if (rc != ATTNRES_OK) return rc;
  if (backward != 0) {
    *bytes = (int64_t)batch * heads * q_len * 4;
    return ATTNRES_OK;
  }
  int64_t ml = 0;
  return forward_workspace(batch, heads, kv_heads, q_len, kv_slots, head_dim, &ml, bytes);
}

int attnres_attention_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                          const void* v, const int64_t* v_strides, int batch, int heads, int kv_heads, int64_t q_len,
                          int64_t kv_slots, int head_dim, int dtype, int causal, float scale, const void* kv_lens,
                          const void* q_start, int index_dtype, int64_t q_start_value, void* out,
                          const int64_t* out_strides, float* lse, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  int rc = check_attention(batch, heads, kv_heads, q_len, kv_slots, head_dim, dtype);
  if (rc != ATTNRES_OK) return rc;
  lm_attn_params P;
  std::memset(&P, 0, sizeof(P));
  rc = fill_attention(&P, batch, heads, kv_heads, q_len, kv_slots, head_dim, causal, scale, kv_lens, q_start,
                      index_dtype, q_start_value);
  if (rc != ATTNRES_OK) return rc;
  if (batch == 0 || q_len == 0) return ATTNRES_OK;
  const int es = esize(dtype);
  if ((rc = take_strides("attention: q", q, q_strides, batch, heads, q_len, es, 16, &P.sq)) != ATTNRES_OK) return rc;
  if ((rc = take_strides("attention: out", out, out_strides, batch, heads, q_len, es, 16, &P.so)) != ATTNRES_OK)
    return rc;
  if (kv_slots > 0) {
    if ((rc = take_strides("attention: k", k, k_strides, batch, kv_heads, kv_slots, es, 16, &P.sk)) != ATTNRES_OK ||
        (rc = take_strides("attention: v", v, v_strides, batch, kv_heads, kv_slots, es, 16, &P.sv)) != ATTNRES_OK)
      return rc;
  }
  const int group = heads / kv_heads;
  if ((rc = check_span("attention: k", P.sk, es)) != ATTNRES_OK ||
      (rc = check_span("attention: v", P.sv, es)) != ATTNRES_OK)
    return rc;
  int64_t ml = 0, need = 0;
  if ((rc = forward_workspace(batch, heads, kv_heads, q_len, kv_slots, head_dim, &ml, &need)) != ATTNRES_OK) return rc;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(ATTNRES_ERR_ARG, "attention: workspace of %lld bytes needed", (long long)need);
  if (need > 0 && !aligned(workspace, 16))
    return fail(ATTNRES_ERR_ALIGN, "attention: workspace must be 16-byte aligned");
  P.part = static_cast<float*>(workspace);
  P.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + ml);
  P.q = q;
  P.k = k;
  P.v = v;
  P.o = out;
  P.lse = lse;
  rc = launch_attention(kAttnFwd, "fwd", P, dtype, q_len * group, stream);
  if (rc != ATTNRES_OK || P.splits < 2) return rc;
  const bool f32 = dtype == ATTNRES_DTYPE_F32;
  return launch(kAttnJoin + (f32 ? 1 : 0), f32 ? kAttnF32Part : kAttnBf16Part,
                f32 ? "attnres_attention_join_f32" : "attnres_attention_join_bf16", (unsigned)((int64_t)batch * heads * q_len),
                1, 256, 0, P, stream);
}

int attnres_attention_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                          const void* v, const int64_t* v_strides, const void* out, const int64_t* out_strides,
                          const void* grad_out, const int64_t* grad_out_strides, const float* lse,
                          const float* grad_lse, int batch, int heads, int kv_heads, int64_t q_len, int64_t kv_slots,
                          int head_dim, int dtype, int causal, float scale, const void* kv_lens, const void* q_start,
                          int index_dtype, int64_t q_start_value, void* grad_q, const int64_t* grad_q_strides,
                          void* grad_k, const int64_t* grad_k_strides, void* grad_v, const int64_t* grad_v_strides,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_attention(batch, heads, kv_heads, q_len, kv_slots, head_dim, dtype);
  if (rc != ATTNRES_OK) return rc;
  lm_attn_params P;
  std::memset(&P, 0, sizeof(P));
  rc = fill_attention(&P, batch, heads, kv_heads, q_len, kv_slots, head_dim, causal, scale, kv_lens, q_start,
                      index_dtype, q_start_value);
  if (rc != ATTNRES_OK) return rc;
  if (batch == 0) return ATTNRES_OK;
  const int es = esize(dtype);
  if (q_len > 0) {
    if ((rc = take_strides("attention: q", q, q_strides, batch, heads, q_len, es, 16, &P.sq)) != ATTNRES_OK ||
        (rc = take_strides("attention: out", out, out_strides, batch, heads, q_len, es, 16, &P.sout)) != ATTNRES_OK ||
        (rc = take_strides("attention: grad_out", grad_out, grad_out_strides, batch, heads, q_len, es, 16, &P.sdo)) !=
            ATTNRES_OK ||
        (rc = take_strides("attention: grad_q", grad_q, grad_q_strides, batch, heads, q_len, es, 16, &P.sdq)) !=
            ATTNRES_OK)
      return rc;
    if (lse == nullptr) return fail(ATTNRES_ERR_ARG, "attention: lse is NULL");
    const int64_t need = (int64_t)batch * heads * q_len * 4;
    if (workspace == nullptr || workspace_bytes < need)
      return fail(ATTNRES_ERR_ARG, "attention: workspace of %lld bytes needed", (long long)need);
    if (!aligned(workspace, 16) || !aligned(lse, 4) || !aligned(grad_lse, 4))
      return fail(ATTNRES_ERR_ALIGN, "attention: workspace, lse or grad_lse not aligned");
  }
  if (kv_slots > 0) {
    if ((rc = take_strides("attention: k", k, k_strides, batch, kv_heads, kv_slots, es, 16, &P.sk)) != ATTNRES_OK ||
        (rc = take_strides("attention: v", v, v_strides, batch, kv_heads, kv_slots, es, 16, &P.sv)) != ATTNRES_OK ||
        (rc = take_strides("attention: grad_k", grad_k, grad_k_strides, batch, kv_heads, kv_slots, es, 16, &P.sdk)) !=
            ATTNRES_OK ||
        (rc = take_strides("attention: grad_v", grad_v, grad_v_strides, batch, kv_heads, kv_slots, es, 16, &P.sdv)) !=
            ATTNRES_OK)
      return rc;
  }
  const int group = heads / kv_heads;
  if ((rc = check_span("attention: k", P.sk, es)) != ATTNRES_OK ||
      (rc = check_span("attention: v", P.sv, es)) != ATTNRES_OK ||
      (rc = check_span("attention: q", P.sq, es)) != ATTNRES_OK ||
      (rc = check_span("attention: grad_out", P.sdo, es)) != ATTNRES_OK)
    return rc;
  P.q = q;
  P.k = k;
  P.v = v;
  P.out = out;
  P.grad_out = grad_out;
  P.lse = const_cast<float*>(lse);
  P.grad_lse = grad_lse;
  P.delta = static_cast<float*>(workspace);
  P.dq = grad_q;
  P.dk = grad_k;
  P.dv = grad_v;
  if (q_len > 0) {
    rc = launch_attention(kAttnDq, "dq", P, dtype, q_len * group, stream);
    if (rc != ATTNRES_OK) return rc;
  }
  if (kv_slots == 0) return ATTNRES_OK;
  return launch_attention(kAttnDkv, "dkv", P, dtype, kv_slots, stream);
}

int attnres_qk_norm_rope_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                             int batch, int q_heads, int k_heads, int64_t tokens, int head_dim, int dtype,
                             const void* q_weight, const void* k_weight, const void* cos, int64_t cos_ld,
                             const void* sin, int64_t sin_ld, int64_t table_rows, int table_dtype,
                             const void* positions, int index_dtype, int64_t pos_batch_stride,
                             int64_t pos_token_stride, float eps, void* q_out, const int64_t* q_out_strides,
                             void* k_out, const int64_t* k_out_strides, void* stream) {
  lm_rope_params P;
  std::memset(&P, 0, sizeof(P));
  bool vec = false;
  int rc = fill_rope(&P, q, q_strides, k, k_strides, batch, q_heads, k_heads, tokens, head_dim, dtype, q_weight,
                     k_weight, cos, cos_ld, sin, sin_ld, table_rows, table_dtype, positions, index_dtype,
                     pos_batch_stride, pos_token_stride, eps, &vec);
  if (rc != ATTNRES_OK || batch == 0 || tokens == 0 || q_heads + k_heads == 0) return rc;
  const int es = esize(dtype);
  if ((rc = rope_extra("qk_norm_rope: q_out", q_out, q_out_strides, P, 0, es, &P.sy[0], &vec)) != ATTNRES_OK ||
      (rc = rope_extra("qk_norm_rope: k_out", k_out, k_out_strides, P, 1, es, &P.sy[1], &vec)) != ATTNRES_OK)
    return rc;
  P.y[0] = q_out;
  P.y[1] = k_out;
  const bool f32 = dtype == ATTNRES_DTYPE_F32;
  P.lanes = rope_lanes(head_dim / 2, vec ? 16 / es : 1);
  int cus = 0;
  if ((rc = attnres_internal_num_cus(&cus)) != ATTNRES_OK) return rc;
  // Four heads of a token per lane group share its table rows and keep more
  // reads in flight; with too few rows to fill the card that way, one.
  const int64_t n = (int64_t)batch * tokens;
  const int rows4 = (q_heads + 3) / 4 + (k_heads + 3) / 4;
  const bool h4 = n * rows4 * P.lanes >= (int64_t)cus * 256;
  const int groups = kRopeThreads / P.lanes;
  const int64_t grid = (n + groups - 1) / groups;
  char name[64];
  snprintf(name, sizeof(name), "attnres_qk_norm_rope_%s_h%d", rope_kind(f32, vec), h4 ? 4 : 1);
  return launch(kRopeFwd + (f32 ? 4 : 0) + (vec ? 0 : 2) + (h4 ? 1 : 0), kLmPart, name, (unsigned)grid,
                (unsigned)(h4 ? rows4 : q_heads + k_heads), kRopeThreads, 0, P, stream);
}

int attnres_qk_norm_rope_workspace_size(int head_dim, int64_t* bytes) {
  if (bytes == nullptr || head_dim < 2 || head_dim > kRopeMaxDim || head_dim % 2 != 0)
    return fail(ATTNRES_ERR_ARG, "qk_norm_rope: bad head_dim or bytes");
  int cus = 0;
  int rc = attnres_internal_num_cus(&cus);
  if (rc != ATTNRES_OK) return rc;
  *bytes = ((int64_t)kRopeBwdPerCu * cus + 2 * kRopeMaxChunks) * head_dim * 4;
  return ATTNRES_OK;
}

int attnres_qk_norm_rope_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                             const void* grad_q_out, const int64_t* grad_q_out_strides, const void* grad_k_out,
                             const int64_t* grad_k_out_strides, int batch, int q_heads, int k_heads, int64_t tokens,
                             int head_dim, int dtype, const void* q_weight, const void* k_weight, const void* cos,
                             int64_t cos_ld, const void* sin, int64_t sin_ld, int64_t table_rows, int table_dtype,
                             const void* positions, int index_dtype, int64_t pos_batch_stride,
                             int64_t pos_token_stride, float eps, void* grad_q, const int64_t* grad_q_strides,
                             void* grad_k, const int64_t* grad_k_strides, void* grad_q_weight, void* grad_k_weight,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  lm_rope_params P;
  std::memset(&P, 0, sizeof(P));
  bool vec = false;
  int rc = fill_rope(&P, q, q_strides, k, k_strides, batch, q_heads, k_heads, tokens, head_dim, dtype, q_weight,
                     k_weight, cos, cos_ld, sin, sin_ld, table_rows, table_dtype, positions, index_dtype,
                     pos_batch_stride, pos_token_stride, eps, &vec);
  if (rc != ATTNRES_OK) return rc;
  const int es = esize(dtype);
  if (!aligned(grad_q_weight, es) || !aligned(grad_k_weight, es) || !aligned(workspace, 16))
    return fail(ATTNRES_ERR_ALIGN, "qk_norm_rope: weight gradients or workspace not aligned");
  const bool f32 = dtype == ATTNRES_DTYPE_F32;
  const bool rows = batch > 0 && tokens > 0 && q_heads + k_heads > 0;
  P.dim = head_dim;
  P.dw[0] = grad_q_weight;
  P.dw[1] = grad_k_weight;
  P.dw_part = static_cast<float*>(workspace);
  char name[64];
  if (rows) {
    if ((rc = rope_extra("qk_norm_rope: grad_q_out", grad_q_out, grad_q_out_strides, P, 0, es, &P.sg[0], &vec)) !=
            ATTNRES_OK ||
        (rc = rope_extra("qk_norm_rope: grad_k_out", grad_k_out, grad_k_out_strides, P, 1, es, &P.sg[1], &vec)) !=
            ATTNRES_OK ||
        (rc = rope_extra("qk_norm_rope: grad_q", grad_q, grad_q_strides, P, 0, es, &P.sy[0], &vec)) != ATTNRES_OK ||
        (rc = rope_extra("qk_norm_rope: grad_k", grad_k, grad_k_strides, P, 1, es, &P.sy[1], &vec)) != ATTNRES_OK)
      return rc;
    P.g[0] = grad_q_out;
    P.g[1] = grad_k_out;
    P.y[0] = grad_q;
    P.y[1] = grad_k;
    P.lanes = rope_lanes(head_dim / 2, vec ? 16 / es : 1);
    int cus = 0;
    if ((rc = attnres_internal_num_cus(&cus)) != ATTNRES_OK) return rc;
    const int groups = kRopeThreads / P.lanes;
    // rows of 4 heads (2 at a time), more where there would be too many rows
    int chunk = 4;
    while ((q_heads + chunk - 1) / chunk > kRopeMaxChunks || (k_heads + chunk - 1) / chunk > kRopeMaxChunks) chunk *= 2;
    P.chunk = chunk;
    P.q_chunks = (q_heads + chunk - 1) / chunk;
    P.chunks = P.q_chunks + (k_heads + chunk - 1) / chunk;
    int64_t parts = ((int64_t)batch * tokens + groups - 1) / groups, most = (int64_t)kRopeBwdPerCu * cus / P.chunks;
    if (parts > most) parts = most > 0 ? most : 1;
    P.parts = (int)parts;
    const int64_t need = parts * P.chunks * head_dim * 4;
    if (workspace == nullptr || workspace_bytes < need)
      return fail(ATTNRES_ERR_ARG, "qk_norm_rope: workspace of %lld bytes needed", (long long)need);
    snprintf(name, sizeof(name), "attnres_qk_norm_rope_bwd_%s", rope_kind(f32, vec));
    rc = launch(kRopeBwd + (f32 ? 2 : 0) + (vec ? 0 : 1), kLmPart, name, (unsigned)parts, (unsigned)P.chunks, kRopeThreads,
                (unsigned)(groups * head_dim * 4), P, stream);
    if (rc != ATTNRES_OK) return rc;
  }
  if (grad_q_weight == nullptr && grad_k_weight == nullptr) return ATTNRES_OK;
  snprintf(name, sizeof(name), "attnres_qk_norm_rope_dw_%s", f32 ? "f32" : "bf16");
  return launch(kRopeDw + (f32 ? 1 : 0), kLmPart, name, (unsigned)((head_dim + 31) / 32), 2, 1024, 0, P, stream);
}

int attnres_embedding_fwd(const void* ids, int index_dtype, int64_t num_ids, const void* weight, int64_t weight_ld,
                          int64_t rows, int hidden, int dtype, float scale, void* out, void* stream) {
  int rc = check_embedding(ids, index_dtype, num_ids, rows, hidden, dtype, scale);
  if (rc != ATTNRES_OK) return rc;
  if (rows > 1 && weight_ld < hidden) return fail(ATTNRES_ERR_ARG, "embedding: weight_ld < hidden");
  if (num_ids == 0) return ATTNRES_OK;
  if (out == nullptr || (rows > 0 && weight == nullptr)) return fail(ATTNRES_ERR_ARG, "embedding: weight or out is NULL");
  const int es = esize(dtype), v = 16 / es;
  if (!aligned(weight, es) || !aligned(out, es))
    return fail(ATTNRES_ERR_ALIGN, "embedding: weight and out must be aligned to their type");
  const bool f32 = dtype == ATTNRES_DTYPE_F32;
  const bool vec = hidden % v == 0 && aligned(weight, 16) && aligned(out, 16) && (rows <= 1 || weight_ld % v == 0);
  lm_embed_params P;
  std::memset(&P, 0, sizeof(P));
  P.ids = ids;
  P.ids64 = index_dtype == ATTNRES_INDEX_I64;
  P.n = num_ids;
  P.w = weight;
  P.w_ld = weight_ld;
  P.rows = rows;
  P.dim = hidden;
  P.scale = scale;
  P.out = out;
  const int chunks = vec ? hidden / v : hidden;
  int tpr = 1;
  while (tpr < chunks && tpr < 256) tpr <<= 1;
  P.threads_per_row = tpr;
  const int64_t grid = (num_ids + 256 / tpr - 1) / (256 / tpr);
  char name[64];
  snprintf(name, sizeof(name), "attnres_embedding_fwd_%s", embed_kind(f32, vec));
  return launch(kEmbedFwd + (f32 ? 2 : 0) + (vec ? 0 : 1), kLmPart, name, (unsigned)grid, 1, 256, 0, P, stream);
}

int attnres_embedding_workspace_size(int64_t num_ids, int64_t rows, int hidden, int64_t* bytes) {
  if (bytes == nullptr) return fail(ATTNRES_ERR_ARG, "embedding: bytes is NULL");
  int rc = check_embedding_sizes(num_ids, rows, hidden);
  if (rc != ATTNRES_OK) return rc;
  *bytes = embed_plan(num_ids, rows, hidden).bytes;
  return ATTNRES_OK;
}

int attnres_embedding_bwd(const void* ids, int index_dtype, int64_t num_ids, const void* grad_out, int64_t grad_out_ld,
                          int64_t rows, int hidden, int dtype, float scale, int64_t padding_idx, void* grad_weight,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_embedding(ids, index_dtype, num_ids, rows, hidden, dtype, scale);
  if (rc != ATTNRES_OK) return rc;
  if (num_ids > 1 && grad_out_ld < hidden) return fail(ATTNRES_ERR_ARG, "embedding: grad_out_ld < hidden");
  if (padding_idx < -1) return fail(ATTNRES_ERR_ARG, "embedding: bad padding_idx");
  if (rows == 0) return ATTNRES_OK;
  if (grad_weight == nullptr || (num_ids > 0 && grad_out == nullptr))
    return fail(ATTNRES_ERR_ARG, "embedding: grad_out or grad_weight is NULL");
  const int es = esize(dtype), v = 16 / es;
  if (!aligned(grad_out, es) || !aligned(grad_weight, es))
    return fail(ATTNRES_ERR_ALIGN, "embedding: grad_out and grad_weight must be aligned to their type");
  const EmbedPlan plan = embed_plan(num_ids, rows, hidden);
  if (workspace == nullptr || workspace_bytes < plan.bytes)
    return fail(ATTNRES_ERR_ARG, "embedding: workspace of %lld bytes needed", (long long)plan.bytes);
  if (!aligned(workspace, 16)) return fail(ATTNRES_ERR_ALIGN, "embedding: workspace must be 16-byte aligned");
  const bool f32 = dtype == ATTNRES_DTYPE_F32;
  const bool vec =
      hidden % v == 0 && aligned(grad_out, 16) && aligned(grad_weight, 16) && (num_ids <= 1 || grad_out_ld % v == 0);
  char* ws = static_cast<char*>(workspace);
  lm_embed_params P;
  std::memset(&P, 0, sizeof(P));
  P.ids = ids;
  P.ids64 = index_dtype == ATTNRES_INDEX_I64;
  P.n = num_ids;
  P.g = grad_out;
  P.g_ld = grad_out_ld;
  P.rows = rows;
  P.dim = hidden;
  P.scale = scale;
  P.padding = padding_idx;
  P.dw = grad_weight;
  P.counts = reinterpret_cast<int32_t*>(ws);
  P.row_count = reinterpret_cast<int32_t*>(ws + plan.at_rows);
  P.row_start = reinterpret_cast<int32_t*>(ws + plan.at_start);
  P.sorted_token = reinterpret_cast<int32_t*>(ws + plan.at_token);
  P.sorted_row = reinterpret_cast<int32_t*>(ws + plan.at_row);
  P.part = reinterpret_cast<float*>(ws + plan.at_part);
  P.range = plan.range;
  P.seg = plan.seg;
  P.stretches = (int32_t)plan.stretches;
  rc = launch(kEmbedSort, kLmPart, "attnres_embedding_sort", (unsigned)plan.ranges, 1, 64 * LM_EMBED_WAVES, 0, P,
              stream);
  if (rc != ATTNRES_OK) return rc;
  const char* kind = embed_kind(f32, vec);
  const int idx = (f32 ? 2 : 0) + (vec ? 0 : 1);
  char name[64];
  const int chunks = vec ? hidden / v : hidden;
  const int block = chunks >= 512 ? 512 : (chunks + 63) / 64 * 64;
  const int64_t slices = (chunks + block - 1) / block;
  snprintf(name, sizeof(name), "attnres_embedding_sum_%s", kind);
  rc = launch(kEmbedSum + idx, kLmPart, name, (unsigned)(plan.stretches + (rows + LM_EMBED_ZERO - 1) / LM_EMBED_ZERO),
              (unsigned)slices, (unsigned)block, 0, P,
              stream);
  if (rc != ATTNRES_OK || plan.stretches < 2) return rc;
  snprintf(name, sizeof(name), "attnres_embedding_join_%s", f32 ? "f32" : "bf16");
  return launch(kEmbedJoin + (f32 ? 1 : 0), kLmPart, name, (unsigned)((plan.stretches - 1 + LM_EMBED_JOIN - 1) / LM_EMBED_JOIN),
                (unsigned)((hidden + 255) / 256), 64 * LM_EMBED_JOIN_WAVES, 0, P, stream);
}

}  // extern "C"
