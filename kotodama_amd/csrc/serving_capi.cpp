// Host side of the serving operators of libattnres_hip.so (paged_attention_kernels.hip,
// serving_kernels.hip): argument checks, launch shapes and launches.  As in
// attnres_capi.cpp: no allocation, no synchronisation, every argument checked
// before any HIP call.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "attnres.h"
#include "attnres_internal.h"
#include "lm_host.h"
#include "lm_params.h"
#include "paged_schedule.h"

namespace {

// Code-object parts and kernel slots.
constexpr int kPagedBf16Part = 15, kPagedF32Part = 16, kServingPart = 17;
enum Slot {
  kPagedAttn = kServingSlots,   // + 8 * (fp32) + 4 * (many rows) + (head_dim - 1) / 32
  kPagedJoin = kPagedAttn + 16, // + (fp32)
  kPagedSlots = kPagedJoin + 2,
  kPagedRelease,
  kPagedWrite,
  kVerifyRows,
  kVerifyPieces,
  kVerifyPick,
  kEnd
};
static_assert(kEnd <= ATTNRES_INTERNAL_SLOTS, "kernel slots");

constexpr int64_t kMaxTokens = (int64_t)1 << 30;  // of one sequence, and new ones of a call
constexpr int kMaxPage = 1 << 16;                 // rows
constexpr int kMaxGroup = 4096;                   // query heads per key head
constexpr int kMaxSeqs = 1 << 20;
constexpr int kMaxVocab = 1 << 21;

int index_size(int code) { return code == ATTNRES_INDEX_I64 ? 8 : 4; }

int check_index(const char* what, const void* p, int code, bool need) {
  if (!valid_index(code)) return fail(ATTNRES_ERR_ARG, "%s: bad index dtype %d", what, code);
  if (need && p == nullptr) return fail(ATTNRES_ERR_ARG, "%s is NULL", what);
  if (!aligned(p, index_size(code))) return fail(ATTNRES_ERR_ALIGN, "%s must be aligned to its type", what);
  return ATTNRES_OK;
}

// log2 of a page size that the kernels take.
int page_shift(int page_size, int* shift) {
  int s = 0;
  while ((1 << s) < page_size && s < 30) ++s;
  if (page_size < LM_PAGED_MIN_PAGE || page_size > kMaxPage || (1 << s) != page_size)
    return fail(ATTNRES_ERR_UNSUPPORTED, "paged: page size %d is not a power of two from %d to %d", page_size,
                LM_PAGED_MIN_PAGE, kMaxPage);
  *shift = s;
  return ATTNRES_OK;
}

// A cache tensor (pages, kv_heads, page_size, head_dim).
int take_cache(const char* what, const void* p, const int64_t* st, int64_t pages, int kv_heads, int page_size, int es,
               lm_strides* out) {
  if (pages == 0) return ATTNRES_OK;
  if (p == nullptr || st == nullptr) return fail(ATTNRES_ERR_ARG, "%s or its strides are NULL", what);
  out->b = pages > 1 ? st[0] : 0;
  out->h = kv_heads > 1 ? st[1] : 0;
  out->t = st[2];
  const int64_t m = 16 / es;
  if (!aligned(p, 16) || out->b % m || out->h % m || out->t % m)
    return fail(ATTNRES_ERR_ALIGN, "%s: pointer and strides must be multiples of 16 bytes", what);
  if (out->b < 0 || out->h < 0 || out->t < 0) return fail(ATTNRES_ERR_ARG, "%s: a stride is negative", what);
  if (out->t > INT32_MAX / es / page_size || out->b > INT32_MAX / es)
    return fail(ATTNRES_ERR_UNSUPPORTED, "%s: a head's rows of a page span 2^31 bytes, or its pages lie so far apart",
                what);
  return ATTNRES_OK;
}

// No two rows of a cache lie on one another: strides that each lead past all that the smaller ones reach.
bool rows_apart(const lm_strides& st, int64_t pages, int kv_heads, int page_size, int head_dim) {
  struct Axis {
    int64_t stride, size;
  } a[3] = {{st.b, pages}, {st.h, kv_heads}, {st.t, page_size}};
  std::sort(a, a + 3, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
  __int128 reach = head_dim - 1;
  for (const Axis& x : a) {
    if (x.size <= 1) continue;
    if (x.stride <= reach) return false;
    reach += (__int128)x.stride * (x.size - 1);
  }
  return true;
}

// A (tokens, heads, head_dim) tensor's strides (token, head).
int take_rows(const char* what, const void* p, const int64_t* st, int64_t tokens, int heads, int es, int64_t* t,
              int64_t* h) {
  if (p == nullptr || st == nullptr) return fail(ATTNRES_ERR_ARG, "%s or its strides are NULL", what);
  *t = tokens > 1 ? st[0] : 0;
  *h = heads > 1 ? st[1] : 0;
  const int64_t m = 16 / es;
  if (!aligned(p, 16) || *t % m || *h % m)
    return fail(ATTNRES_ERR_ALIGN, "%s: pointer and strides must be multiples of 16 bytes", what);
  return ATTNRES_OK;
}

int check_rows(const char* op, int64_t tokens, int kv_heads, int head_dim, int dtype) {
  if (!valid_dtype(dtype)) return fail(ATTNRES_ERR_ARG, "%s: bad dtype %d", op, dtype);
  if (tokens < 0 || kv_heads < 1) return fail(ATTNRES_ERR_ARG, "%s: bad sizes", op);
  if (head_dim < 8 || head_dim > LM_ATTN_MAX_DIM || head_dim % 8 != 0)
    return fail(ATTNRES_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 8 up to %d", op, head_dim,
                LM_ATTN_MAX_DIM);
  if (tokens > kMaxTokens) return fail(ATTNRES_ERR_UNSUPPORTED, "%s: over 2^30 tokens", op);
  return ATTNRES_OK;
}

// ------------------------------------------------------------- attention --

int plan_attention(int64_t tokens, int seqs, int heads, int kv_heads, int head_dim, int dtype, int64_t capacity,
                   PagedPlan* p) {
  int cus = 0;
  const int rc = attnres_internal_num_cus(&cus);
  if (rc != ATTNRES_OK) return rc;
  if (!paged_plan(cus, tokens, seqs, heads, kv_heads, head_dim, dtype == ATTNRES_DTYPE_F32, capacity, p))
    return fail(ATTNRES_ERR_UNSUPPORTED, "paged_attention: too many keys for one call");
  return ATTNRES_OK;
}

int check_attention(int64_t tokens, int seqs, int heads, int kv_heads, int head_dim, int dtype, int table_width,
                    int page_size, int* shift) {
  int rc = check_rows("paged_attention", tokens, kv_heads, head_dim, dtype);
  if (rc != ATTNRES_OK) return rc;
  if (heads < 1 || heads % kv_heads != 0 || seqs < 0 || table_width < 0)
    return fail(ATTNRES_ERR_ARG, "paged_attention: bad sizes (seqs %d, heads %d, kv_heads %d, table_width %d)", seqs,
                heads, kv_heads, table_width);
  if ((rc = page_shift(page_size, shift)) != ATTNRES_OK) return rc;
  if (heads / kv_heads > kMaxGroup || tokens * (heads / kv_heads) > kMaxTokens || seqs > kMaxSeqs)
    return fail(ATTNRES_ERR_UNSUPPORTED,
                "paged_attention: over 4096 query heads per key head, 2^30 rows of them or 2^20 sequences");
  if ((int64_t)table_width * page_size > kMaxTokens)
    return fail(ATTNRES_ERR_UNSUPPORTED, "paged_attention: a row of the table is over 2^30 tokens");
  return ATTNRES_OK;
}

// ----------------------------------------------------------------- slots --

int fill_slots(const char* op, lm_slots_params* P, void* table, int64_t table_ld, int seqs, int table_width,
               const void* held, int held_dtype, const void* change, int change_dtype, const void* free_pages,
               int free_len, const void* free_count, int page_size, void* count_out) {
  if (seqs < 0 || table_width < 0 || free_len < 0) return fail(ATTNRES_ERR_ARG, "%s: bad sizes", op);
  if (seqs > kMaxSeqs) return fail(ATTNRES_ERR_UNSUPPORTED, "%s: over 2^20 sequences", op);
  int rc = page_shift(page_size, &P->shift);
  if (rc != ATTNRES_OK) return rc;
  if ((int64_t)table_width * page_size > kMaxTokens)
    return fail(ATTNRES_ERR_UNSUPPORTED, "%s: a row of the table is over 2^30 tokens", op);
  if ((rc = check_index(op, held, held_dtype, seqs > 0)) != ATTNRES_OK ||
      (rc = check_index(op, change, change_dtype, seqs > 0)) != ATTNRES_OK)
    return rc;
  if (free_count == nullptr || count_out == nullptr || (free_len > 0 && free_pages == nullptr) ||
      (seqs > 0 && table_width > 0 && table == nullptr))
    return fail(ATTNRES_ERR_ARG, "%s: the table, the free pages or their counts are NULL", op);
  if (seqs > 1 && table_ld < table_width) return fail(ATTNRES_ERR_ARG, "%s: table_ld < table_width", op);
  if (!aligned(table, 4) || !aligned(free_pages, 4) || !aligned(free_count, 4) || !aligned(count_out, 4))
    return fail(ATTNRES_ERR_ALIGN, "%s: the table, the free pages and their counts must be aligned to their type", op);
  P->table = static_cast<int32_t*>(table);
  P->table_ld = table_ld;
  P->free = static_cast<int32_t*>(const_cast<void*>(free_pages));
  P->count = static_cast<const int32_t*>(free_count);
  P->held = held;
  P->held64 = held_dtype == ATTNRES_INDEX_I64;
  P->change = change;
  P->change64 = change_dtype == ATTNRES_INDEX_I64;
  P->count_out = static_cast<int32_t*>(count_out);
  P->seqs = seqs;
  P->table_width = table_width;
  P->free_len = free_len;
  P->page_limit = ((int64_t)1 << 31) >> P->shift;
  return ATTNRES_OK;
}

// ---------------------------------------------------------------- verify --

struct VerifyPlan {
  int64_t parts, slices, at_pieces, at_chosen, at_top, at_at, bytes;
};

VerifyPlan verify_plan(int64_t rows, int64_t seqs, int vocab) {
  VerifyPlan p;
  p.parts = (vocab + LM_VERIFY_PART - 1) / LM_VERIFY_PART;
  p.slices = (vocab + LM_VERIFY_SLICE - 1) / LM_VERIFY_SLICE;
  const int64_t n = rows * p.parts;
  p.at_pieces = n * 8;
  p.at_chosen = p.at_pieces + seqs * p.slices * (LM_VERIFY_SLICE / LM_VERIFY_PIECE) * 16;
  p.at_top = p.at_chosen + seqs * (int64_t)sizeof(lm_verify_choice);
  p.at_at = p.at_top + n * 4;
  p.bytes = p.at_at + n * 4;
  return p;
}

// Workgroups for so many tokens or pages.  Every one scans all lengths, which costs nothing where they run
// side by side (66000 tokens of 512 sequences: 6.4 us with a token a thread, 8.3 with four).
unsigned slot_groups(int64_t items) {
  const int64_t n = (items + LM_SLOTS_THREADS - 1) / LM_SLOTS_THREADS;
  return (unsigned)(n < 1 ? 1 : n > 256 ? 256 : n);
}

}  // namespace

extern "C" {

int attnres_paged_slots(void* block_table, int64_t table_ld, int seqs, int table_width, const void* held,
                        int held_dtype, const void* new_tokens, int new_dtype, const void* free_pages, int free_len,
                        const void* free_count, int page_size, int64_t tokens, void* slots, void* positions,
                        void* q_starts, void* kv_lens, void* free_count_out, void* stream) {
  lm_slots_params P;
  std::memset(&P, 0, sizeof(P));
  int rc = fill_slots("paged_slots", &P, block_table, table_ld, seqs, table_width, held, held_dtype, new_tokens,
                      new_dtype, free_pages, free_len, free_count, page_size, free_count_out);
  if (rc != ATTNRES_OK) return rc;
  if (tokens < 0) return fail(ATTNRES_ERR_ARG, "paged_slots: bad tokens");
  if (tokens > kMaxTokens) return fail(ATTNRES_ERR_UNSUPPORTED, "paged_slots: over 2^30 tokens");
  if (q_starts == nullptr || (seqs > 0 && kv_lens == nullptr) ||
      (tokens > 0 && (slots == nullptr || positions == nullptr)))
    return fail(ATTNRES_ERR_ARG, "paged_slots: a result is NULL");
  if (!aligned(q_starts, 4) || !aligned(kv_lens, 4) || !aligned(slots, 4) || !aligned(positions, 4))
    return fail(ATTNRES_ERR_ALIGN, "paged_slots: a result is not aligned to its type");
  P.tokens = (int32_t)tokens;
  P.slots = static_cast<int32_t*>(slots);
  P.positions = static_cast<int32_t*>(positions);
  P.q_starts = static_cast<int32_t*>(q_starts);
  P.kv_lens = static_cast<int32_t*>(kv_lens);
  return launch(kPagedSlots, kServingPart, "attnres_paged_slots", slot_groups(tokens), 1, LM_SLOTS_THREADS, 0, P,
                stream);
}

int attnres_paged_release(const void* block_table, int64_t table_ld, int seqs, int table_width, const void* held,
                          int held_dtype, const void* kept, int kept_dtype, void* free_pages, int free_len,
                          const void* free_count, int page_size, void* free_count_out, void* stream) {
  lm_slots_params P;
  std::memset(&P, 0, sizeof(P));
  const int rc = fill_slots("paged_release", &P, const_cast<void*>(block_table), table_ld, seqs, table_width, held,
                            held_dtype, kept, kept_dtype, free_pages, free_len, free_count, page_size, free_count_out);
  if (rc != ATTNRES_OK) return rc;
  return launch(kPagedRelease, kServingPart, "attnres_paged_release", slot_groups((int64_t)seqs * table_width / 16), 1,
                LM_SLOTS_THREADS, 0, P, stream);
}

int attnres_paged_write(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                        int64_t tokens, int kv_heads, int head_dim, int dtype, void* k_cache,
                        const int64_t* k_cache_strides, void* v_cache, const int64_t* v_cache_strides, int64_t pages,
                        int page_size, const void* slots, int slots_dtype, void* stream) {
  int rc = check_rows("paged_write", tokens, kv_heads, head_dim, dtype);
  if (rc != ATTNRES_OK) return rc;
  if (pages < 0 || pages > INT32_MAX) return fail(ATTNRES_ERR_ARG, "paged_write: bad pages");
  if (kv_heads > (1 << 14)) return fail(ATTNRES_ERR_UNSUPPORTED, "paged_write: over 2^14 heads");
  lm_write_params P;
  std::memset(&P, 0, sizeof(P));
  if ((rc = page_shift(page_size, &P.shift)) != ATTNRES_OK ||
      (rc = check_index("paged_write: slots", slots, slots_dtype, tokens > 0)) != ATTNRES_OK)
    return rc;
  if (tokens == 0 || pages == 0) return ATTNRES_OK;
  const int es = esize(dtype);
  if ((rc = take_rows("paged_write: k", k, k_strides, tokens, kv_heads, es, &P.k_t, &P.k_h)) != ATTNRES_OK ||
      (rc = take_rows("paged_write: v", v, v_strides, tokens, kv_heads, es, &P.v_t, &P.v_h)) != ATTNRES_OK ||
      (rc = take_cache("paged_write: k_cache", k_cache, k_cache_strides, pages, kv_heads, page_size, es, &P.sk)) !=
          ATTNRES_OK ||
      (rc = take_cache("paged_write: v_cache", v_cache, v_cache_strides, pages, kv_heads, page_size, es, &P.sv)) !=
          ATTNRES_OK)
    return rc;
  for (const lm_strides* c : {&P.sk, &P.sv})
    if (!rows_apart(*c, pages, kv_heads, page_size, head_dim))
      return fail(ATTNRES_ERR_ARG, "paged_write: rows of the cache may lie on one another: a stride does not lead past "
                                   "what the smaller ones reach");
  for (int64_t* st : {&P.k_t, &P.k_h, &P.v_t, &P.v_h, &P.sk.b, &P.sk.h, &P.sk.t, &P.sv.b, &P.sv.h, &P.sv.t}) *st *= es;
  P.k = k;
  P.v = v;
  P.k_cache = k_cache;
  P.v_cache = v_cache;
  P.slots = slots;
  P.slots64 = slots_dtype == ATTNRES_INDEX_I64;
  P.limit = pages * page_size;
  P.tokens = (int32_t)tokens;
  P.chunks = head_dim * es / 16;
  P.per_token = kv_heads * P.chunks;
  const int64_t grid = (tokens * P.per_token + 255) / 256;
  if (grid > INT32_MAX) return fail(ATTNRES_ERR_UNSUPPORTED, "paged_write: too many rows for one call");
  return launch(kPagedWrite, kServingPart, "attnres_paged_write", (unsigned)grid, 1, 256, 0, P, stream);
}

int attnres_paged_attention_workspace_size(int64_t tokens, int seqs, int heads, int kv_heads, int head_dim, int dtype,
                                           int table_width, int page_size, int64_t* bytes) {
  if (bytes == nullptr) return fail(ATTNRES_ERR_ARG, "paged_attention: bytes is NULL");
  int shift = 0;
  int rc = check_attention(tokens, seqs, heads, kv_heads, head_dim, dtype, table_width, page_size, &shift);
  if (rc != ATTNRES_OK) return rc;
  PagedPlan plan;
  rc = plan_attention(tokens, seqs, heads, kv_heads, head_dim, dtype, (int64_t)table_width * page_size, &plan);
  *bytes = plan.bytes;
  return rc;
}

int attnres_paged_attention_fwd(const void* q, const int64_t* q_strides, const void* k_cache, const int64_t* k_strides,
                                const void* v_cache, const int64_t* v_strides, int64_t tokens, int seqs, int heads,
                                int kv_heads, int head_dim, int dtype, int64_t pages, int page_size,
                                const void* block_table, int64_t table_ld, int table_width, const void* kv_lens,
                                int lens_dtype, const void* q_starts, int starts_dtype, float scale, void* out,
                                const int64_t* out_strides, float* lse, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  lm_paged_params P;
  std::memset(&P, 0, sizeof(P));
  int rc = check_attention(tokens, seqs, heads, kv_heads, head_dim, dtype, table_width, page_size, &P.shift);
  if (rc != ATTNRES_OK) return rc;
  if (pages < 0 || pages > INT32_MAX) return fail(ATTNRES_ERR_ARG, "paged_attention: bad pages");
  if (!(scale > 0.f) || !std::isfinite(scale * 1.44269504088896340736f))
    return fail(ATTNRES_ERR_ARG, "paged_attention: scale is not positive and finite");
  if ((rc = check_index("paged_attention: kv_lens", kv_lens, lens_dtype, seqs > 0)) != ATTNRES_OK ||
      (rc = check_index("paged_attention: q_starts", q_starts, starts_dtype, false)) != ATTNRES_OK)
    return rc;
  if (q_starts == nullptr && tokens != seqs)
    return fail(ATTNRES_ERR_ARG, "paged_attention: without q_starts every sequence has one new token");
  if (seqs > 0 && table_width > 0 && block_table == nullptr)
    return fail(ATTNRES_ERR_ARG, "paged_attention: block_table is NULL");
  if (seqs > 1 && table_ld < table_width) return fail(ATTNRES_ERR_ARG, "paged_attention: table_ld < table_width");
  if (!aligned(block_table, 4) || !aligned(lse, 4))
    return fail(ATTNRES_ERR_ALIGN, "paged_attention: block_table or lse not aligned to its type");
  if (tokens == 0) return ATTNRES_OK;
  const int es = esize(dtype);
  if ((rc = take_rows("paged_attention: q", q, q_strides, tokens, heads, es, &P.q_t, &P.q_h)) != ATTNRES_OK ||
      (rc = take_rows("paged_attention: out", out, out_strides, tokens, heads, es, &P.o_t, &P.o_h)) != ATTNRES_OK ||
      (rc = take_cache("paged_attention: k_cache", k_cache, k_strides, pages, kv_heads, page_size, es, &P.sk)) !=
          ATTNRES_OK ||
      (rc = take_cache("paged_attention: v_cache", v_cache, v_strides, pages, kv_heads, page_size, es, &P.sv)) !=
          ATTNRES_OK)
    return rc;
  const int64_t capacity = pages == 0 ? 0 : (int64_t)table_width * page_size;
  PagedPlan plan;
  if ((rc = plan_attention(tokens, seqs, heads, kv_heads, head_dim, dtype, (int64_t)table_width * page_size, &plan)) !=
      ATTNRES_OK)
    return rc;
  if (plan.bytes > 0 && (workspace == nullptr || workspace_bytes < plan.bytes))
    return fail(ATTNRES_ERR_ARG, "paged_attention: workspace of %lld bytes needed", (long long)plan.bytes);
  if (plan.bytes > 0 && !aligned(workspace, 16))
    return fail(ATTNRES_ERR_ALIGN, "paged_attention: workspace must be 16-byte aligned");
  P.q = q;
  P.k = k_cache;
  P.v = v_cache;
  P.o = out;
  P.lse = lse;
  P.part = static_cast<float*>(workspace);
  P.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.at_ml);
  P.notes = reinterpret_cast<lm_paged_note*>(static_cast<char*>(workspace) + plan.at_notes);
  P.table = static_cast<const int32_t*>(block_table);
  P.table_ld = table_ld;
  P.kv_lens = kv_lens;
  P.lens64 = lens_dtype == ATTNRES_INDEX_I64;
  P.q_starts = q_starts;
  P.starts64 = starts_dtype == ATTNRES_INDEX_I64;
  P.tokens = (int32_t)tokens;
  P.seqs = seqs;
  P.heads = heads;
  P.kv_heads = kv_heads;
  P.pages = (int32_t)pages;
  P.capacity = (int32_t)capacity;
  P.dim = head_dim;
  P.group = heads / kv_heads;
  while ((1 << P.group_shift) < P.group) ++P.group_shift;
  P.group_mul =
      (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << P.group_shift) - (uint64_t)P.group)) / (uint64_t)P.group + 1);
  P.wide = plan.wide;
  P.turn = plan.turn;
  P.target = plan.target;
  P.slots = (int32_t)(plan.slots / kv_heads);
  P.part_rows = plan.part_rows;
  P.scale_log2 = scale * 1.44269504088896340736f;
  if (plan.grid > INT32_MAX) return fail(ATTNRES_ERR_UNSUPPORTED, "paged_attention: too many rows for one call");
  const bool f32 = dtype == ATTNRES_DTYPE_F32;
  const int blocks = (head_dim - 1) / 32, part = f32 ? kPagedF32Part : kPagedBf16Part;
  char name[64];
  snprintf(name, sizeof(name), "attnres_paged_%s_%s_d%d", plan.wide ? "tiles" : "stream", f32 ? "f32" : "bf16",
           32 * (blocks + 1));
  rc = launch(kPagedAttn + (f32 ? 8 : 0) + (plan.wide ? 4 : 0) + blocks, part, name, (unsigned)plan.grid, 1,
              LM_PAGED_THREADS, 0, P, stream);
  if (rc != ATTNRES_OK || !plan.split) return rc;
  // workgroups of a note, over its rows (11 sequences, one of 301 new tokens, fp32: 6.4 us with 16, 10.8 with 4)
  const int lines = plan.wide ? 8 : plan.part_rows < 16 ? plan.part_rows : 16;
  return launch(kPagedJoin + (f32 ? 1 : 0), part, f32 ? "attnres_paged_join_f32" : "attnres_paged_join_bf16",
                (unsigned)plan.notes, (unsigned)lines, LM_PAGED_THREADS, 0, P, stream);
}

int attnres_verify_drafts_workspace_size(int64_t rows, int seqs, int vocab, int64_t* bytes) {
  if (bytes == nullptr || rows < 0 || vocab < 1 || seqs < 0)
    return fail(ATTNRES_ERR_ARG, "verify_drafts: bad sizes or bytes");
  if (vocab > kMaxVocab || rows > (1 << 24) || seqs > kMaxSeqs)
    return fail(ATTNRES_ERR_UNSUPPORTED, "verify_drafts: a vocabulary over 2^21, over 2^24 rows or 2^20 sequences");
  *bytes = verify_plan(rows, seqs, vocab).bytes;
  return ATTNRES_OK;
}

int attnres_verify_drafts(const void* logits, int64_t logits_ld, int logits_dtype, const void* draft_probs,
                          int64_t draft_ld, int draft_dtype, int64_t rows, int vocab, const void* ids, int ids_dtype,
                          const void* q_starts, int starts_dtype, int seqs, const float* uniforms, float temperature,
                          void* tokens, void* counts, void* workspace, int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  int rc = attnres_verify_drafts_workspace_size(rows, seqs, vocab, &need);
  if (rc != ATTNRES_OK) return rc;
  if (!valid_dtype(logits_dtype) || (draft_probs != nullptr && !valid_dtype(draft_dtype)))
    return fail(ATTNRES_ERR_ARG, "verify_drafts: bad dtype");
  if (!(temperature >= 0) || !std::isfinite(temperature) || (temperature > 0 && temperature < 1e-6f))
    return fail(ATTNRES_ERR_ARG, "verify_drafts: temperature is not 0 or from 1e-6 up");
  if ((rc = check_index("verify_drafts: ids", ids, ids_dtype, rows > 0)) != ATTNRES_OK ||
      (rc = check_index("verify_drafts: q_starts", q_starts, starts_dtype, true)) != ATTNRES_OK)
    return rc;
  if ((rows > 0 && (logits == nullptr || uniforms == nullptr || tokens == nullptr)) || (seqs > 0 && counts == nullptr))
    return fail(ATTNRES_ERR_ARG, "verify_drafts: logits, uniforms or a result is NULL");
  if (rows > 1 && (logits_ld < vocab || (draft_probs != nullptr && draft_ld < vocab)))
    return fail(ATTNRES_ERR_ARG, "verify_drafts: rows overlap");
  if (!aligned(logits, esize(logits_dtype)) || (draft_probs != nullptr && !aligned(draft_probs, esize(draft_dtype))) ||
      !aligned(uniforms, 4) || !aligned(tokens, index_size(ids_dtype)) || !aligned(counts, 4))
    return fail(ATTNRES_ERR_ALIGN, "verify_drafts: a tensor is not aligned to its type");
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(ATTNRES_ERR_ARG, "verify_drafts: workspace of %lld bytes needed", (long long)need);
  if (!aligned(workspace, 16)) return fail(ATTNRES_ERR_ALIGN, "verify_drafts: workspace must be 16-byte aligned");
  if (rows == 0 && seqs == 0) return ATTNRES_OK;
  lm_verify_params P;
  std::memset(&P, 0, sizeof(P));
  P.logits = logits;
  P.logits_ld = rows > 1 ? logits_ld : 0;
  P.logits_f32 = logits_dtype == ATTNRES_DTYPE_F32;
  P.logits_vec = aligned(logits, 16) && P.logits_ld * esize(logits_dtype) % 16 == 0;
  P.draft = draft_probs;
  if (draft_probs != nullptr) {
    P.draft_ld = rows > 1 ? draft_ld : 0;
    P.draft_f32 = draft_dtype == ATTNRES_DTYPE_F32;
    P.draft_vec = aligned(draft_probs, 16) && P.draft_ld * esize(draft_dtype) % 16 == 0;
  }
  P.ids = ids;
  P.ids64 = ids_dtype == ATTNRES_INDEX_I64;
  P.q_starts = q_starts;
  P.starts64 = starts_dtype == ATTNRES_INDEX_I64;
  P.uniforms = uniforms;
  P.tokens = tokens;
  P.counts = static_cast<int32_t*>(counts);
  P.rows = (int32_t)rows;
  P.seqs = seqs;
  P.vocab = vocab;
  const VerifyPlan plan = verify_plan(rows, seqs, vocab);
  P.parts = (int32_t)plan.parts;
  P.slices = (int32_t)plan.slices;
  P.greedy = temperature == 0;
  P.scale_log2 = temperature == 0 ? 1.0 : 1.44269504088896340736 / (double)temperature;
  char* ws = static_cast<char*>(workspace);
  P.part_sum = reinterpret_cast<double*>(ws);
  P.piece_sum = reinterpret_cast<double*>(ws + plan.at_pieces);
  P.part_top = reinterpret_cast<float*>(ws + plan.at_top);
  P.part_at = reinterpret_cast<int32_t*>(ws + plan.at_at);
  P.chosen = reinterpret_cast<lm_verify_choice*>(ws + plan.at_chosen);
  if (rows * plan.parts > INT32_MAX - 4 || seqs * plan.slices > INT32_MAX)
    return fail(ATTNRES_ERR_UNSUPPORTED, "verify_drafts: too many rows for one call");
  if (rows > 0) {
    rc = launch(kVerifyRows, kServingPart, "attnres_verify_rows", (unsigned)((rows * plan.parts + 3) / 4), 1, 256, 0, P,
                stream);
    if (rc != ATTNRES_OK) return rc;
  }
  if (seqs == 0) return ATTNRES_OK;
  if (rows > 0 && !P.greedy) {
    rc = launch(kVerifyPieces, kServingPart, "attnres_verify_pieces", (unsigned)(seqs * plan.slices), 1, 256, 0, P,
                stream);
    if (rc != ATTNRES_OK) return rc;
  }
  return launch(kVerifyPick, kServingPart, "attnres_verify_pick", (unsigned)seqs, 1, P.greedy ? 256 : 64, 0, P, stream);
}

}  // extern "C"
