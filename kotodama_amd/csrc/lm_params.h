/*
 * Kernel-argument blocks of the language-model operators (lm_kernels.hip, attention_kernels.hip,
 * paged_attention_kernels.hip, serving_kernels.hip), shared by the gfx950 code objects and the
 * host launchers (lm_capi.cpp, serving_capi.cpp), as attnres_params.h is for the routing kernels.
 *
 * Plain C types only: included by g++ (host) and by hipcc (device) alike.
 */
#ifndef KOTODAMA_AMD_LM_PARAMS_H
#define KOTODAMA_AMD_LM_PARAMS_H

#include <stdint.h>

#define LM_ATTN_WAVES 4 /* waves per workgroup of the attention kernels; a wave owns 32 rows or 32 keys */
#define LM_ATTN_MAX_DIM 128
#define LM_ATTN_MAX_SPLITS 512 /* parts of the key axis */

/* Strides in elements; element (b, h, t, d) of X at X + b*sb + h*sh + t*st + d. */
typedef struct lm_strides {
  int64_t b, h, t;
} lm_strides;

/*
 * One attention call: heads query heads over kv_heads key heads (query head h
 * reads key head h / (heads / kv_heads)).  Query i of sequence b is at position
 * start_b + i, start_b = q_start[b], or q_start_const, or (start_from_end)
 * kv_len_b - q_len.  causal: it sees keys 0 .. position if 0 <= position <
 * kv_len_b, else none; otherwise keys 0 .. kv_len_b - 1.
 */
typedef struct lm_attn_params {
  const void* q;
  const void* k;
  const void* v;
  const void* out;       /* backward: the forward's output */
  const void* grad_out;  /* backward */
  void* o;               /* forward: output */
  void* dq;
  void* dk;
  void* dv;
  float* lse;            /* (batch, heads, q_len) natural log of the softmax sum; -inf for a row with no keys */
  float* delta;          /* (batch, heads, q_len): rowsum(grad_out * out) - grad_lse, written by the dq kernel */
  const float* grad_lse; /* (batch, heads, q_len) or NULL */
  float* part;           /* (rows, splits, dim): sums of a part of the keys, where splits > 1 */
  float* part_ml;        /* (rows, splits, 2): their maxima (times log2 e) and sums of weights */
  const void* kv_lens;   /* (batch,) int32 or int64, or NULL: kv_len */
  const void* q_start;   /* (batch,) int32 or int64, or NULL */
  lm_strides sq, sk, sv, so, sdo, sout, sdq, sdk, sdv;
  int64_t q_start_const;
  int32_t batch;
  int32_t heads;
  int32_t kv_heads;
  int32_t q_len;
  int32_t kv_len;
  int32_t dim;
  int32_t causal;
  int32_t start_from_end;
  int32_t lens64;        /* kv_lens holds 64-bit numbers */
  int32_t start64;       /* q_start does */
  int32_t n_tiles;       /* tiles along the axis that the grid splits */
  int32_t splits;        /* parts of the key axis, each a workgroup (forward, four waves a row) */
  int32_t cus_per_xcd;
  float scale;           /* of the scores */
  float scale_log2;      /* scale * log2(e) */
} lm_attn_params;

/*
 * Per-head RMSNorm with the position rotation; index 0: queries, 1: keys.
 * Token (b, t) is rotated by row positions[b * pos_b + t * pos_t] (or t) of the
 * tables; a row outside them gives NaN.
 */
typedef struct lm_rope_params {
  const void* x[2];
  const void* g[2];  /* backward: dL/dy */
  void* y[2];        /* outputs; backward: dL/dx */
  const void* w[2];
  void* dw[2];       /* weight gradients */
  float* dw_part;    /* (chunks, parts, dim) */
  const void* cos;   /* (table_rows, dim), rows cos_ld apart, x's type or (table_f32) fp32 */
  const void* sin;
  const void* positions;
  lm_strides sx[2], sg[2], sy[2];
  int64_t cos_ld, sin_ld;
  int64_t pos_b, pos_t;
  int64_t table_rows;
  int64_t tokens;    /* per sequence */
  int32_t batch;
  int32_t heads[2];
  int32_t dim;
  int32_t lanes;     /* lanes per head row (a power of two) */
  int32_t chunk;     /* backward: heads per workgroup row, */
  int32_t q_chunks;  /* rows of the queries, */
  int32_t chunks;    /* rows in all, */
  int32_t parts;     /* workgroups per row */
  int32_t table_f32;
  int32_t pos64;
  float eps;
  float inv_dim;
} lm_rope_params;

/* Embedding lookup and its gradient. */
#define LM_EMBED_WAVES 16       /* waves of the sort's workgroups */
#define LM_EMBED_BATCH 16       /* ids a lane requests at once there */
#define LM_EMBED_MAX_RANGE 768  /* table rows per workgroup of the sort: 48 KiB of counters */
#define LM_EMBED_MAX_SEG 64     /* sorted tokens per stretch: one per lane */
#define LM_EMBED_ZERO 32        /* table rows per zeroing workgroup */
#define LM_EMBED_JOIN 32        /* stretches per workgroup of the join */
#define LM_EMBED_JOIN_WAVES 8   /* waves of the join's workgroups */
typedef struct lm_embed_params {
  const void* ids;       /* (n,) int32 or int64 */
  const void* w;         /* (rows, dim), rows w_ld apart */
  const void* g;         /* (n, dim) dL/dout, rows g_ld apart */
  void* out;             /* (n, dim) */
  void* dw;              /* (rows, dim) */
  int32_t* counts;       /* [0]: tokens that count */
  int32_t* row_count;    /* (rows,) tokens of each row */
  int32_t* row_start;    /* (rows,) and the place of its first among the sorted */
  int32_t* sorted_token; /* (n,) tokens by row, in order */
  int32_t* sorted_row;   /* (n,) their rows */
  float* part;           /* (stretches, 2, dim) */
  int64_t n;
  int64_t rows;
  int64_t w_ld;
  int64_t g_ld;
  int64_t padding;       /* this id has no gradient; -1: none */
  int32_t dim;
  int32_t ids64;
  int32_t range;         /* table rows per workgroup of the sort */
  int32_t seg;           /* sorted tokens per stretch */
  int32_t stretches;
  int32_t threads_per_row;
  float scale;
} lm_embed_params;

/*
 * Attention of packed new tokens over a paged cache.  Sequence s has the tokens
 * q_starts[s] .. q_starts[s + 1] - 1 (s, where q_starts is NULL), the last at position
 * kv_lens[s] - 1; key j is row j % page_size of page table[s][j / page_size].
 */
#define LM_PAGED_THREADS (64 * LM_ATTN_WAVES)
#define LM_PAGED_MIN_PAGE 16 /* rows of a wave's load lie in one page */
/* A tile of rows whose keys several workgroups shared: their sums lie in the slots first, next, next + step ... */
typedef struct lm_paged_note {
  int32_t token;         /* its sequence's first */
  int32_t row0;          /* its first row */
  int32_t rows;          /* of the sequence */
  int32_t head;          /* key head */
  int32_t parts;         /* under two: nothing to join */
  int32_t first, next, step;
} lm_paged_note;
typedef struct lm_paged_params {
  const void* q;         /* (tokens, heads, dim) */
  const void* k;         /* (pages, kv_heads, page_size, dim) */
  const void* v;
  void* o;               /* (tokens, heads, dim) */
  float* lse;            /* (tokens, heads) or NULL */
  float* part;           /* (slots, kv_heads, part_rows, dim): sums of a part of the keys */
  float* part_ml;        /* (slots, kv_heads, part_rows, 2): their maxima (times log2 e) and sums of weights */
  lm_paged_note* notes;  /* few rows: (target, kv_heads); many: (slots, kv_heads) */
  const int32_t* table;  /* (seqs, table_width), rows table_ld apart */
  const void* kv_lens;   /* (seqs,) */
  const void* q_starts;  /* (seqs + 1,) or NULL */
  lm_strides sk, sv;     /* page, head, token */
  int64_t q_t, q_h, o_t, o_h;
  int64_t table_ld;
  int32_t tokens;
  int32_t seqs;
  int32_t heads;
  int32_t kv_heads;
  int32_t pages;
  int32_t capacity;      /* keys of a table row: table_width * page_size */
  int32_t shift;         /* log2 of page_size */
  int32_t dim;
  int32_t group;         /* heads / kv_heads; a number under 2^31 over it: (umulhi(n, mul) + n) >> shift */
  uint32_t group_mul;
  int32_t group_shift;
  int32_t wide;          /* many rows: sequences of over 32 in tiles of 128 */
  int32_t turn;          /* many rows: a head's parts from this one on go the shortest first; 0: none */
  int32_t target;        /* workgroups (few rows: of a key head) to deal the key blocks out to */
  int32_t slots;         /* parts of tiles that the workspace holds */
  int32_t part_rows;     /* rows of one */
  int32_t lens64;
  int32_t starts64;
  float scale_log2;
} lm_paged_params;

/*
 * Block tables, slot maps and the free list of a paged cache.  A sequence that holds n tokens
 * has ceil(n / page_size) pages in its row of the table; free[0 .. count - 1] are the pages that
 * none has, taken from the end.
 */
#define LM_SLOTS_THREADS 1024
typedef struct lm_slots_params {
  int32_t* table;        /* (seqs, table_width), rows table_ld apart */
  int32_t* free;         /* (free_len,); slots: read, release: written behind count */
  const int32_t* count;  /* [0] */
  const void* held;      /* (seqs,) tokens held before */
  const void* change;    /* (seqs,) slots: new tokens, release: tokens kept */
  int32_t* slots;        /* (tokens,) page * page_size + row, or -1 */
  int32_t* positions;    /* (tokens,) */
  int32_t* q_starts;     /* (seqs + 1,) */
  int32_t* kv_lens;      /* (seqs,) tokens held after; 0: refused */
  int32_t* count_out;    /* [0] */
  int64_t table_ld;
  int64_t page_limit;    /* 2^31 / page_size: pages whose slots 32 bits count */
  int32_t tokens;
  int32_t seqs;
  int32_t table_width;
  int32_t free_len;
  int32_t shift;         /* log2 of page_size */
  int32_t held64;
  int32_t change64;
} lm_slots_params;

/* Rows of new keys and values into their slots of the cache. */
typedef struct lm_write_params {
  const void* k;         /* (tokens, kv_heads, dim) */
  const void* v;
  void* k_cache;         /* (pages, kv_heads, page_size, dim) */
  void* v_cache;
  const void* slots;     /* (tokens,) */
  lm_strides sk, sv;     /* bytes: page, head, token */
  int64_t k_t, k_h, v_t, v_h; /* bytes */
  int64_t limit;         /* pages * page_size */
  int32_t tokens;
  int32_t chunks;        /* 16-byte pieces of a head's row */
  int32_t per_token;     /* kv_heads * chunks */
  int32_t shift;
  int32_t slots64;
} lm_write_params;

/*
 * Drafted tokens against the target's logits.  Sequence s has the rows q_starts[s] ..
 * q_starts[s + 1] - 1; row r's draft is ids[r + 1].
 */
#define LM_VERIFY_PART 2048  /* logits of a wave of the first launch, */
#define LM_VERIFY_SLICE 4096 /* of a workgroup of the second, */
#define LM_VERIFY_PIECE 512  /* and of a wave's step there */
/* What a sequence's token is taken from: the row behind the drafts that stay, its largest logit and its sum. */
typedef struct lm_verify_choice {
  double sum;
  float top;
  int32_t accepted;
} lm_verify_choice;
typedef struct lm_verify_params {
  const void* logits;       /* (rows, vocab), rows logits_ld apart */
  const void* draft;        /* (rows, vocab) probabilities or NULL */
  const void* ids;          /* (rows,) */
  const void* q_starts;     /* (seqs + 1,) */
  const float* uniforms;    /* (rows, 2) */
  void* tokens;             /* (rows,) as ids */
  int32_t* counts;          /* (seqs,) */
  double* part_sum;         /* (rows, parts) sums of exp((x - top) / temperature) */
  float* part_top;          /* (rows, parts) */
  int32_t* part_at;         /* (rows, parts) where it is first, greedily */
  double* piece_sum;        /* (seqs, slices, pieces, 2): of the weights, and of the exponentials */
  lm_verify_choice* chosen; /* (seqs,) */
  int64_t logits_ld, draft_ld;
  int32_t rows;
  int32_t seqs;
  int32_t vocab;
  int32_t parts;            /* of a row, a wave each */
  int32_t slices;           /* of a row, a workgroup each */
  int32_t logits_f32, draft_f32;
  int32_t logits_vec, draft_vec; /* rows load in 16-byte pieces */
  int32_t ids64;
  int32_t starts64;
  int32_t greedy;
  double scale_log2;        /* log2(e) / temperature */
} lm_verify_params;

#endif /* KOTODAMA_AMD_LM_PARAMS_H */
