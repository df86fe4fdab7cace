/*
 * Kernel-argument blocks of the language-model operators (lm_kernels.hip,
 * attention_kernels.hip), shared by the gfx950 code objects and the host
 * launcher (lm_capi.cpp), as attnres_params.h is for the routing kernels.
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

#endif /* KOTODAMA_AMD_LM_PARAMS_H */
