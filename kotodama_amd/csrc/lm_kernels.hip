// Memory-bound language-model operators for gfx950: per-head RMSNorm with the
// position rotation of queries and keys, and the embedding lookup with its
// gradient by sorted tokens.  Sums and statistics are fp32; results are
// rounded once.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lm_params.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr float kNan = __builtin_nanf("");

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  bf16x2 r = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, r);
}

// V consecutive elements of type T (V = 1, or a 16-byte chunk) as fp32.
struct Bf16 {
  typedef uint16_t raw;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(uint16_t r) { return __builtin_bit_cast(float, (uint32_t)r << 16); }
  static __device__ __forceinline__ void chunk(const u32x4& w, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i];
      v[2 * i] = __builtin_bit_cast(float, u << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, u & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 unchunk(const float* v) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    return w;
  }
  static __device__ __forceinline__ uint16_t from(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
struct F32 {
  typedef float raw;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float one(float r) { return r; }
  static __device__ __forceinline__ void chunk(const u32x4& w, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i];
      v[i] = __builtin_bit_cast(float, u);
    }
  }
  static __device__ __forceinline__ u32x4 unchunk(const float* v) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, v[i]);
    return w;
  }
  static __device__ __forceinline__ float from(float v) { return v; }
};

template <typename T, int V>
__device__ __forceinline__ void load(const void* base, int64_t at, float* v) {
  const typename T::raw* p = (const typename T::raw*)base + at;
  if constexpr (V == 1) {
    v[0] = T::one(*p);
  } else {
    T::chunk(*(const u32x4*)p, v);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store(void* base, int64_t at, const float* v) {
  typename T::raw* p = (typename T::raw*)base + at;
  if constexpr (V == 1) {
    *p = T::from(v[0]);
  } else {
    *(u32x4*)p = T::unchunk(v);
  }
}

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int is64) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// Sum over the G lanes of a row's group (G a power of two).
__device__ __forceinline__ float group_sum(float v, int g) {
  for (int m = 1; m < g; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// ---------------------------------------------------------- qk_norm_rope --
//
//   n = x r w,  r = rsqrt(mean x^2 + eps)
//   y_i = n_i cos_i - n_{i+h} sin_i,  y_{i+h} = n_{i+h} cos_{i+h} + n_i sin_{i+h}   (i < h = dim / 2)
// and backward, from g = dL/dy:
//   dn_i = g_i cos_i + g_{i+h} sin_{i+h},  dn_{i+h} = g_{i+h} cos_{i+h} - g_i sin_i
//   dx = r (w dn - x r^2 mean(w dn x)),   dw = sum over rows of dn x r
//
// A group of G lanes holds one head row, a lane the V elements from V l of
// each half, so the rotation needs nothing from other lanes and the mean is a
// sum over the group.  Bound by memory: one read and one write of a row.  8192
// tokens x 12 heads x 128 in bf16: 10.8 us (50 MB at 4.6 TB/s), backward 18.7
// (75 MB at 4.0) and 3.1 for the weights' partial rows; a copy runs at 5.0.
// Four heads of a token per lane group share its table row (one: 11.8 us).

// Lanes past the half (a group is a power of two) repeat its first elements,
// so that no load has a branch, and count for nothing.
template <typename T, int V, int C>
struct Half {
  int d[C];    // this lane's elements of each half
  bool in[C];  // they exist
  __device__ __forceinline__ Half(int half, int l, int g) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      d[c] = (c * g + l) * V;
      in[c] = d[c] < half;
      d[c] = in[c] ? d[c] : 0;
    }
  }
  __device__ __forceinline__ void read(const void* base, int64_t at, int half, float (&lo)[C][V],
                                       float (&hi)[C][V]) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      load<T, V>(base, at + d[c], lo[c]);
      load<T, V>(base, at + half + d[c], hi[c]);
    }
  }
  __device__ __forceinline__ void write(void* base, int64_t at, int half, int c, const float (&lo)[V],
                                        const float (&hi)[V]) const {
    if (!in[c]) return;
    store<T, V>(base, at + d[c], lo);
    store<T, V>(base, at + half + d[c], hi);
  }
};

// cos and sin of a token: the tables' row, or NaN outside them.
template <typename T, int V, int C>
struct Rope {
  float clo[C][V], chi[C][V], slo[C][V], shi[C][V];
  __device__ __forceinline__ void read(const lm_rope_params& P, int64_t pos, const Half<T, V, C>& H) {
    const int half = P.dim >> 1;
    if (pos < 0 || pos >= P.table_rows) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) clo[c][j] = chi[c][j] = slo[c][j] = shi[c][j] = kNan;
      return;
    }
    const int64_t ac = pos * P.cos_ld, as = pos * P.sin_ld;
    if (P.table_f32) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          clo[c][j] = ((const float*)P.cos)[ac + H.d[c] + j];
          chi[c][j] = ((const float*)P.cos)[ac + half + H.d[c] + j];
          slo[c][j] = ((const float*)P.sin)[as + H.d[c] + j];
          shi[c][j] = ((const float*)P.sin)[as + half + H.d[c] + j];
        }
    } else {
      H.read(P.cos, ac, half, clo, chi);
      H.read(P.sin, as, half, slo, shi);
    }
  }
};

// Token n of the call as (sequence, token of it), and the position it is rotated by.
struct Token {
  uint32_t b, t;
  int64_t pos;
  __device__ __forceinline__ Token(const lm_rope_params& P, uint32_t n) {
    b = P.tokens == 1 ? n : n / (uint32_t)P.tokens;
    t = n - b * (uint32_t)P.tokens;
    pos = P.positions == nullptr ? (int64_t)t : index_at(P.positions, b * P.pos_b + t * P.pos_t, P.pos64);
  }
};

// blockIdx.y: HPG heads of the queries, then of the keys; a lane group takes them for one token.
template <typename T, int V, int C, int HPG>
__device__ __forceinline__ void qk_norm_rope_fwd(const lm_rope_params& P) {
  const int g = P.lanes, l = threadIdx.x & (g - 1);
  const uint32_t n = blockIdx.x * (blockDim.x / g) + threadIdx.x / g;
  if (n >= (uint32_t)P.batch * (uint32_t)P.tokens) return;
  const int qc = (P.heads[0] + HPG - 1) / HPG;
  const int x = (int)blockIdx.y < qc ? 0 : 1;
  const int h0 = ((int)blockIdx.y - (x ? qc : 0)) * HPG;
  const int half = P.dim >> 1;
  const lm_strides sx = x ? P.sx[1] : P.sx[0], sy = x ? P.sy[1] : P.sy[0];
  const int heads = x ? P.heads[1] : P.heads[0];
  const void* src = x ? P.x[1] : P.x[0];
  void* dst = x ? P.y[1] : P.y[0];
  const Token tok(P, n);
  const Half<T, V, C> H(half, l, g);
  const int64_t at = tok.b * sx.b + tok.t * sx.t, to = tok.b * sy.b + tok.t * sy.t;

  float lo[HPG][C][V], hi[HPG][C][V], wlo[C][V], whi[C][V];
#pragma unroll
  for (int i = 0; i < HPG; ++i)  // heads past the last repeat it
    H.read(src, at + (int64_t)(h0 + i < heads ? h0 + i : heads - 1) * sx.h, half, lo[i], hi[i]);
  Rope<T, V, C> R;
  R.read(P, tok.pos, H);
  H.read(x ? P.w[1] : P.w[0], 0, half, wlo, whi);
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s = __builtin_fmaf(lo[i][c][j], lo[i][c][j], s);
        s = __builtin_fmaf(hi[i][c][j], hi[i][c][j], s);
      }
      ss += H.in[c] ? s : 0.f;
    }
    const float r = __builtin_amdgcn_rsqf(group_sum(ss, g) * P.inv_dim + P.eps);
    if (h0 + i >= heads) break;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float ylo[V], yhi[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float a = lo[i][c][j] * r * wlo[c][j], e = hi[i][c][j] * r * whi[c][j];
        ylo[j] = a * R.clo[c][j] - e * R.slo[c][j];
        yhi[j] = e * R.chi[c][j] + a * R.shi[c][j];
      }
      H.write(dst, to + (int64_t)(h0 + i) * sy.h, half, c, ylo, yhi);
    }
  }
}

// blockIdx.y: P.chunk heads of the queries, then of the keys; the lane groups
// walk over the tokens.  Each lane keeps its columns' weight gradient; the
// workgroup adds its groups' in a fixed order and writes one row of partials.
template <typename T, int V, int C, int HPG>
__device__ __forceinline__ void qk_norm_rope_bwd(const lm_rope_params& P, float* red) {
  const int g = P.lanes, l = threadIdx.x & (g - 1);
  const int x = (int)blockIdx.y < P.q_chunks ? 0 : 1;
  const int half = P.dim >> 1;
  const lm_strides sx = x ? P.sx[1] : P.sx[0], sy = x ? P.sy[1] : P.sy[0], sg = x ? P.sg[1] : P.sg[0];
  const void* src = x ? P.x[1] : P.x[0];
  const void* gsrc = x ? P.g[1] : P.g[0];
  void* dst = x ? P.y[1] : P.y[0];
  const int heads = x ? P.heads[1] : P.heads[0];
  const int first = ((int)blockIdx.y - (x ? P.q_chunks : 0)) * P.chunk;
  const int end = first + P.chunk < heads ? first + P.chunk : heads;
  const int groups = blockDim.x / g, grp = threadIdx.x / g;
  const uint32_t tokens = (uint32_t)P.batch * (uint32_t)P.tokens;
  const Half<T, V, C> H(half, l, g);
  float wlo[C][V], whi[C][V], dwlo[C][V], dwhi[C][V];
  H.read(x ? P.w[1] : P.w[0], 0, half, wlo, whi);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) dwlo[c][j] = dwhi[c][j] = 0.f;
  for (uint32_t n = blockIdx.x * groups + grp; n < tokens; n += gridDim.x * groups) {
    const Token tok(P, n);
    const int64_t ax = tok.b * sx.b + tok.t * sx.t, ag = tok.b * sg.b + tok.t * sg.t, ay = tok.b * sy.b + tok.t * sy.t;
    Rope<T, V, C> R;
    for (int h0 = first; h0 < end; h0 += HPG) {
      float lo[HPG][C][V], hi[HPG][C][V], glo[HPG][C][V], ghi[HPG][C][V];
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        const int64_t h = h0 + i < end ? h0 + i : end - 1;
        H.read(src, ax + h * sx.h, half, lo[i], hi[i]);
        H.read(gsrc, ag + h * sg.h, half, glo[i], ghi[i]);
      }
      if (h0 == first) R.read(P, tok.pos, H);
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        float ss = 0.f, mx = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float s = 0.f, m = 0.f;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = lo[i][c][j], e = hi[i][c][j];
            s = __builtin_fmaf(a, a, s);
            s = __builtin_fmaf(e, e, s);
            const float da = glo[i][c][j] * R.clo[c][j] + ghi[i][c][j] * R.shi[c][j];
            const float de = ghi[i][c][j] * R.chi[c][j] - glo[i][c][j] * R.slo[c][j];
            glo[i][c][j] = da;
            ghi[i][c][j] = de;
            m = __builtin_fmaf(da * wlo[c][j], a, m);
            m = __builtin_fmaf(de * whi[c][j], e, m);
          }
          ss += H.in[c] ? s : 0.f;
          mx += H.in[c] ? m : 0.f;
        }
        ss = group_sum(ss, g);
        mx = group_sum(mx, g);
        const float r = __builtin_amdgcn_rsqf(ss * P.inv_dim + P.eps);
        const float k = r * r * mx * P.inv_dim;
        if (h0 + i >= end) break;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float olo[V], ohi[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = lo[i][c][j], e = hi[i][c][j], da = glo[i][c][j], de = ghi[i][c][j];
            olo[j] = r * (wlo[c][j] * da - a * k);
            ohi[j] = r * (whi[c][j] * de - e * k);
            dwlo[c][j] = __builtin_fmaf(da * a, r, dwlo[c][j]);
            dwhi[c][j] = __builtin_fmaf(de * e, r, dwhi[c][j]);
          }
          H.write(dst, ay + (int64_t)(h0 + i) * sy.h, half, c, olo, ohi);
        }
      }
    }
  }
  // the workgroup's weight gradient: groups in order
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (H.in[c]) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        red[grp * P.dim + H.d[c] + j] = dwlo[c][j];
        red[grp * P.dim + half + H.d[c] + j] = dwhi[c][j];
      }
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < P.dim; d += blockDim.x) {
    float s = 0.f;
    for (int i = 0; i < groups; ++i) s += red[i * P.dim + d];
    P.dw_part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * P.dim + d] = s;
  }
}

// Sums the partial rows: workgroup (32 columns, queries or keys), 32 row
// strides, added in a fixed order.
template <typename T>
__device__ __forceinline__ void rope_dw_sum(const lm_rope_params& P, float* red) {
  const int x = blockIdx.y, col = threadIdx.x & 31, str = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + col;
  const int first = x ? P.parts * P.q_chunks : 0, end = P.parts * (x ? P.chunks : P.q_chunks);
  float s = 0.f;
  if (d < P.dim) {
#pragma unroll 8
    for (int i = first + str; i < end; i += 32) s += P.dw_part[(int64_t)i * P.dim + d];
  }
  red[str * 33 + col] = s;
  __syncthreads();
  if (threadIdx.x < 32 && d < P.dim) {
    float tot = 0.f;
    for (int i = 0; i < 32; ++i) tot += red[i * 33 + col];
    void* dw = x ? P.dw[1] : P.dw[0];
    if (dw != nullptr) store<T, 1>(dw, d, &tot);
  }
}

// ------------------------------------------------------------- embedding --
//
//   out_n = scale w[id_n]          dw_r = scale sum over {n: id_n = r} of g_n
//
// The gradient sorts the tokens by row, stably, so that every row's sum has a
// fixed order whatever the launch.  Three launches:
//   sort   one workgroup per range of table rows.  Each scans all ids (they
//          stay in L2): its 16 waves, each a stretch of the tokens in order,
//          count their tokens per row in LDS; a scan over rows and waves
//          gives every (row, wave) its place, and the ids below the range the
//          range's own; a second walk places the tokens.  A wave requests
//          1024 ids at a time, so up to 16384 tokens are one round trip.
//   sum    one workgroup per stretch of `seg` sorted tokens and column slice:
//          runs of one row are added in order and written; a run that crosses
//          the stretch's ends is left as an fp32 partial row.  Further
//          workgroups zero the rows without tokens.
//   join   the crossing runs' partial rows are added in order.
// 16384 tokens of a text's frequencies, 49152 x 4096 in bf16: 13 + 89 (530 MB
// at 5.9 TB/s) + 9 us, the lookup 40 (190 MB or more at 4.7).

template <typename T, int V>
__device__ __forceinline__ void embedding_fwd(const lm_embed_params& P) {
  const int tpr = P.threads_per_row;
  const int64_t n = (int64_t)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  if (n >= P.n) return;
  const int64_t id = index_at(P.ids, n, P.ids64);
  const bool ok = id >= 0 && id < P.rows;
  for (int c = threadIdx.x & (tpr - 1); c * V < P.dim; c += tpr) {
    float v[V];
    if (ok) {
      load<T, V>(P.w, id * P.w_ld + c * V, v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= P.scale;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = kNan;
    }
    store<T, V>(P.out, n * P.dim + c * V, v);
  }
}

// A wave's next 64 x LM_EMBED_BATCH tokens: each lane's rows within the range, -1 elsewhere.
__device__ __forceinline__ void load_ids(const lm_embed_params& P, int64_t tb, int64_t t1, int lane, int64_t lo,
                                         int64_t hi, int (&rel)[LM_EMBED_BATCH], int& below) {
  int64_t id[LM_EMBED_BATCH];
#pragma unroll
  for (int i = 0; i < LM_EMBED_BATCH; ++i) {
    const int64_t t = tb + i * 64 + lane;
    id[i] = t < t1 ? index_at(P.ids, t, P.ids64) : -1;
  }
#pragma unroll
  for (int i = 0; i < LM_EMBED_BATCH; ++i) {
    const bool ok = id[i] >= 0 && id[i] != P.padding;
    rel[i] = ok && id[i] >= lo && id[i] < hi ? (int)(id[i] - lo) : -1;
    below += ok && id[i] < lo ? 1 : 0;
  }
}

// cnt: LM_EMBED_WAVES x range counters; scan: one word per wave
__device__ __forceinline__ void embedding_sort(const lm_embed_params& P, int* cnt, int* scan) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int range = P.range;
  const int64_t lo = (int64_t)blockIdx.x * range;
  const int64_t hi = lo + range < P.rows ? lo + range : P.rows;
  int* mine = cnt + wave * range;
  for (int i = threadIdx.x; i < range * LM_EMBED_WAVES; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int64_t per = ((P.n + LM_EMBED_WAVES - 1) / LM_EMBED_WAVES + 63) / 64 * 64;
  const int64_t t0 = per * wave, t1 = t0 + per < P.n ? t0 + per : P.n;
  int below = 0;
  int rel[LM_EMBED_BATCH];
  for (int64_t tb = t0; tb < t1; tb += 64 * LM_EMBED_BATCH) {
    load_ids(P, tb, t1, lane, lo, hi, rel, below);
#pragma unroll
    for (int i = 0; i < LM_EMBED_BATCH; ++i)
      if (rel[i] >= 0) atomicAdd(&mine[rel[i]], 1);
  }
  for (int m = 1; m < 64; m <<= 1) below += __shfl_xor(below, m);
  if (lane == 0) scan[wave] = below;
  __syncthreads();
  int base = 0;
  for (int i = 0; i < LM_EMBED_WAVES; ++i) base += scan[i];
  __syncthreads();
  // thread r: row lo + r
  const int r = threadIdx.x;
  int total = 0;
  if (r < range)
    for (int i = 0; i < LM_EMBED_WAVES; ++i) total += cnt[i * range + r];
  int incl = total;
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(incl, m);
    if (lane >= m) incl += o;
  }
  if (lane == 63) scan[wave] = incl;
  __syncthreads();
  int at = base + incl - total;
  for (int i = 0; i < wave; ++i) at += scan[i];
  if (r < range) {
    if (lo + r < P.rows) {
      P.row_count[lo + r] = total;
      P.row_start[lo + r] = at;
    }
    for (int i = 0; i < LM_EMBED_WAVES; ++i) {
      const int c = cnt[i * range + r];
      cnt[i * range + r] = at;
      at += c;
    }
  }
  if (blockIdx.x == gridDim.x - 1 && r == range - 1) P.counts[0] = at;  // tokens in all
  __syncthreads();
  // The walk that places: equal rows of a wave's 64 tokens take the next
  // places in the order of the lanes.
  for (int64_t tb = t0; tb < t1; tb += 64 * LM_EMBED_BATCH) {
    if (per > 64 * LM_EMBED_BATCH) load_ids(P, tb, t1, lane, lo, hi, rel, below);
#pragma unroll
    for (int i = 0; i < LM_EMBED_BATCH; ++i) {
      const int row = rel[i];
      uint64_t left = __ballot(row >= 0);
      while (left != 0) {
        const int lead = __builtin_ctzll(left);
        const int rr = __builtin_amdgcn_readlane(row, lead);
        const uint64_t same = __ballot(row == rr);
        const int from = *(volatile int*)&mine[rr];
        if (row == rr) {
          const int p = from + __popcll(same & (((uint64_t)1 << lane) - 1));
          P.sorted_token[p] = (int32_t)(tb + i * 64 + lane);
          P.sorted_row[p] = (int32_t)(lo + rr);
        }
        if (lane == lead) *(volatile int*)&mine[rr] = from + __popcll(same);
        left &= ~same;
      }
    }
  }
}

// The rows without tokens among LM_EMBED_ZERO rows from row0, this slice's columns.
template <typename T, int V>
__device__ __forceinline__ void embedding_zero(const lm_embed_params& P, int64_t row0) {
  const int lane = threadIdx.x & 63;
  const int64_t row = row0 + lane;
  const bool none = lane < LM_EMBED_ZERO && row < P.rows && P.row_count[row < P.rows ? row : 0] == 0;
  uint64_t left = __ballot(none);
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  if (c * V >= P.dim) return;
  float z[V];
#pragma unroll
  for (int j = 0; j < V; ++j) z[j] = 0.f;
  while (left != 0) {
    const int i = __builtin_ctzll(left);
    store<T, V>(P.dw, (row0 + i) * P.dim + c * V, z);
    left &= left - 1;
  }
}

template <typename T, int V>
__device__ __forceinline__ void embedding_sum(const lm_embed_params& P) {
  const int count = P.counts[0];
  if ((int)blockIdx.x >= P.stretches) {
    embedding_zero<T, V>(P, (int64_t)((int)blockIdx.x - P.stretches) * LM_EMBED_ZERO);
    return;
  }
  const int s0 = blockIdx.x * P.seg;
  if (s0 >= count) return;
  const int s1 = s0 + P.seg < count ? s0 + P.seg : count;
  // lane i: the stretch's i-th token and row (seg is at most 64)
  const int lane = threadIdx.x & 63;
  const int k = s0 + lane < s1 ? s0 + lane : s1 - 1;
  const int toks = P.sorted_token[k], rows = P.sorted_row[k];
  const int before = s0 > 0 ? P.sorted_row[s0 - 1] : -1;
  const int after = s1 < count ? P.sorted_row[s1] : -1;
  // Lanes past the row's end stay on, as they hold tokens and rows that the
  // others read: they sum its first columns and write nothing.
  const int at = blockIdx.y * blockDim.x + threadIdx.x;
  if ((at - lane) * V >= P.dim) return;
  const bool writes = at * V < P.dim;
  const int c = writes ? at : 0;
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  int row = __builtin_amdgcn_readlane(rows, 0);
  auto flush = [&](bool end) {
    // crossing the start: partial 0; crossing the end only: partial 1
    const bool head = row == before, tail = end && row == after;
    if (!writes) {
    } else if (head || tail) {
      float* p = P.part + ((int64_t)blockIdx.x * 2 + (head ? 0 : 1)) * P.dim + c * V;
#pragma unroll
      for (int j = 0; j < V; ++j) p[j] = acc[j];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] *= P.scale;
      store<T, V>(P.dw, (int64_t)row * P.dim + c * V, acc);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
  };
  constexpr int U = 8;
  const int len = s1 - s0;
  for (int i = 0; i < len; i += U) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)  // lanes past the stretch repeat its last token
      load<T, V>(P.g, (int64_t)__builtin_amdgcn_readlane(toks, i + u) * P.g_ld + c * V, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < len) {
        const int r = __builtin_amdgcn_readlane(rows, i + u);
        if (r != row) {
          flush(false);
          row = r;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += v[u][j];
      }
    }
  }
  flush(true);
}

// The partial rows first, first + step, ... of the run of stretches s .. e, 256
// columns d of them, added in order.  Columns past the row's end repeat its
// last: loads without a branch stay in flight together.
__device__ __forceinline__ void add_partials(const lm_embed_params& P, int s, int first, int e, int step,
                                             const int (&d)[4], float (&sum)[4]) {
  constexpr int U = 8;
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = 0.f;
  for (int k = first; k <= e; k += U * step) {
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = k + u * step <= e ? k + u * step : k;
      const float* p = P.part + ((int64_t)q * 2 + (q == s ? 1 : 0)) * P.dim;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[u][j] = p[d[j]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += k + u * step <= e ? v[u][j] : 0.f;
  }
}

// Workgroup (LM_EMBED_JOIN stretches, 256 columns), for each run that starts in
// one of them and leaves it.  A run of few partial rows is one wave's; the
// partial rows of a longer one are dealt out to the waves, and their sums
// added in order.  (One stretch per workgroup spent 27 us on dispatching 16368
// workgroups that mostly found no run, at 16384 tokens x 4096 in stretches of 16.)
template <typename T>
__device__ __forceinline__ void embedding_join(const lm_embed_params& P, float* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int total = P.counts[0];
  const int mine = blockIdx.x * LM_EMBED_JOIN + (lane & (LM_EMBED_JOIN - 1));  // this lane's stretch
  int row = -1, end = 0;
  if (lane < LM_EMBED_JOIN && mine < P.stretches - 1 && (mine + 1) * P.seg < total) {
    row = P.sorted_row[(mine + 1) * P.seg];
    const int start = P.row_start[row];
    if (start >= mine * P.seg && start < (mine + 1) * P.seg) end = (start + P.row_count[row] - 1) / P.seg;
    else row = -1;  // the run at this end starts elsewhere, or at the next stretch
  }
  uint64_t left = __ballot(row >= 0);
  const uint64_t lng = __ballot(row >= 0 && end - mine >= 2 * LM_EMBED_JOIN_WAVES);
  int d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    d[j] = blockIdx.y * 256 + 64 * j + lane;
    d[j] = d[j] < P.dim ? d[j] : P.dim - 1;
  }
  float sum[4];
  int turn = 0;
  while (left != 0) {
    const int i = __builtin_ctzll(left);
    left &= left - 1;
    const int s = blockIdx.x * LM_EMBED_JOIN + i;
    const int r = __builtin_amdgcn_readlane(row, i), e = __builtin_amdgcn_readlane(end, i);
    if (((lng >> i) & 1) == 0) {
      if ((turn++ & (LM_EMBED_JOIN_WAVES - 1)) != wave) continue;
      add_partials(P, s, s, e, 1, d, sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = sum[j] * P.scale;
        if ((int)(blockIdx.y * 256) + 64 * j + lane < P.dim) store<T, 1>(P.dw, (int64_t)r * P.dim + d[j], &v);
      }
      continue;
    }
    add_partials(P, s, s + wave, e, LM_EMBED_JOIN_WAVES, d, sum);
#pragma unroll
    for (int j = 0; j < 4; ++j) red[wave * 256 + 64 * j + lane] = sum[j];
    __syncthreads();
    if (threadIdx.x < 256 && (int)(blockIdx.y * 256 + threadIdx.x) < P.dim) {
      float v = 0.f;
      for (int w = 0; w < LM_EMBED_JOIN_WAVES; ++w) v += red[w * 256 + threadIdx.x];
      v *= P.scale;
      store<T, 1>(P.dw, (int64_t)r * P.dim + blockIdx.y * 256 + threadIdx.x, &v);
    }
    __syncthreads();
  }
}

}  // namespace

// C: chunks of a half row per lane; one except for scalar rows wider than 128.
#define LM_ROPE(NAME, T, V, C)                                                                      \
  extern "C" __global__ void __launch_bounds__(256) attnres_qk_norm_rope_##NAME##_h1(lm_rope_params P) { \
    qk_norm_rope_fwd<T, V, C, 1>(P);                                                                \
  }                                                                                                 \
  extern "C" __global__ void __launch_bounds__(256) attnres_qk_norm_rope_##NAME##_h4(lm_rope_params P) { \
    qk_norm_rope_fwd<T, V, C, 4>(P);                                                                \
  }                                                                                                 \
  extern "C" __global__ void __launch_bounds__(256) attnres_qk_norm_rope_bwd_##NAME(lm_rope_params P) { \
    extern __shared__ float lm_red[];                                                               \
    qk_norm_rope_bwd<T, V, C, 2>(P, lm_red);                                                        \
  }
LM_ROPE(bf16_v8, Bf16, 8, 1)
LM_ROPE(bf16_v1, Bf16, 1, 2)
LM_ROPE(f32_v4, F32, 4, 1)
LM_ROPE(f32_v1, F32, 1, 2)

#define LM_ROPE_SUM(NAME, T)                                                                          \
  extern "C" __global__ void __launch_bounds__(1024) attnres_qk_norm_rope_dw_##NAME(lm_rope_params P) { \
    __shared__ float red[32 * 33];                                                                    \
    rope_dw_sum<T>(P, red);                                                                           \
  }
LM_ROPE_SUM(bf16, Bf16)
LM_ROPE_SUM(f32, F32)

#define LM_EMBED(NAME, T, V)                                                                              \
  extern "C" __global__ void __launch_bounds__(256) attnres_embedding_fwd_##NAME(lm_embed_params P) {     \
    embedding_fwd<T, V>(P);                                                                               \
  }                                                                                                       \
  extern "C" __global__ void __launch_bounds__(512) attnres_embedding_sum_##NAME(lm_embed_params P) {     \
    embedding_sum<T, V>(P);                                                                               \
  }
LM_EMBED(bf16_v8, Bf16, 8)
LM_EMBED(bf16_v1, Bf16, 1)
LM_EMBED(f32_v4, F32, 4)
LM_EMBED(f32_v1, F32, 1)

extern "C" __global__ void __launch_bounds__(64 * LM_EMBED_WAVES) attnres_embedding_sort(lm_embed_params P) {
  __shared__ int cnt[LM_EMBED_WAVES * LM_EMBED_MAX_RANGE];
  __shared__ int scan[LM_EMBED_WAVES];
  embedding_sort(P, cnt, scan);
}
#define LM_EMBED_JOIN_K(NAME, T)                                                                       \
  extern "C" __global__ void __launch_bounds__(64 * LM_EMBED_JOIN_WAVES)                              \
      attnres_embedding_join_##NAME(lm_embed_params P) {                                              \
    __shared__ float red[256 * LM_EMBED_JOIN_WAVES];                                                  \
    embedding_join<T>(P, red);                                                                        \
  }
LM_EMBED_JOIN_K(bf16, Bf16)
LM_EMBED_JOIN_K(f32, F32)
