// Causal grouped-query attention for gfx950 (CDNA4): forward with the row
// log-sum-exp, and the backward that recomputes the probabilities from it.
//
//   s = scale q k^T (masked)   lse = log sum_j exp(s_j)   p = exp(s - lse)
//   o = p v
//   delta = sum_d do o - dlse   dp = do v^T   ds = p (dp - delta)
//   dq = scale ds k   dk = scale ds^T q   dv = p^T do
//
// The products run on the matrix cores in 32x32 tiles (v_mfma_f32_32x32x16 for
// bf16, eight v_mfma_f32_32x32x2 for fp32), everything else in fp32.  A wave
// owns 32 query rows (forward, dq) or 32 keys (dk, dv) and always forms the
// score tile with its own rows along the lanes: in the 32x32 result layout a
// lane holds one column and the rows 8a + 4h + b (a, b = 0..3, h = lane / 32),
// so the row statistics are a reduction over a lane's own registers and one
// exchange between lane halves.  The same registers are the next product's
// B operand as they stand: its 16-long k axis takes the rows in the order
// (h, j) -> 16 s + 8 (j / 4) + 4h + j % 4 that the lane already holds, and the
// A operand is read from LDS in that order (for bf16 with the transposing
// ds_read_b64_tr_b16: four rows of one column per lane), so probabilities
// never cross lanes or go through LDS.
//
// Tiles go from HBM to LDS directly (global_load_lds, 16 bytes per lane), the
// next one requested before the current one is worked on.  A tile row is held
// as 16-byte chunks, chunk c of row r at place c ^ g(r) with
// g = 2 (r % 8) + (r / 8) % 2: 16 rows of one chunk and 4 rows of a chunk pair
// each fall on distinct banks, so the row reads and the transposed reads of a
// tile are both free of conflicts.
//
// Rows beyond a sequence are never read: a tile's row index is clamped to the
// last row that exists, and what it gives is masked.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lm_params.h"

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

#define LM_LDS __attribute__((address_space(3)))
#define LM_GLOBAL __attribute__((address_space(1)))

namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  bf16x2 r = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float bf_lo(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __builtin_bit_cast(float, u & 0xffff0000u); }

// 2^x; v_exp_f32 gives 0 for -inf and flushes results under 2^-126.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// The value of the lane 32 away.
__device__ __forceinline__ float other_half(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(((int)(threadIdx.x & 63) ^ 32) << 2,
                                                                __builtin_bit_cast(int, v)));
}

// ------------------------------------------------------------- fragments --
//
// Frag<T>: eight elements of an operand along k: A row (or B column) lane % 32,
// k = 8 (lane / 32) + j of a 16-long step.

struct Bf16 {
  static constexpr int kBytes = 2;
  struct Frag {
    u32x4 w;
  };
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.w), __builtin_bit_cast(bf16x8, b.w),
                                                   c, 0, 0, 0);
  }
  static __device__ __forceinline__ Frag zero() { return Frag{u32x4{0, 0, 0, 0}}; }
  static __device__ __forceinline__ Frag load(const char* p) { return Frag{*reinterpret_cast<const u32x4*>(p)}; }
  // registers 8s .. 8s+7 of a result tile as the B operand of step s (rounded to bf16)
  static __device__ __forceinline__ Frag from_acc(const f32x16& c, int s) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.w[i] = pack_bf16(c[8 * s + 2 * i], c[8 * s + 2 * i + 1]);
    return f;
  }
  static __device__ __forceinline__ float get(const Frag& f, int j) {
    return (j & 1) ? bf_hi(f.w[j >> 1]) : bf_lo(f.w[j >> 1]);
  }
};

struct F32 {
  static constexpr int kBytes = 4;
  struct Frag {
    f32x4 lo, hi;
  };
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo[j], b.lo[j], c, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi[j], b.hi[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag zero() { return Frag{f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}}; }
  static __device__ __forceinline__ Frag load(const char* p) {
    return Frag{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 16)};
  }
  static __device__ __forceinline__ Frag from_acc(const f32x16& c, int s) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.lo[i] = c[8 * s + i];
      f.hi[i] = c[8 * s + 4 + i];
    }
    return f;
  }
  static __device__ __forceinline__ float get(const Frag& f, int j) { return j < 4 ? f.lo[j] : f.hi[j - 4]; }
};

// ------------------------------------------------------------- LDS tiles --

// A tile of R rows of DP elements in LDS (layout in the head comment).
template <typename T, int DP, int R>
struct Tile {
  static constexpr int kRowBytes = DP * T::kBytes;
  static constexpr int kChunks = kRowBytes / 16;  // per row
  static constexpr int kBytes = R * kRowBytes;
  static constexpr int kLoads = kBytes / 1024;  // wave-wide 16-byte loads

  static __device__ __forceinline__ int place(int row) {
    if constexpr (kChunks >= 16) return ((row << 1) & 14) | ((row >> 3) & 1);
    return ((row & 6) | ((row >> 3) & 1));  // 8 chunks: row r and r + 1 share 256 bytes
  }

  // Request rows row0 .. row0+R-1 of `src` (row stride `stride` bytes, `chunks`
  // 16-byte chunks each) into `lds`; the wave `wave` of `waves` takes its part.
  // Rows are clamped to first .. last, chunks to those that exist.
  static __device__ __forceinline__ void request(char* lds, const char* src, int64_t stride, int row0, int first,
                                                 int last, int chunks, int wave, int waves, int lane) {
#pragma unroll
    for (int i = 0; i < (kLoads + LM_ATTN_WAVES - 1) / LM_ATTN_WAVES; ++i) {
      const int ld = i * waves + wave;
      const int p = ld * 64 + lane;  // place in the tile, in chunks
      const int row = p / kChunks;
      int c = (p % kChunks) ^ place(row);
      c = c < chunks ? c : chunks - 1;
      int r = row0 + row;
      r = r < last ? r : last;
      r = r > first ? r : first;
      const char* g = src + (int64_t)r * stride + c * 16;
      __builtin_amdgcn_global_load_lds((const LM_GLOBAL void*)g, (LM_LDS void*)(lds + ld * 1024), 16, 0, 0);
    }
  }

  // Row `row`'s elements 16 step + 8h .. + 7 (an A operand with rows along m).
  static __device__ __forceinline__ typename T::Frag row_frag(const char* lds, int row, int step, int h) {
    typename T::Frag f;
    if constexpr (T::kBytes == 2) {
      f.w = *reinterpret_cast<const u32x4*>(lds + row * kRowBytes + (((2 * step + h) ^ place(row)) << 4));
    } else {
      const int c = 4 * step + 2 * h;
      f.lo = *reinterpret_cast<const f32x4*>(lds + row * kRowBytes + ((c ^ place(row)) << 4));
      f.hi = *reinterpret_cast<const f32x4*>(lds + row * kRowBytes + (((c + 1) ^ place(row)) << 4));
    }
    return f;
  }

  // Column 32 dt + lane % 32 over the rows row0 + 8 (j / 4) + 4h + j % 4, j = 0..7 (an A
  // operand with columns along m and a step's 16 rows along k); row0 a multiple of 16.
  static __device__ __forceinline__ typename T::Frag col_frag(const char* lds, int row0, int dt, int lane) {
    typename T::Frag f;
    const int h = lane >> 5;
    if constexpr (T::kBytes == 2) {
      const int s = lane & 15;
      const int r = row0 + 4 * h + (s >> 2);
      const int c = 4 * dt + 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
      const char* a = lds + r * kRowBytes + ((c ^ place(r)) << 4) + ((s & 1) << 3);
      const char* b = lds + (r + 8) * kRowBytes + ((c ^ place(r + 8)) << 4) + ((s & 1) << 3);
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LM_LDS i16x4*)a));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LM_LDS i16x4*)b));
      f.w = u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      const int d = 32 * dt + (lane & 31);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = row0 + 4 * h + j;
        f.lo[j] = *reinterpret_cast<const float*>(lds + r * kRowBytes + (((d >> 2) ^ place(r)) << 4) + ((d & 3) << 2));
        f.hi[j] = *reinterpret_cast<const float*>(lds + (r + 8) * kRowBytes + (((d >> 2) ^ place(r + 8)) << 4) +
                                                  ((d & 3) << 2));
      }
    }
    return f;
  }
};

// A global row as B operands: elements 16 step + 8h .. + 7; zero past `dim` or
// where the row does not exist.
template <typename T, int DP>
__device__ __forceinline__ void load_rows(typename T::Frag (&f)[DP / 16], const char* row, int dim, int h, bool live) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * h;
    f[s] = (live && d < dim) ? T::load(row + d * T::kBytes) : T::zero();
  }
}

// Four consecutive elements of an output row.
template <typename T>
__device__ __forceinline__ void store4(char* p, float a, float b, float c, float d) {
  if constexpr (T::kBytes == 2) {
    *reinterpret_cast<u32x2*>(p) = u32x2{pack_bf16(a, b), pack_bf16(c, d)};
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
  }
}

// A wave's 32 rows x DP result held as its transpose (lane: row lane % 32,
// registers: columns), scaled and stored; only columns under dim.
template <typename T, int DP>
__device__ __forceinline__ void store_rows(char* row, const f32x16 (&acc)[DP / 32], float scale, int dim, int h) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * dt + 8 * a + 4 * h;
      if (d < dim)
        store4<T>(row + d * T::kBytes, acc[dt][4 * a] * scale, acc[dt][4 * a + 1] * scale, acc[dt][4 * a + 2] * scale,
                  acc[dt][4 * a + 3] * scale);
    }
  }
}

// ------------------------------------------------------------ work items --

// Consecutive workgroups go to the eight XCDs in turn, each with an L2 of its
// own; item w of XCD x is x * per + w, so a head's tiles stay on one XCD and
// its keys and values in that L2.  -1: no work.
__device__ __forceinline__ int work_item(int n) {
  const int per = (n + 7) >> 3;
  const int w = (int)(blockIdx.x >> 3);
  const int item = (int)(blockIdx.x & 7) * per + w;
  return w < per && item < n ? item : -1;
}

struct Seq {
  int kv_len;  // keys that exist
  int start;   // position of query 0
  int lo, hi;  // queries lo .. hi-1 see keys (causal: those at positions 0 .. kv_len-1)
};
__device__ __forceinline__ int64_t index_at(const void* p, int i, int is64) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
__device__ __forceinline__ Seq sequence(const lm_attn_params& P, int b) {
  Seq s;
  int n = P.kv_len;
  if (P.kv_lens != nullptr) {
    const int64_t len = index_at(P.kv_lens, b, P.lens64);
    n = len < 0 ? 0 : len > P.kv_len ? P.kv_len : (int)len;
  }
  int64_t st = P.q_start_const;
  if (P.q_start != nullptr) st = index_at(P.q_start, b, P.start64);
  st = st < -((int64_t)1 << 40) ? -((int64_t)1 << 40) : st > ((int64_t)1 << 40) ? (int64_t)1 << 40 : st;
  if (P.start_from_end) st = (int64_t)n - P.q_len;
  int64_t lo = 0, hi = P.q_len;
  if (P.causal) {
    if (-st > lo) lo = -st;
    if ((int64_t)n - st < hi) hi = (int64_t)n - st;
  } else if (n == 0) {
    hi = 0;
  }
  if (lo > P.q_len) lo = P.q_len;
  if (hi < lo) hi = lo;
  s.kv_len = n;
  s.lo = (int)lo;
  s.hi = (int)hi;
  // out of range only where no query is live
  s.start = (int)(st < -(1 << 30) ? -(1 << 30) : st > (1 << 30) ? (1 << 30) : st);
  return s;
}

// --------------------------------------------------------------- forward --

template <typename T, int DP>
__device__ __forceinline__ void attention_fwd(const lm_attn_params& P, char* k0, char* k1, char* v0, char* v1) {
  using KT = Tile<T, DP, LM_ATTN_KEYS>;
  const int item = work_item(P.n_items);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int tile = P.n_tiles - 1 - item % P.n_tiles;  // the longest rows first
  const int head = (item / P.n_tiles) % P.heads;
  const int b = item / (P.n_tiles * P.heads);
  const int kvh = head / (P.heads / P.kv_heads);
  const Seq S = sequence(P, b);
  const int row = tile * LM_ATTN_ROWS + wave * 32 + (lane & 31);
  const bool live = row >= S.lo && row < S.hi;
  const int lim = live ? (P.causal ? S.start + row + 1 : S.kv_len) : 0;  // keys the row sees
  // over the wave's rows: the most any row sees, and what every row sees; over the workgroup's: tiles to read
  const int r0 = tile * LM_ATTN_ROWS + wave * 32;
  const int w_hi = r0 + 32 < S.hi ? r0 + 32 : S.hi, w_lo = r0 > S.lo ? r0 : S.lo;
  const int w_max = w_hi <= w_lo ? 0 : P.causal ? S.start + w_hi : S.kv_len;
  const int w_min = (r0 < S.lo || r0 + 32 > S.hi) ? 0 : P.causal ? S.start + r0 + 1 : S.kv_len;
  const int g0 = tile * LM_ATTN_ROWS;
  const int g_hi = g0 + LM_ATTN_ROWS < S.hi ? g0 + LM_ATTN_ROWS : S.hi, g_lo = g0 > S.lo ? g0 : S.lo;
  const int g_max = g_hi <= g_lo ? 0 : P.causal ? S.start + g_hi : S.kv_len;
  const int tiles = (g_max + LM_ATTN_KEYS - 1) / LM_ATTN_KEYS;

  const int chunks = P.dim * T::kBytes / 16;
  const char* kp = (const char*)P.k + ((int64_t)b * P.sk.b + (int64_t)kvh * P.sk.h) * T::kBytes;
  const char* vp = (const char*)P.v + ((int64_t)b * P.sv.b + (int64_t)kvh * P.sv.h) * T::kBytes;
  const int64_t kst = P.sk.t * T::kBytes, vst = P.sv.t * T::kBytes;
  const int last = S.kv_len - 1;

  typename T::Frag qf[DP / 16];
  load_rows<T, DP>(qf, (const char*)P.q + ((int64_t)b * P.sq.b + (int64_t)head * P.sq.h + (int64_t)row * P.sq.t) * T::kBytes,
                   P.dim, h, live);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = zero16();
  float m = kNegInf, l = 0.f;  // running maximum (of scores times log2 e) and this lane's part of the sum

  if (tiles > 0) {
    KT::request(k0, kp, kst, 0, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
    KT::request(v0, vp, vst, 0, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
  }
  auto step = [&](int t, const char* kc, const char* vc, char* kn, char* vn) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < tiles) {
      KT::request(kn, kp, kst, (t + 1) * LM_ATTN_KEYS, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
      KT::request(vn, vp, vst, (t + 1) * LM_ATTN_KEYS, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
    }
    const int key0 = t * LM_ATTN_KEYS;
    if (key0 >= w_max) return;
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = zero16();
#pragma unroll
      for (int st = 0; st < DP / 16; ++st)
        s[kb] = T::mma(KT::row_frag(kc, 32 * kb + (lane & 31), st, h), qf[st], s[kb]);
    }
    if (key0 + LM_ATTN_KEYS > w_min) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key0 + 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3);
          s[kb][i] = key < lim ? s[kb][i] : kNegInf;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    top = fmaxf(top, other_half(top)) * P.scale_log2;
    const float mn = fmaxf(m, top);
    const float ref = mn == kNegInf ? 0.f : mn;
    const float fade = exp2_fast(m - ref);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb][i] = exp2_fast(__builtin_fmaf(s[kb][i], P.scale_log2, -ref));
        sum += s[kb][i];
      }
    l = __builtin_fmaf(l, fade, sum);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[dt][i] *= fade;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const typename T::Frag p = T::from_acc(s[kb], st);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
          acc[dt] = T::mma(KT::col_frag(vc, 32 * kb + 16 * st, dt, lane), p, acc[dt]);
      }
  };
  for (int t = 0; t < tiles; t += 2) {
    step(t, k0, v0, k1, v1);
    if (t + 1 < tiles) step(t + 1, k1, v1, k0, v0);
  }

  l += other_half(l);
  if (row < P.q_len) {
    const float inv = l > 0.f ? 1.f / l : 0.f;
    char* op = (char*)P.o + ((int64_t)b * P.so.b + (int64_t)head * P.so.h + (int64_t)row * P.so.t) * T::kBytes;
    store_rows<T, DP>(op, acc, inv, P.dim, h);
    if (P.lse != nullptr && h == 0)
      P.lse[((int64_t)b * P.heads + head) * P.q_len + row] = l > 0.f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : kNegInf;
  }
}

// -------------------------------------------------------- query gradients --

template <typename T, int DP>
__device__ __forceinline__ void attention_bwd_dq(const lm_attn_params& P, char* k0, char* k1, char* v0, char* v1) {
  using KT = Tile<T, DP, LM_ATTN_KEYS>;
  const int item = work_item(P.n_items);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int tile = P.n_tiles - 1 - item % P.n_tiles;
  const int head = (item / P.n_tiles) % P.heads;
  const int b = item / (P.n_tiles * P.heads);
  const int kvh = head / (P.heads / P.kv_heads);
  const Seq S = sequence(P, b);
  const int r0 = tile * LM_ATTN_ROWS + wave * 32;
  const int row = r0 + (lane & 31);
  const bool live = row >= S.lo && row < S.hi;
  const int lim = live ? (P.causal ? S.start + row + 1 : S.kv_len) : 0;
  const int w_hi = r0 + 32 < S.hi ? r0 + 32 : S.hi, w_lo = r0 > S.lo ? r0 : S.lo;
  const int w_max = w_hi <= w_lo ? 0 : P.causal ? S.start + w_hi : S.kv_len;
  const int w_min = (r0 < S.lo || r0 + 32 > S.hi) ? 0 : P.causal ? S.start + r0 + 1 : S.kv_len;
  const int g0 = tile * LM_ATTN_ROWS;
  const int g_hi = g0 + LM_ATTN_ROWS < S.hi ? g0 + LM_ATTN_ROWS : S.hi, g_lo = g0 > S.lo ? g0 : S.lo;
  const int g_max = g_hi <= g_lo ? 0 : P.causal ? S.start + g_hi : S.kv_len;
  const int tiles = (g_max + LM_ATTN_KEYS - 1) / LM_ATTN_KEYS;

  const int chunks = P.dim * T::kBytes / 16;
  const char* kp = (const char*)P.k + ((int64_t)b * P.sk.b + (int64_t)kvh * P.sk.h) * T::kBytes;
  const char* vp = (const char*)P.v + ((int64_t)b * P.sv.b + (int64_t)kvh * P.sv.h) * T::kBytes;
  const int64_t kst = P.sk.t * T::kBytes, vst = P.sv.t * T::kBytes;
  const int last = S.kv_len - 1;
  if (tiles > 0) {
    KT::request(k0, kp, kst, 0, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
    KT::request(v0, vp, vst, 0, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
  }

  typename T::Frag qf[DP / 16], gf[DP / 16];
  load_rows<T, DP>(qf, (const char*)P.q + ((int64_t)b * P.sq.b + (int64_t)head * P.sq.h + (int64_t)row * P.sq.t) * T::kBytes,
                   P.dim, h, live);
  load_rows<T, DP>(gf, (const char*)P.grad_out +
                           ((int64_t)b * P.sdo.b + (int64_t)head * P.sdo.h + (int64_t)row * P.sdo.t) * T::kBytes,
                   P.dim, h, live);
  const int64_t stat = ((int64_t)b * P.heads + head) * P.q_len + row;
  float delta = 0.f, lse2 = 0.f;
  {
    typename T::Frag of[DP / 16];
    load_rows<T, DP>(of, (const char*)P.out +
                             ((int64_t)b * P.sout.b + (int64_t)head * P.sout.h + (int64_t)row * P.sout.t) * T::kBytes,
                     P.dim, h, live);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = __builtin_fmaf(T::get(gf[s], j), T::get(of[s], j), delta);
    delta += other_half(delta);
    if (live) {
      lse2 = P.lse[stat] * kLog2e;
      if (P.grad_lse != nullptr) delta -= P.grad_lse[stat];
    }
    if (row < P.q_len && h == 0) P.delta[stat] = delta;
  }

  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = zero16();
  auto step = [&](int t, const char* kc, const char* vc, char* kn, char* vn) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < tiles) {
      KT::request(kn, kp, kst, (t + 1) * LM_ATTN_KEYS, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
      KT::request(vn, vp, vst, (t + 1) * LM_ATTN_KEYS, 0, last, chunks, wave, LM_ATTN_WAVES, lane);
    }
    const int key0 = t * LM_ATTN_KEYS;
    if (key0 >= w_max) return;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int st = 0; st < DP / 16; ++st) {
        s = T::mma(KT::row_frag(kc, 32 * kb + (lane & 31), st, h), qf[st], s);
        dp = T::mma(KT::row_frag(vc, 32 * kb + (lane & 31), st, h), gf[st], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = exp2_fast(__builtin_fmaf(s[i], P.scale_log2, -lse2)) * (dp[i] - delta);
      if (key0 + LM_ATTN_KEYS > w_min) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key0 + 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3);
          s[i] = key < lim ? s[i] : 0.f;
        }
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const typename T::Frag ds = T::from_acc(s, st);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
          acc[dt] = T::mma(KT::col_frag(kc, 32 * kb + 16 * st, dt, lane), ds, acc[dt]);
      }
    }
  };
  for (int t = 0; t < tiles; t += 2) {
    step(t, k0, v0, k1, v1);
    if (t + 1 < tiles) step(t + 1, k1, v1, k0, v0);
  }
  if (row < P.q_len) {
    char* op = (char*)P.dq + ((int64_t)b * P.sdq.b + (int64_t)head * P.sdq.h + (int64_t)row * P.sdq.t) * T::kBytes;
    store_rows<T, DP>(op, acc, P.scale, P.dim, h);
  }
}

// ------------------------------------------------ key and value gradients --

template <typename T, int DP>
__device__ __forceinline__ void attention_bwd_dkv(const lm_attn_params& P, char* q0, char* q1, char* g0, char* g1,
                                                  float* st0, float* st1) {
  using QT = Tile<T, DP, LM_ATTN_BWD_ROWS>;
  constexpr int R = LM_ATTN_BWD_ROWS;
  const int item = work_item(P.n_items);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int tile = item % P.n_tiles;  // causal: the first keys are seen by the most queries
  const int kvh = (item / P.n_tiles) % P.kv_heads;
  const int b = item / (P.n_tiles * P.kv_heads);
  const int group = P.heads / P.kv_heads;
  const Seq S = sequence(P, b);
  const int w0 = tile * LM_ATTN_BWD_KEYS + wave * 32;
  const int key = w0 + (lane & 31);
  const bool live = key < S.kv_len;

  typename T::Frag kf[DP / 16], vf[DP / 16];
  load_rows<T, DP>(kf, (const char*)P.k + ((int64_t)b * P.sk.b + (int64_t)kvh * P.sk.h + (int64_t)key * P.sk.t) * T::kBytes,
                   P.dim, h, live);
  load_rows<T, DP>(vf, (const char*)P.v + ((int64_t)b * P.sv.b + (int64_t)kvh * P.sv.h + (int64_t)key * P.sv.t) * T::kBytes,
                   P.dim, h, live);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) {
    dk[i] = zero16();
    dv[i] = zero16();
  }
  // the first query that sees the workgroup's (the wave's) first key, rounded down to a tile; queries of a head
  const int key_wg = tile * LM_ATTN_BWD_KEYS;
  int first = S.lo, w_first = S.lo, w_full = S.lo;  // from w_full on a query sees all of the wave's keys
  if (P.causal) {
    if (key_wg - S.start > first) first = key_wg - S.start;
    if (w0 - S.start > w_first) w_first = w0 - S.start;
    if (w0 + 31 - S.start > w_full) w_full = w0 + 31 - S.start;
  }
  if (w0 + 32 > S.kv_len) w_full = S.hi;  // not every key exists
  const int k_first = live ? (P.causal && key - S.start > S.lo ? key - S.start : S.lo) : S.hi;
  const int base = first / R * R;
  const int per = key_wg < S.kv_len && first < S.hi ? (S.hi - base + R - 1) / R : 0;  // tiles of a head
  const int tiles = per * group;

  const int chunks = P.dim * T::kBytes / 16;
  const int64_t qst = P.sq.t * T::kBytes, gst = P.sdo.t * T::kBytes;
  const int last = S.hi - 1;
  auto request = [&](int t, char* qn, char* gn, float* sn) {
    const int head = kvh * group + t / per;
    const int row0 = base + (t % per) * R;
    const char* qp = (const char*)P.q + ((int64_t)b * P.sq.b + (int64_t)head * P.sq.h) * T::kBytes;
    const char* gp = (const char*)P.grad_out + ((int64_t)b * P.sdo.b + (int64_t)head * P.sdo.h) * T::kBytes;
    QT::request(qn, qp, qst, row0, S.lo, last, chunks, wave, LM_ATTN_WAVES, lane);
    QT::request(gn, gp, gst, row0, S.lo, last, chunks, wave, LM_ATTN_WAVES, lane);
    if (wave == 0) {  // the rows' lse (lanes 0 .. 31) and delta
      int r = row0 + (lane & (R - 1));
      r = r < last ? r : last;
      r = r > S.lo ? r : S.lo;
      const float* src = (h ? P.delta : P.lse) + ((int64_t)b * P.heads + head) * P.q_len + r;
      __builtin_amdgcn_global_load_lds((const LM_GLOBAL void*)src, (LM_LDS void*)sn, 4, 0, 0);
    }
  };
  if (tiles > 0) request(0, q0, g0, st0);
  auto step = [&](int t, const char* qc, const char* gc, const float* sc, char* qn, char* gn, float* sn) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < tiles) request(t + 1, qn, gn, sn);
    const int row0 = base + (t % per) * R;
    if (row0 + R <= w_first || w0 >= S.kv_len) return;
    f32x16 s = zero16(), dp = zero16();
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) {
      s = T::mma(QT::row_frag(qc, lane & 31, st, h), kf[st], s);
      dp = T::mma(QT::row_frag(gc, lane & 31, st, h), vf[st], dp);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 lse = *reinterpret_cast<const f32x4*>(sc + 8 * a + 4 * h);
      const f32x4 dl = *reinterpret_cast<const f32x4*>(sc + 32 + 8 * a + 4 * h);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[4 * a + c] = exp2_fast(__builtin_fmaf(s[4 * a + c], P.scale_log2, -lse[c] * kLog2e));
        dp[4 * a + c] -= dl[c];
      }
    }
    if (row0 < w_full || row0 + R > S.hi) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = row0 + 8 * (i >> 2) + 4 * h + (i & 3);
        const bool seen = r >= k_first && r < S.hi;
        s[i] = seen ? s[i] : 0.f;
        dp[i] = seen ? dp[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] *= s[i];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const typename T::Frag p = T::from_acc(s, st), ds = T::from_acc(dp, st);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        dv[dt] = T::mma(QT::col_frag(gc, 16 * st, dt, lane), p, dv[dt]);
        dk[dt] = T::mma(QT::col_frag(qc, 16 * st, dt, lane), ds, dk[dt]);
      }
    }
  };
  for (int t = 0; t < tiles; t += 2) {
    step(t, q0, g0, st0, q1, g1, st1);
    if (t + 1 < tiles) step(t + 1, q1, g1, st1, q0, g0, st0);
  }
  if (key < P.kv_len) {
    char* kp = (char*)P.dk + ((int64_t)b * P.sdk.b + (int64_t)kvh * P.sdk.h + (int64_t)key * P.sdk.t) * T::kBytes;
    char* vp = (char*)P.dv + ((int64_t)b * P.sdv.b + (int64_t)kvh * P.sdv.h + (int64_t)key * P.sdv.t) * T::kBytes;
    store_rows<T, DP>(kp, dk, P.scale, P.dim, h);
    store_rows<T, DP>(vp, dv, 1.f, P.dim, h);
  }
}

}  // namespace

#define LM_ATTN_FWD(NAME, T, DP, WPE)                                                                   \
  extern "C" __global__ void __launch_bounds__(64 * LM_ATTN_WAVES) __attribute__((amdgpu_waves_per_eu(WPE))) \
      attnres_attention_fwd_##NAME(lm_attn_params P) {                                                  \
    __shared__ __align__(16) char k0[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    __shared__ __align__(16) char k1[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    __shared__ __align__(16) char v0[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    __shared__ __align__(16) char v1[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    attention_fwd<T, DP>(P, k0, k1, v0, v1);                                                            \
  }
#define LM_ATTN_DQ(NAME, T, DP, WPE)                                                                    \
  extern "C" __global__ void __launch_bounds__(64 * LM_ATTN_WAVES) __attribute__((amdgpu_waves_per_eu(WPE))) \
      attnres_attention_dq_##NAME(lm_attn_params P) {                                                   \
    __shared__ __align__(16) char k0[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    __shared__ __align__(16) char k1[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    __shared__ __align__(16) char v0[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    __shared__ __align__(16) char v1[Tile<T, DP, LM_ATTN_KEYS>::kBytes];                                \
    attention_bwd_dq<T, DP>(P, k0, k1, v0, v1);                                                         \
  }
#define LM_ATTN_DKV(NAME, T, DP, WPE)                                                                   \
  extern "C" __global__ void __launch_bounds__(64 * LM_ATTN_WAVES) __attribute__((amdgpu_waves_per_eu(WPE))) \
      attnres_attention_dkv_##NAME(lm_attn_params P) {                                                  \
    __shared__ __align__(16) char q0[Tile<T, DP, LM_ATTN_BWD_ROWS>::kBytes];                            \
    __shared__ __align__(16) char q1[Tile<T, DP, LM_ATTN_BWD_ROWS>::kBytes];                            \
    __shared__ __align__(16) char g0[Tile<T, DP, LM_ATTN_BWD_ROWS>::kBytes];                            \
    __shared__ __align__(16) char g1[Tile<T, DP, LM_ATTN_BWD_ROWS>::kBytes];                            \
    __shared__ __align__(16) float st0[64];                                                             \
    __shared__ __align__(16) float st1[64];                                                             \
    attention_bwd_dkv<T, DP>(P, q0, q1, g0, g1, st0, st1);                                              \
  }

#if LM_PART == 13
LM_ATTN_FWD(bf16_d64, Bf16, 64, 2)
LM_ATTN_FWD(bf16_d128, Bf16, 128, 2)
LM_ATTN_DQ(bf16_d64, Bf16, 64, 2)
LM_ATTN_DQ(bf16_d128, Bf16, 128, 2)
LM_ATTN_DKV(bf16_d64, Bf16, 64, 2)
LM_ATTN_DKV(bf16_d128, Bf16, 128, 1)
#endif
#if LM_PART == 14
LM_ATTN_FWD(f32_d64, F32, 64, 1)
LM_ATTN_FWD(f32_d128, F32, 128, 1)
LM_ATTN_DQ(f32_d64, F32, 64, 1)
LM_ATTN_DQ(f32_d128, F32, 128, 1)
LM_ATTN_DKV(f32_d64, F32, 64, 1)
LM_ATTN_DKV(f32_d128, F32, 128, 1)
#endif
