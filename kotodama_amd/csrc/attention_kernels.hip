// Causal grouped-query attention for gfx950 (CDNA4): forward with the row
// log-sum-exp, and the backward that recomputes the probabilities from it.
//
//   s = scale q k^T (masked)   lse = log sum_j exp(s_j)   p = exp(s - lse)
//   o = p v
//   delta = sum_d do o - dlse   dp = do v^T   ds = p (dp - delta)
//   dq = scale ds k   dk = scale ds^T q   dv = p^T do
//
// A wave owns 32 query rows (forward, dq) or 32 keys (dk, dv); products, tiles and
// the softmax of its rows are those of attention_tiles.h.
//
// The rows of a key head's query group are taken together, query by query:
// row r is head r % group of query r / group.  Consecutive rows then end at
// (nearly) the same key, a workgroup reads a key tile once for the whole
// group, and few queries still fill a tile.
//
// A tile is requested before the one in front of it is worked on.  The transposed
// reads' conflicts (attention_tiles.h) take 33, 25 and 28% of the cycles of the LDS in the
// forward, dq and (dk, dv) at 2 x 4096 tokens, 32/8 heads of 128.
//
// Rows beyond a sequence are never read: a tile's row index is clamped to the
// last row that exists, and what it gives is masked.

#include "attention_tiles.h"

namespace {

constexpr int kExactKeys = 256;  // rows of up to so many keys: delta from the probabilities (attention_bwd_dq)

// ------------------------------------------------------------ work items --

// Workgroup -> (tile rank, sequence and key head).  Consecutive workgroups go
// to the eight XCDs in turn, each with an L2 of its own: where the key heads
// divide by eight, each XCD takes an eighth of them, so that a head's keys and
// values stay in one L2.  Ranks are in order of falling work (causal), all
// heads' first tiles before their second.  Where all of an XCD's workgroups
// run at once, two on a CU, the second half is in rising order: a long one and
// a short one meet on each CU.
struct Item {
  int rank, head;  // rank < 0: no work
};
__device__ __forceinline__ Item work_item(const lm_attn_params& P) {
  const int heads = P.batch * P.kv_heads;
  const int x = (int)(blockIdx.x & 7);
  const int per = (int)(gridDim.x >> 3);
  int w = (int)(blockIdx.x >> 3);
  if (per <= 2 * P.cus_per_xcd && w >= P.cus_per_xcd) w = per - 1 - (w - P.cus_per_xcd);
  Item it;
  if ((heads & 7) == 0) {
    const int hx = heads >> 3;
    it.rank = w / hx;
    it.head = x * hx + (w - it.rank * hx);
  } else {
    const int i = w * 8 + x;
    it.rank = i / heads;
    it.head = i - it.rank * heads;
  }
  if (it.rank >= P.n_tiles) it.rank = -1;
  return it;
}

struct Seq {
  int kv_len;  // keys that exist
  int start;   // position of query 0
  int lo, hi;  // rows lo .. hi-1 see keys (causal: those of queries at positions 0 .. kv_len-1)
};
__device__ __forceinline__ Seq sequence(const lm_attn_params& P, int b, int group) {
  Seq s;
  int n = P.kv_len;
  if (P.kv_lens != nullptr) {
    const int64_t len = index_at(P.kv_lens, b, P.lens64);
    n = len < 0 ? 0 : len > P.kv_len ? P.kv_len : (int)len;
  }
  int64_t st = P.q_start_const;
  if (P.q_start != nullptr) st = index_at(P.q_start, b, P.start64);
  if (P.start_from_end) st = (int64_t)n - P.q_len;
  // a start this far out leaves no query a key, and is held where 32 bits can count from it
  st = st < -(1 << 30) ? -(1 << 30) : st > (1 << 30) ? (1 << 30) : st;
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
  s.lo = (int)lo * group;
  s.hi = (int)hi * group;
  s.start = (int)st;
  return s;
}

// The keys that rows r0 .. r0+n-1 see: the most any sees, and what all see.
struct Span {
  int most, all;
};
__device__ __forceinline__ Span span(const lm_attn_params& P, const Seq& S, int group, int r0, int n) {
  const int hi = r0 + n < S.hi ? r0 + n : S.hi, lo = r0 > S.lo ? r0 : S.lo;
  Span k;
  k.most = hi <= lo ? 0 : P.causal ? S.start + (hi - 1) / group + 1 : S.kv_len;
  k.all = (r0 < S.lo || r0 + n > S.hi) ? 0 : P.causal ? S.start + r0 / group + 1 : S.kv_len;
  return k;
}

// What a kernel whose waves own 32 rows each starts from.  KS waves share their
// rows and split each key tile.
template <int KS>
struct Rows {
  static constexpr int kPerGroup = 32 * LM_ATTN_WAVES / KS;  // rows of a workgroup
  static constexpr int kKeys = KS == 4 ? 128 : 64;           // keys of a tile
  static constexpr int kBlocks = kKeys / 32 / KS;            // 32-key blocks of a wave in a tile
  int lane, wave, h, part;  // part: which of the KS
  int b, kvh, head;         // this lane's row's query head
  int row, query;           // this lane's row, and its query
  bool exists, live;        // the row is there; it sees a key
  int lim;                  // keys it sees
  Span mine;                // the wave's rows'
  int split;                // which part of the key tiles this workgroup takes
  int t0, t1;               // its key tiles
  Seq S;

  __device__ __forceinline__ bool init(const lm_attn_params& P) {
    const Item it = work_item(P);
    if (it.rank < 0) return false;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    h = lane >> 5;
    part = wave % KS;
    kvh = it.head % P.kv_heads;
    b = it.head / P.kv_heads;
    const int group = P.heads / P.kv_heads;
    const int rows = P.q_len * group;
    split = 0;
    int rank = it.rank;
    if (KS == 4 && P.splits > 1) {
      rank = it.rank / P.splits;
      split = it.rank - rank * P.splits;
    }
    const int g0 = (P.n_tiles / (KS == 4 ? P.splits : 1) - 1 - rank) * kPerGroup;
    const int r0 = g0 + wave / KS * 32;
    S = sequence(P, b, group);
    row = r0 + (lane & 31);
    query = row / group;
    head = kvh * group + (row - query * group);
    exists = row < rows;
    live = row >= S.lo && row < S.hi;
    lim = live ? (P.causal ? S.start + query + 1 : S.kv_len) : 0;
    mine = span(P, S, group, r0, 32);
    t0 = 0;
    t1 = (span(P, S, group, g0, kPerGroup).most + kKeys - 1) / kKeys;
    if (KS == 4 && P.splits > 1) {
      const int each = (t1 + P.splits - 1) / P.splits;
      t0 = split * each < t1 ? split * each : t1;
      t1 = t0 + each < t1 ? t0 + each : t1;
    }
    return true;
  }
  // this row among all rows of the call
  __device__ __forceinline__ int64_t index(const lm_attn_params& P) const {
    return ((int64_t)b * P.kv_heads + kvh) * ((int64_t)P.q_len * (P.heads / P.kv_heads)) + row;
  }
  __device__ __forceinline__ int64_t stat(const lm_attn_params& P) const {
    return ((int64_t)b * P.heads + head) * P.q_len + query;
  }
};

// Runs step(t, k, v) over the key tiles t0 .. t1-1 in LDS.  NBUF 2: the waves
// share the tiles; tile t+1 is requested before t is worked on.  NBUF 1 (four
// waves share their rows): each reads only its own 32 keys of a tile, so it
// loads them itself, up to `most` keys, and no wave waits for another.
template <typename KT, int NBUF, typename Step>
__device__ __forceinline__ void over_keys(const char* kp, int64_t kst, const char* vp, int64_t vst, int t0, int t1,
                                          int last, int chunks, int wave, int lane, int most, char* k0, char* k1,
                                          char* v0, char* v1, Step&& step) {
  if constexpr (NBUF == 1) {
    using MT = typename KT::Mine;
    static_assert(KT::kRows == 32 * LM_ATTN_WAVES, "a tile has 32 keys for each wave");
    const int own = 32 * wave;
    for (int t = t0; t < t1 && t * KT::kRows + own < most; ++t) {
      int ln = lane;  // opaque: offsets formed anew for each tile instead of held in registers
      asm volatile("" : "+v"(ln));
      MT::request(k0 + own * KT::kRowBytes, kp, kst, t * KT::kRows + own, last, chunks, 0, ln);
      MT::request(v0 + own * KT::kRowBytes, vp, vst, t * KT::kRows + own, last, chunks, 0, ln);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      step(t, k0, v0);
    }
  } else {
    auto request = [&](int t, char* k, char* v) {
      KT::request(k, kp, kst, t * KT::kRows, last, chunks, wave, lane);
      KT::request(v, vp, vst, t * KT::kRows, last, chunks, wave, lane);
    };
    auto arrived = [] {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    };
    if (t0 < t1) request(t0, k0, v0);
    for (int t = t0; t < t1; t += 2) {
      arrived();
      if (t + 1 < t1) request(t + 1, k1, v1);
      step(t, k0, v0);
      if (t + 1 < t1) {
        arrived();
        if (t + 2 < t1) request(t + 2, k0, v0);
        step(t + 1, k1, v1);
      }
    }
  }
}

// --------------------------------------------------------------- forward --

// Per 32 rows and 64 keys: 32 matrix instructions of 32 cycles, about 170
// vector instructions (exponentials most of all), 32 KiB read from LDS.  2 x
// 4096 tokens, 32/8 heads of 128, causal, bf16: 310 us, 0.89 PFLOP/s; 2048
// queries behind 14336 keys 510 us, 1.0 PFLOP/s (the library's 8192^3 product
// reaches 1.17).  There matrix, vector and LDS units are busy 48, 44 and 37% of
// the cycles, at a clock that the load holds to 1.8 GHz: two waves a SIMD
// overlap them in part.  One token over 32768 keys (8 key heads): 27 us, its
// 134 MB at 5.0 TB/s, and 4 us for the join of 64 parts.
template <typename T, int DP, int DC, int KS, int NBUF>
__device__ __forceinline__ void attention_fwd(const lm_attn_params& P, char* k0, char* k1, char* v0, char* v1,
                                              float* ml) {
  using RW = Rows<KS>;
  using KT = Tile<T, DP, RW::kKeys>;
  RW R;
  if (!R.init(P)) return;
  const int lane = R.lane, h = R.h;
  const int chunks = P.dim * T::kBytes / 16;
  const char* kp = (const char*)P.k + ((int64_t)R.b * P.sk.b + (int64_t)R.kvh * P.sk.h) * T::kBytes;
  const char* vp = (const char*)P.v + ((int64_t)R.b * P.sv.b + (int64_t)R.kvh * P.sv.h) * T::kBytes;

  typename T::Frag qf[DC / 16];
  load_rows<T, DC>(qf, (const char*)P.q + row_offset(P.sq, R.b, R.head, R.query) * T::kBytes, P.dim, h, R.live);
  f32x16 acc[DC / 32];
#pragma unroll
  for (int i = 0; i < DC / 32; ++i) acc[i] = zero16();
  float m = kNegInf, l = 0.f;  // reference maximum (of scores times log2 e) and this lane's part of the sum
  const int row_at = KT::row_at(lane), col_at = KT::col_at(lane);

  over_keys<KT, NBUF>(
      kp, P.sk.t * T::kBytes, vp, P.sv.t * T::kBytes, R.t0, R.t1, R.S.kv_len - 1, chunks, R.wave, lane, R.mine.most, k0,
      k1, v0, v1,
      [&](int t, const char* kc, const char* vc) {
        constexpr int NB = RW::kBlocks;
        const int first = KS == 1 ? 0 : 32 * NB * R.part;  // this wave's keys of the tile
        const int key0 = t * RW::kKeys + first;
        if (key0 >= R.mine.most) return;
        attend<T, KT, DC, NB>(kc, vc, first, key0, R.mine.all, R.lim, qf, acc, m, l, P.scale_log2, row_at, col_at, lane, h);
      });

  l += other_half(l);
  if constexpr (KS > 1) {
    // one part after another to part 0, which rescales both to their common maximum
    join_waves<DC, KS>(reinterpret_cast<float*>((R.wave / KS) == 0 ? k0 : v0), ml + (R.wave / KS) * 128, R.part, acc, m, l,
                       lane);
    if (R.part != 0) return;
  }
  if constexpr (KS == 4) {
    if (P.splits > 1) {  // this part's sums as they stand, for the join
      if (!R.exists) return;
      const int64_t at = R.index(P) * P.splits + R.split;
      if (l != 0.f) store_rows<F32, DC>(reinterpret_cast<char*>(P.part + at * P.dim), acc, 1.f, P.dim, h);
      if (h == 0) {
        P.part_ml[at * 2] = m;
        P.part_ml[at * 2 + 1] = l;
      }
      return;
    }
  }
  if (R.exists) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
    store_rows<T, DC>((char*)P.o + row_offset(P.so, R.b, R.head, R.query) * T::kBytes, acc, inv, P.dim, h);
    if (P.lse != nullptr && h == 0) P.lse[R.stat(P)] = l == 0.f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

// Joins the parts of a row (64 parts of 32 rows: 4.0 us, 6.3 with the parts'
// weights found on the way): a workgroup per row, 32 lanes over its columns (four
// each), eight parts at a time.  All of a row's maxima and sums are requested
// together with the first parts, so that the join is one round trip to memory
// for up to 64 parts.  weights: one float per part.
template <typename T>
__device__ __forceinline__ void attention_join(const lm_attn_params& P, float* red, float* weights) {
  const int group = P.heads / P.kv_heads, rows = P.q_len * group;
  const int64_t at = blockIdx.x;
  const int row = (int)(at % rows), query = row / group;
  const int kvh = (int)(at / rows % P.kv_heads), b = (int)(at / rows / P.kv_heads);
  const int head = kvh * group + (row - query * group);
  const int lane = threadIdx.x & 63;
  const float* ml = P.part_ml + at * P.splits * 2;
  const int d = 4 * (threadIdx.x & 31), part = threadIdx.x >> 5;
  const float* rowp = P.part + at * P.splits * P.dim + (d < P.dim ? d : 0);
  constexpr int U = 8;
  f32x4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s = part + 8 * u < P.splits ? part + 8 * u : 0;
    v[u] = *reinterpret_cast<const f32x4*>(rowp + (int64_t)s * P.dim);
  }
  // every wave: the common maximum and the sum; wave 0: the parts' weights
  float ms[LM_ATTN_MAX_SPLITS / 64], ls[LM_ATTN_MAX_SPLITS / 64], m = kNegInf, l = 0.f;
#pragma unroll
  for (int i = 0; i < LM_ATTN_MAX_SPLITS / 64; ++i) {
    const int s = i * 64 + lane;
    ms[i] = s < P.splits ? ml[2 * s] : kNegInf;
    ls[i] = s < P.splits ? ml[2 * s + 1] : 0.f;
    m = fmaxf(m, ms[i]);
  }
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
#pragma unroll
  for (int i = 0; i < LM_ATTN_MAX_SPLITS / 64; ++i) {
    const float w = ls[i] == 0.f ? 0.f : exp2_fast(ms[i] - m);  // 0: saw no key, nothing was written
    l = __builtin_fmaf(w, ls[i], l);
    if (threadIdx.x < 64 && i * 64 + lane < P.splits) weights[i * 64 + lane] = w;
  }
  for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
  __syncthreads();
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = part; s0 < P.splits; s0 += 8 * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = s0 + 8 * u < P.splits ? weights[s0 + 8 * u] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = w != 0.f ? __builtin_fmaf(v[u][j], w, sum[j]) : sum[j];
    }
    if (s0 + 8 * U < P.splits) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + 8 * (U + u) < P.splits ? s0 + 8 * (U + u) : 0;
        v[u] = *reinterpret_cast<const f32x4*>(rowp + (int64_t)s * P.dim);
      }
    }
  }
  *reinterpret_cast<f32x4*>(red + threadIdx.x * 4) = sum;
  __syncthreads();
  if (threadIdx.x < 32 && d < P.dim) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < 8; ++p) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(red + (p * 32 + threadIdx.x) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += x[j];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
    store4<T>((char*)P.o + (row_offset(P.so, b, head, query) + d) * T::kBytes, o[0] * inv, o[1] * inv, o[2] * inv,
              o[3] * inv);
    if (P.lse != nullptr && threadIdx.x == 0)
      P.lse[((int64_t)b * P.heads + head) * P.q_len + query] =
          l == 0.f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

// -------------------------------------------------------- query gradients --

// As the forward, with 48 matrix instructions per 32 rows and 64 keys: 412 us
// at the forward's first shape, 1.0 PFLOP/s of what it executes.
template <typename T, int DP, int DC, int KS, int NBUF>
__device__ __forceinline__ void attention_bwd_dq(const lm_attn_params& P, char* k0, char* k1, char* v0, char* v1) {
  using RW = Rows<KS>;
  using KT = Tile<T, DP, RW::kKeys>;
  RW R;
  if (!R.init(P)) return;
  const int lane = R.lane, h = R.h;
  const int chunks = P.dim * T::kBytes / 16;
  const char* kp = (const char*)P.k + ((int64_t)R.b * P.sk.b + (int64_t)R.kvh * P.sk.h) * T::kBytes;
  const char* vp = (const char*)P.v + ((int64_t)R.b * P.sv.b + (int64_t)R.kvh * P.sv.h) * T::kBytes;

  typename T::Frag qf[DC / 16], gf[DC / 16];
  load_rows<T, DC>(qf, (const char*)P.q + row_offset(P.sq, R.b, R.head, R.query) * T::kBytes, P.dim, h, R.live);
  load_rows<T, DC>(gf, (const char*)P.grad_out + row_offset(P.sdo, R.b, R.head, R.query) * T::kBytes, P.dim, h, R.live);
  float delta = 0.f, lse2 = 0.f;
  {
    typename T::Frag of[DC / 16];
    load_rows<T, DC>(of, (const char*)P.out + row_offset(P.sout, R.b, R.head, R.query) * T::kBytes, P.dim, h, R.live);
#pragma unroll
    for (int s = 0; s < DC / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = __builtin_fmaf(T::get(gf[s], j), T::get(of[s], j), delta);
    delta += other_half(delta);
    if (R.live) lse2 = P.lse[R.stat(P)] * kLog2e;
  }
  const int row_at = KT::row_at(lane), col_at = KT::col_at(lane);
  // One 32-key block of a tile: the probabilities in s, do v^T in dp, for the keys from `first` of the tile.
  auto recompute = [&](const char* kc, const char* vc, int first, int key0, f32x16& s, f32x16& dp) {
    s = zero16();
    dp = zero16();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int st = 0; st < DC / 16; ++st) {
      s = T::mma(KT::row_frag(kc, first, st, row_at), qf[st], s);
      dp = T::mma(KT::row_frag(vc, first, st, row_at), gf[st], dp);
    }
    if constexpr (T::kBytes == 2) interleave<4, DC / 8, 1, 0, 0>();
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = exp2_fast(__builtin_fmaf(s[i], P.scale_log2, -lse2));
    if (key0 + 32 > R.mine.all) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool seen = key0 + 8 * (i >> 2) + 4 * h + (i & 3) < R.lim;
        s[i] = seen ? s[i] : 0.f;
        dp[i] = seen ? dp[i] : 0.f;
      }
    }
  };
  constexpr int NB = RW::kBlocks;
  const int mine = KS == 1 ? 0 : 32 * NB * R.part;  // this wave's keys of a tile
  // sum_d do o = sum_j p dp.  The first is one product a row, but the output it
  // reads was rounded to bf16, the only form the forward stores (an fp32 copy
  // would be two thirds of its writes); where a row sees few keys that rounding is as
  // large as any other in dq (an output of few values is as large as they
  // are).  Tiles of such rows are walked once more for the second: 1% of the
  // pairs of a sequence of 4096, and dq and dk keep the error of their own
  // roundings (2.4e-3 against 2.6e-3 of the norm at 777 tokens).
  if constexpr (T::kBytes == 2) {
    if (R.t1 * RW::kKeys <= kExactKeys && R.t1 > 0) {
      float d = 0.f;
      over_keys<KT, NBUF>(kp, P.sk.t * T::kBytes, vp, P.sv.t * T::kBytes, 0, R.t1, R.S.kv_len - 1, chunks, R.wave, lane,
                          R.mine.most, k0, k1, v0, v1, [&](int t, const char* kc, const char* vc) {
#pragma unroll
                            for (int kb = 0; kb < NB; ++kb) {
                              const int key0 = t * RW::kKeys + mine + 32 * kb;
                              if (key0 >= R.mine.most) continue;
                              f32x16 s, dp;
                              recompute(kc, vc, mine + 32 * kb, key0, s, dp);
#pragma unroll
                              for (int i = 0; i < 16; ++i) d = __builtin_fmaf(s[i], dp[i], d);
                            }
                          });
      delta = d + other_half(d);
      __syncthreads();  // the tiles' last readers are done
      if constexpr (KS > 1) {
        float* x = reinterpret_cast<float*>(k0);
        x[R.wave * 64 + lane] = delta;
        __syncthreads();
        delta = 0.f;
#pragma unroll
        for (int o = 0; o < KS; ++o) delta += x[(R.wave - R.part + o) * 64 + lane];
        __syncthreads();
      }
    }
  }
  if (R.live && P.grad_lse != nullptr) delta -= P.grad_lse[R.stat(P)];
  if (R.exists && h == 0 && R.part == 0) P.delta[R.stat(P)] = delta;
  f32x16 acc[DC / 32];
#pragma unroll
  for (int i = 0; i < DC / 32; ++i) acc[i] = zero16();
  over_keys<KT, NBUF>(kp, P.sk.t * T::kBytes, vp, P.sv.t * T::kBytes, 0, R.t1, R.S.kv_len - 1, chunks, R.wave, lane,
                      R.mine.most, k0, k1, v0, v1, [&](int t, const char* kc, const char* vc) {
#pragma unroll
                        for (int kb = 0; kb < NB; ++kb) {
                          const int key0 = t * RW::kKeys + mine + 32 * kb;
                          if (key0 >= R.mine.most) continue;
                          f32x16 s, dp;
                          recompute(kc, vc, mine + 32 * kb, key0, s, dp);
#pragma unroll
                          for (int i = 0; i < 16; ++i) s[i] *= dp[i] - delta;
#pragma unroll
                          for (int st = 0; st < 2; ++st) {
                            const typename T::Frag ds = T::from_acc(s, st);
#pragma unroll
                            for (int dt = 0; dt < DC / 32; ++dt)
                              acc[dt] = T::mma(KT::col_frag(kc, mine + 32 * kb + 16 * st, dt, col_at, lane), ds, acc[dt]);
                          }
                          if constexpr (T::kBytes == 2) interleave<8, DC / 16, 2, 0, 0>();
                        }
                      });

  if constexpr (KS > 1) {
    float* x = reinterpret_cast<float*>((R.wave / KS) == 0 ? k0 : v0);
#pragma unroll
    for (int o = 1; o < KS; ++o) {
      __syncthreads();
      if (R.part == o) put<DC>(x, acc, lane);
      __syncthreads();
      if (R.part == 0) add<DC>(x, acc, lane, 1.f, 1.f);
    }
    if (R.part != 0) return;
  }
  if (R.exists)
    store_rows<T, DC>((char*)P.dq + row_offset(P.sdq, R.b, R.head, R.query) * T::kBytes, acc, P.scale, P.dim, h);
}

// ------------------------------------------------ key and value gradients --

// A wave owns 32 keys; KS waves share them and split each tile of 32 KS rows:
// queries of one head, the heads of the group one after another.  The keys'
// and values' operands and both gradients stay in registers (192 of 256 at
// head size 128, where the offsets into LDS are formed anew for each tile), so
// a tile is read twice, once as rows and once as columns.  620 us at the
// forward's first shape, 0.88 PFLOP/s; 8 x 4096 tokens, 24/8 heads 1577 us, 1.05.
template <typename T, int DP, int DC, int KS, int NBUF>
__device__ __forceinline__ void attention_bwd_dkv(const lm_attn_params& P, char* q0, char* q1, char* g0, char* g1,
                                                  float* st0, float* st1) {
  constexpr int R = 32 * KS;
  using QT = Tile<T, DP, R>;
  const Item it = work_item(P);
  if (it.rank < 0) return;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave % KS;
  const int kvh = it.head % P.kv_heads, b = it.head / P.kv_heads;
  const int group = P.heads / P.kv_heads;
  const Seq S = sequence(P, b, 1);
  const int wg0 = it.rank * (32 * LM_ATTN_WAVES / KS);  // causal: the first keys are seen by the most queries
  const int w0 = wg0 + wave / KS * 32;
  const int key = w0 + (lane & 31);
  const bool live = key < S.kv_len;

  typename T::Frag kf[DC / 16], vf[DC / 16];
  load_rows<T, DC>(kf, (const char*)P.k + row_offset(P.sk, b, kvh, key) * T::kBytes, P.dim, h, live);
  load_rows<T, DC>(vf, (const char*)P.v + row_offset(P.sv, b, kvh, key) * T::kBytes, P.dim, h, live);
  f32x16 dk[DC / 32], dv[DC / 32];
#pragma unroll
  for (int i = 0; i < DC / 32; ++i) {
    dk[i] = zero16();
    dv[i] = zero16();
  }
  // the first query that sees a key, of the workgroup's keys, the wave's, and
  // this lane's; from w_full on queries see all the wave's
  auto first_query = [&](int k) {
    const int64_t r = P.causal ? (int64_t)k - S.start : 0;
    return (int)(r < S.lo ? S.lo : r > S.hi ? S.hi : r);
  };
  const int base = first_query(wg0);
  const int w_first = first_query(w0);
  const int w_full = w0 + 32 > S.kv_len ? S.hi : first_query(w0 + 31);
  const int k_first = live ? first_query(key) : S.hi;
  const int per = wg0 < S.kv_len ? (S.hi - base + R - 1) / R : 0;  // tiles of a head
  const int tiles = per * group;

  const int chunks = P.dim * T::kBytes / 16;
  const int64_t qst = P.sq.t * T::kBytes, qsh = P.sq.h * T::kBytes, gst = P.sdo.t * T::kBytes, gsh = P.sdo.h * T::kBytes;
  const char* qp = (const char*)P.q + row_offset(P.sq, b, kvh * group, 0) * T::kBytes;
  const char* gp = (const char*)P.grad_out + row_offset(P.sdo, b, kvh * group, 0) * T::kBytes;
  int64_t stat = ((int64_t)b * P.heads + kvh * group) * P.q_len;
  int next = 0;  // the tile of its head to request
  auto request = [&](char* qn, char* gn, float* sn) {
    int ln = lane;  // opaque: the lane's offsets are formed anew for each tile, registers being short
    asm volatile("" : "+v"(ln));
    if constexpr (NBUF == 1) {  // this wave's own 32 rows, where there are any
      using MT = typename QT::Mine;
      const int row0 = base + next * R + 32 * wave;
      if (row0 < S.hi) {
        MT::request(qn + 32 * wave * QT::kRowBytes, qp, qst, row0, S.hi - 1, chunks, 0, ln);
        MT::request(gn + 32 * wave * QT::kRowBytes, gp, gst, row0, S.hi - 1, chunks, 0, ln);
      }
    } else {
      QT::request(qn, qp, qst, base + next * R, S.hi - 1, chunks, wave, ln);
      QT::request(gn, gp, gst, base + next * R, S.hi - 1, chunks, wave, ln);
    }
    if (wave < KS) {  // the queries' lse (lanes 0 .. 31) and delta, 32 a wave
      int r = base + next * R + wave * 32 + (ln & 31);
      r = r < S.hi ? r : S.hi - 1;
      const float* src = ((ln >> 5) ? P.delta : P.lse) + stat + r;
      __builtin_amdgcn_global_load_lds((const LM_GLOBAL void*)src, (LM_LDS void*)(sn + wave * 64), 4, 0, 0);
    }
    if (++next == per) {
      next = 0;
      qp += qsh;
      gp += gsh;
      stat += P.q_len;
    }
  };
  int now = 0;  // the tile of its head to work on
  int row_at = QT::row_at(lane), col_at = QT::col_at(lane);
  auto step = [&](const char* qc, const char* gc, const float* sc) {
    const int mine = KS == 1 ? 0 : 32 * part;  // this wave's rows of the tile
    const int row0 = base + now * R + mine;
    now = now + 1 == per ? 0 : now + 1;
    if (row0 + 32 <= w_first || row0 >= S.hi || w0 >= S.kv_len) return;
    // opaque here, so that the offsets made from these are formed anew (one
    // instruction each) instead of held in registers
    asm volatile("" : "+v"(row_at), "+v"(col_at));
    f32x16 s = zero16(), dp = zero16();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int st = 0; st < DC / 16; ++st) {
      s = T::mma(QT::row_frag(qc, mine, st, row_at), kf[st], s);
      dp = T::mma(QT::row_frag(gc, mine, st, row_at), vf[st], dp);
    }
    if constexpr (T::kBytes == 2) interleave<4, DC / 8, 1, 0, 0>();
    __builtin_amdgcn_s_setprio(0);
    const float* stats = sc + (KS == 1 ? 0 : 64 * part);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 lse = *reinterpret_cast<const f32x4*>(stats + 8 * a + 4 * h);
      const f32x4 dl = *reinterpret_cast<const f32x4*>(stats + 32 + 8 * a + 4 * h);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[4 * a + c] = exp2_fast(__builtin_fmaf(s[4 * a + c], P.scale_log2, -lse[c] * kLog2e));
        dp[4 * a + c] -= dl[c];
      }
    }
    if (row0 < w_full || row0 + 32 > S.hi) {
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
      for (int dt = 0; dt < DC / 32; ++dt) {
        dv[dt] = T::mma(QT::col_frag(gc, mine + 16 * st, dt, col_at, lane), p, dv[dt]);
        dk[dt] = T::mma(QT::col_frag(qc, mine + 16 * st, dt, col_at, lane), ds, dk[dt]);
      }
    }
    if constexpr (T::kBytes == 2) interleave<4, DC / 8, 2, 0, 0>();
  };
  auto arrived = [] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  if constexpr (NBUF == 1) {  // four waves share their keys: each loads the rows it reads itself
    static_assert(KS == LM_ATTN_WAVES, "a tile has 32 rows for each wave");
    for (int t = 0; t < tiles; ++t) {
      request(q0, g0, st0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      step(q0, g0, st0);
    }
  } else {
    if (tiles > 0) request(q0, g0, st0);
    for (int t = 0; t < tiles; t += 2) {
      arrived();
      if (t + 1 < tiles) request(q1, g1, st1);
      step(q0, g0, st0);
      if (t + 1 < tiles) {
        arrived();
        if (t + 2 < tiles) request(q0, g0, st0);
        step(q1, g1, st1);
      }
    }
  }
  if constexpr (KS > 1) {
    float* xk = reinterpret_cast<float*>((wave / KS) == 0 ? q0 : q1);
    float* xv = reinterpret_cast<float*>((wave / KS) == 0 ? g0 : g1);
#pragma unroll
    for (int o = 1; o < KS; ++o) {
      __syncthreads();
      if (part == o) {
        put<DC>(xk, dk, lane);
        put<DC>(xv, dv, lane);
      }
      __syncthreads();
      if (part == 0) {
        add<DC>(xk, dk, lane, 1.f, 1.f);
        add<DC>(xv, dv, lane, 1.f, 1.f);
      }
    }
    if (part != 0) return;
  }
  if (key < P.kv_len) {
    store_rows<T, DC>((char*)P.dk + row_offset(P.sdk, b, kvh, key) * T::kBytes, dk, P.scale, P.dim, h);
    store_rows<T, DC>((char*)P.dv + row_offset(P.sdv, b, kvh, key) * T::kBytes, dv, 1.f, P.dim, h);
  }
}

}  // namespace

// DP: elements of a tile's row in LDS; DC: columns worked on, the head size
// rounded up to 32; KS: waves that share rows (or keys); NBUF: LDS buffers of a tile; WPE: waves
// per SIMD the registers are held to.
#define LM_ATTN_KERNEL(KIND, NAME, WPE) \
  extern "C" __global__ void __launch_bounds__(64 * LM_ATTN_WAVES) __attribute__((amdgpu_waves_per_eu(WPE))) \
      attnres_attention_##KIND##_##NAME(lm_attn_params P)
#define LM_ATTN(NAME, T, DP, DC, KS, NBUF, FWD_WPE, DQ_WPE, DKV_WPE)                                     \
  LM_ATTN_KERNEL(fwd, NAME, FWD_WPE) {                                                               \
    constexpr int kTile = Tile<T, DP, Rows<KS>::kKeys>::kBytes;                                      \
    __shared__ __align__(16) char k0[kTile];                                                         \
    __shared__ __align__(16) char v0[kTile];                                                         \
    __shared__ __align__(16) char k1[NBUF == 2 ? kTile : 16];                                        \
    __shared__ __align__(16) char v1[NBUF == 2 ? kTile : 16];                                        \
    __shared__ float ml[KS > 1 ? LM_ATTN_WAVES / KS * 128 : 1];                                      \
    attention_fwd<T, DP, DC, KS, NBUF>(P, k0, k1, v0, v1, ml);                                           \
  }                                                                                                  \
  LM_ATTN_KERNEL(dq, NAME, DQ_WPE) {                                                                 \
    constexpr int kTile = Tile<T, DP, Rows<KS>::kKeys>::kBytes;                                      \
    __shared__ __align__(16) char k0[kTile];                                                         \
    __shared__ __align__(16) char v0[kTile];                                                         \
    __shared__ __align__(16) char k1[NBUF == 2 ? kTile : 16];                                        \
    __shared__ __align__(16) char v1[NBUF == 2 ? kTile : 16];                                        \
    attention_bwd_dq<T, DP, DC, KS, NBUF>(P, k0, k1, v0, v1);                                            \
  }                                                                                                  \
  LM_ATTN_KERNEL(dkv, NAME, DKV_WPE) {                                                               \
    constexpr int kTile = Tile<T, DP, 32 * KS>::kBytes;                                              \
    __shared__ __align__(16) char q0[kTile];                                                         \
    __shared__ __align__(16) char g0[kTile];                                                         \
    __shared__ __align__(16) char q1[NBUF == 2 ? kTile : 16];                                        \
    __shared__ __align__(16) char g1[NBUF == 2 ? kTile : 16];                                        \
    __shared__ __align__(16) float st0[64 * KS];                                                     \
    __shared__ __align__(16) float st1[NBUF == 2 ? 64 * KS : 4];                                     \
    attention_bwd_dkv<T, DP, DC, KS, NBUF>(P, q0, q1, g0, g1, st0, st1);                                 \
  }

#define LM_ATTN_JOIN(NAME, T)                                                                       \
  extern "C" __global__ void __launch_bounds__(256) attnres_attention_join_##NAME(lm_attn_params P) { \
    __shared__ __align__(16) float red[1024];                                                       \
    __shared__ float weights[LM_ATTN_MAX_SPLITS];                                                   \
    attention_join<T>(P, red, weights);                                                             \
  }

#if LM_PART == 13
LM_ATTN_JOIN(bf16, Bf16)
#define LM_ATTN_BF16(DP, DC)                              \
  LM_ATTN(bf16_d##DC##_s1, Bf16, DP, DC, 1, 2, 2, 2, 2)   \
  LM_ATTN(bf16_d##DC##_s2, Bf16, DP, DC, 2, 2, 2, 2, 2)   \
  LM_ATTN(bf16_d##DC##_s4, Bf16, DP, DC, 4, 1, 2, 2, 2)
LM_ATTN_BF16(64, 32)
LM_ATTN_BF16(64, 64)
LM_ATTN_BF16(128, 96)
LM_ATTN_BF16(128, 128)
#endif
#if LM_PART == 14
LM_ATTN_JOIN(f32, F32)
#define LM_ATTN_F32(DP, DC)                              \
  LM_ATTN(f32_d##DC##_s1, F32, DP, DC, 1, 2, 1, 1, 1)    \
  LM_ATTN(f32_d##DC##_s2, F32, DP, DC, 2, 2, 1, 1, 1)    \
  LM_ATTN(f32_d##DC##_s4, F32, DP, DC, 4, 1, 1, 1, 1)
LM_ATTN_F32(64, 32)
LM_ATTN_F32(64, 64)
LM_ATTN_F32(128, 96)
LM_ATTN_F32(128, 128)
#endif
