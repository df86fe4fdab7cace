// Attention of new tokens over a paged cache for gfx950 (CDNA4): chunks of
// prompts, drafted tokens and single tokens of many sequences in one call.
//
//   s_j = scale q . k_j over the keys j up to the token's own position
//   o = sum_j softmax_j(s) v_j
//
// Products, tiles and the softmax are those of attention_tiles.h.  The rows of a key head's
// query group are taken together, query by query: row r of a sequence is head
// r % group of its new token r / group.
//
// How the work is dealt out.  The host knows how many tokens and sequences a
// call has, the device how long they are; so the grid is a bound, and every
// workgroup finds its own work in the lengths: a tile of a sequence's rows and a
// part of its keys.  Sequences of up to 32 rows (single tokens, drafts) are
// narrow tiles: four waves share the 32 rows and each works on 32 keys of a tile
// of 128.  The rows of longer ones are taken 128 at a time, each wave 32 of
// them over all keys, where the call has rows enough to fill the card so
// (`wide`), else 32 at a time as well.  Tiles of more keys than their
// share (all blocks over `target` workgroups) are split, and
// paged_join adds the parts in order, so that results repeat bit for bit.
//
// Keys are found through the table: a wave-wide load covers at most 8 rows,
// which lie in one page, so the page's address is uniform and a lane's
// offset within it the same for every page.  A wave reads the
// table entries of a tile with one load, a tile ahead of its keys.  An entry outside
// the cache is read as page 0 and makes the rows that are worked on with it NaN.

#include "attention_tiles.h"

namespace {

constexpr int kThreads = LM_PAGED_THREADS;

// ---------------------------------------------------------------- schedule --

// One sequence's share of the call: its tokens, keys, tiles of rows and parts of their keys.
struct Share {
  int first, count;  // new tokens
  int kv_len;
  int rows, tiles, splits;
  bool narrow;
  int per;  // key tiles of a part
};

// The sequences' sizes are taken into what the call has, so that no length
// leads out of its tensors.  Behind the last sequence (s == seqs): the tokens that
// belong to none, as a sequence without keys.
__device__ __forceinline__ Share share_of(const lm_paged_params& P, int s, int group) {
  Share a;
  int64_t lo, hi;
  if (P.q_starts == nullptr) {
    lo = s;
    hi = s < P.seqs ? s + 1 : P.tokens;
  } else {
    lo = s == 0 ? 0 : index_at(P.q_starts, s, P.starts64);
    hi = s < P.seqs ? index_at(P.q_starts, s + 1, P.starts64) : P.tokens;
  }
  lo = lo < 0 ? 0 : lo > P.tokens ? P.tokens : lo;
  hi = hi < lo ? lo : hi > P.tokens ? P.tokens : hi;
  int64_t n = s < P.seqs ? index_at(P.kv_lens, s, P.lens64) : 0;
  n = n < 0 ? 0 : n > P.capacity ? P.capacity : n;
  a.first = (int)lo;
  a.count = (int)(hi - lo);
  a.kv_len = (int)n;
  a.rows = a.count * group;
  a.narrow = !P.wide || a.rows <= 32;
  a.tiles = a.narrow ? (a.rows + 31) >> 5 : (a.rows + 127) >> 7;
  a.splits = a.per = 0;
  return a;
}
// A tile's work: blocks of 32 keys that a wave works on.
__device__ __forceinline__ int blocks_of(const Share& a) {
  return a.narrow ? (a.kv_len + 127) >> 7 : ((a.kv_len + 63) >> 6) * 2;
}
__device__ __forceinline__ void split(Share& a, int most) {
  a.per = a.narrow ? most : (most + 1) >> 1;
  const int n = a.narrow ? (a.kv_len + 127) >> 7 : (a.kv_len + 63) >> 6;
  a.splits = n <= a.per ? 1 : (n + a.per - 1) / a.per;
}

struct Shared {
  float sum[LM_ATTN_WAVES];
  int scan[LM_ATTN_WAVES][2];
  int upto[kThreads][2];
};

// Sum of a float over the workgroup (all threads get it); whole numbers under 2^24 or nearly so.
__device__ __forceinline__ float sum_all(float v, Shared& S) {
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) S.sum[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < LM_ATTN_WAVES; ++i) t += S.sum[i];
  return t;
}

// Inclusive sums of two numbers over the workgroup's threads into S.upto.
__device__ __forceinline__ void scan_all(int a, int b, Shared& S) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int x = __shfl_up(a, m), y = __shfl_up(b, m);
    a += lane >= m ? x : 0;
    b += lane >= m ? y : 0;
  }
  if (lane == 63) {
    S.scan[wave][0] = a;
    S.scan[wave][1] = b;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < LM_ATTN_WAVES - 1; ++i) {
    a += i < wave ? S.scan[i][0] : 0;
    b += i < wave ? S.scan[i][1] : 0;
  }
  S.upto[threadIdx.x][0] = a;
  S.upto[threadIdx.x][1] = b;
  __syncthreads();
}

// The blocks of 32 keys that a part may have: an equal share for `target` workgroups.
// (A float's rounding moves the share by a part in 2^24; every workgroup of
// both launches finds the same.)
__device__ __forceinline__ int most_blocks(const lm_paged_params& P, int group, Shared& S) {
  float work = 0.f;
  for (int s = threadIdx.x; s < P.seqs; s += kThreads) {
    const Share a = share_of(P, s, group);
    work += (float)a.tiles * (float)blocks_of(a);
  }
  work = sum_all(work, S) * (float)P.kv_heads / (float)P.target;
  const int n = work < 1e9f ? (int)__builtin_ceilf(work) : 1 << 30;
  return n < P.least ? P.least : n;
}

// A workgroup's work.
struct Job {
  Share a;
  int seq, tile, part;
  int slot;  // where a split tile's parts begin
};

// Finds part `w` of the call's (all sequences' parts one after another).
__device__ __forceinline__ bool find_job(const lm_paged_params& P, int w, int group, Shared& S, Job& J) {
  const int most = most_blocks(P, group, S);
  int parts = 0, slots = 0;  // before this stretch of sequences
  for (int base = 0; base <= P.seqs; base += kThreads) {
    const int s = base + (int)threadIdx.x;
    int mine = 0, held = 0;
    if (s <= P.seqs) {
      Share a = share_of(P, s, group);
      split(a, most);
      mine = a.tiles * a.splits;
      held = a.splits > 1 ? mine : 0;
    }
    scan_all(mine, held, S);
    const int total = S.upto[kThreads - 1][0];
    if (w - parts < total) {
      int lo = 0;  // the first sequence whose parts end behind w
#pragma unroll
      for (int step = kThreads / 2; step > 0; step >>= 1)
        if (S.upto[lo + step - 1][0] <= w - parts) lo += step;
      const int before = lo > 0 ? S.upto[lo - 1][0] : 0;
      J.seq = __builtin_amdgcn_readfirstlane(base + lo);
      J.a = share_of(P, J.seq, group);
      split(J.a, most);
      const int i = __builtin_amdgcn_readfirstlane(w - parts - before);
      const int rank = i / J.a.splits;
      J.part = i - rank * J.a.splits;
      J.tile = J.a.tiles - 1 - rank;  // the longest first
      J.slot = __builtin_amdgcn_readfirstlane(slots + (lo > 0 ? S.upto[lo - 1][1] : 0)) + rank * J.a.splits;
      return true;
    }
    parts += total;
    slots += S.upto[kThreads - 1][1];
    __syncthreads();
  }
  return false;
}

// ------------------------------------------------------------------- pages --

// A sequence's pages, as one wave reads them.
struct Pages {
  const int32_t* table;
  int shift, pages, last;  // last: the last key that exists
  bool bad;                // an entry outside the cache was met

  // The pages of 64 rows from `row`: lane i holds that of row + i (of the last row behind it).
  __device__ __forceinline__ int of(int row, int lane) const {
    const int r = row + lane;
    return table[(r < last ? r : last) >> shift];
  }
  // Entries as they may be read.
  __device__ __forceinline__ int checked(int page) {
    const bool out = (uint32_t)page >= (uint32_t)pages;
    bad = bad || __any(out);
    return out ? 0 : page;
  }
};

// Requests the R rows of tile KT from key `row0` (a multiple of 32) into `lds`, as
// KT::request does for contiguous keys.  `page`: Pages::of(row0).
template <typename KT>
__device__ __forceinline__ void request_paged(char* lds, const char* src, const lm_strides& st, int es, int row0, int last,
                                              int shift, int page, int chunks, int wave, int lane) {
  constexpr int kPerWave = 64 / KT::kChunks;  // rows of a wave's load
  static_assert(kPerWave <= LM_PAGED_MIN_PAGE, "in one page");
  constexpr int kWaves = KT::kRound / kPerWave;
  const int mask = (1 << shift) - 1;
  const int64_t page_bytes = st.b * es;
  const uint32_t row_bytes = (uint32_t)(st.t * es);
  const int mine = lane / KT::kChunks;
#pragma unroll
  for (int i = 0; i < KT::kRounds; ++i) {
    const int first = i * KT::kRound + wave * kPerWave;
    const int p = __builtin_amdgcn_readlane(page, first);
    const char* base = src + (int64_t)p * page_bytes;
    const int row = row0 + first;
    char* to = lds + (i * kWaves + wave) * 1024;
    const uint32_t chunk = KT::chunk_offset(i, wave, lane, chunks);
    if (row + kPerWave - 1 <= last) {
      KT::load_lds(to, base + (uint64_t)((uint32_t)(row & mask)) * row_bytes, (uint32_t)mine * row_bytes + chunk);
    } else {  // rows behind the last repeat it
      const int r = row + mine < last ? row + mine : last;
      KT::load_lds(to, base, (uint32_t)(r & mask) * row_bytes + chunk);
    }
  }
}

// ----------------------------------------------------------------- forward --

// KS 4: a narrow tile, KS 1: a wide one.
template <typename T, int DP, int DC, int KS>
__device__ __forceinline__ void paged_rows(const lm_paged_params& P, const Job& J, int kvh, int group, char* lds,
                                           float* ml, int* flag) {
  constexpr int kKeys = KS == 4 ? 128 : 64;  // keys of a tile
  constexpr int NB = kKeys / 32 / KS;        // 32-key blocks of a wave in it
  using KT = Tile<T, DP, kKeys>;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave % KS;
  const int g0 = J.tile * (32 * LM_ATTN_WAVES / KS), r0 = g0 + wave / KS * 32;
  const int start = J.a.kv_len - J.a.count;  // position of token 0
  const int row = r0 + (lane & 31), query = row / group;
  const int head = kvh * group + (row - query * group);
  const bool exists = row < J.a.rows;
  const int lim = J.a.kv_len == 0 ? 0 : start + query + 1;  // keys this row sees, if any
  // the keys that the wave's rows see: the most, and what all see (rows that are not there are not stored)
  auto sees = [&](int r) { return J.a.kv_len == 0 ? 0 : start + r / group + 1; };
  auto end = [&](int r) { return r < J.a.rows ? r : J.a.rows; };
  const int most = __builtin_amdgcn_readfirstlane(r0 < J.a.rows ? sees(end(r0 + 32) - 1) : 0);
  const int all = __builtin_amdgcn_readfirstlane(sees(r0));
  const int any = __builtin_amdgcn_readfirstlane(sees(end(g0 + 32 * LM_ATTN_WAVES / KS) - 1));
  const int tiles = any <= 0 ? 0 : (any + kKeys - 1) / kKeys;
  const int t0 = J.part * J.a.per, t1 = tiles < t0 + J.a.per ? tiles : t0 + J.a.per;

  typename T::Frag qf[DC / 16];
  load_rows<T, DC>(qf, (const char*)P.q + ((int64_t)(J.a.first + query) * P.q_t + (int64_t)head * P.q_h) * T::kBytes,
                   P.dim, h, exists);
  f32x16 acc[DC / 32];
#pragma unroll
  for (int i = 0; i < DC / 32; ++i) acc[i] = zero16();
  float m = kNegInf, l = 0.f;
  const int row_at = KT::row_at(lane), col_at = KT::col_at(lane);
  const int chunks = P.dim * T::kBytes / 16;
  const char* kp = (const char*)P.k + (int64_t)kvh * P.sk.h * T::kBytes;
  const char* vp = (const char*)P.v + (int64_t)kvh * P.sv.h * T::kBytes;
  Pages pg;
  pg.table = P.table + (int64_t)J.seq * P.table_ld;
  pg.shift = P.shift;
  pg.pages = P.pages;
  pg.last = J.a.kv_len - 1;
  pg.bad = false;

  if constexpr (KS == 4) {
    // each wave reads only its own 32 keys of a tile, so it loads them itself and waits for no other
    using MT = typename KT::Mine;
    const int own = 32 * wave;
    char* kc = lds;
    char* vc = lds + KT::kBytes;
    int page = t0 < t1 && t0 * kKeys + own < most ? pg.of(t0 * kKeys + own, lane) : 0;
    for (int t = t0; t < t1 && t * kKeys + own < most; ++t) {
      const int key0 = t * kKeys + own;
      int ln = lane;  // opaque: offsets formed anew for each tile instead of held in registers
      asm volatile("" : "+v"(ln));
      const int now = pg.checked(page);
      page = t + 1 < t1 ? pg.of(key0 + kKeys, ln) : 0;
      request_paged<MT>(kc + own * KT::kRowBytes, kp, P.sk, T::kBytes, key0, pg.last, pg.shift, now, chunks, 0, ln);
      request_paged<MT>(vc + own * KT::kRowBytes, vp, P.sv, T::kBytes, key0, pg.last, pg.shift, now, chunks, 0, ln);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      attend<T, KT, DC, NB>(kc, vc, own, key0, all, lim, qf, acc, m, l, P.scale_log2, row_at, col_at, lane, h);
    }
  } else {
    // the waves share the tiles: the next is requested before one is worked on, its pages read a tile before that
    char* kb[2] = {lds, lds + 2 * KT::kBytes};
    char* vb[2] = {lds + KT::kBytes, lds + 3 * KT::kBytes};
    int page = 0;
    auto request = [&](int t, char* k, char* v) {
      const int now = pg.checked(page);
      request_paged<KT>(k, kp, P.sk, T::kBytes, t * kKeys, pg.last, pg.shift, now, chunks, wave, lane);
      request_paged<KT>(v, vp, P.sv, T::kBytes, t * kKeys, pg.last, pg.shift, now, chunks, wave, lane);
      if (t + 1 < t1) page = pg.of((t + 1) * kKeys, lane);
    };
    auto arrived = [] {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    };
    auto step = [&](int t, const char* kc, const char* vc) {
      if (t * kKeys >= most) return;
      attend<T, KT, DC, NB>(kc, vc, 0, t * kKeys, all, lim, qf, acc, m, l, P.scale_log2, row_at, col_at, lane, h);
    };
    if (t0 < t1) {
      page = pg.of(t0 * kKeys, lane);
      request(t0, kb[0], vb[0]);
    }
    for (int t = t0; t < t1; t += 2) {
      arrived();
      if (t + 1 < t1) request(t + 1, kb[1], vb[1]);
      step(t, kb[0], vb[0]);
      if (t + 1 < t1) {
        arrived();
        if (t + 2 < t1) request(t + 2, kb[0], vb[0]);
        step(t + 1, kb[1], vb[1]);
      }
    }
  }
  // a page outside the cache that any wave met
  if (pg.bad && lane == 0) *flag = 1;
  l += other_half(l);
  if constexpr (KS == 4) {
    join_waves<DC, KS>(reinterpret_cast<float*>(lds), ml, part, acc, m, l, lane);
    if (part != 0) return;
  } else {
    __syncthreads();
  }
  if (*flag != 0) l = __builtin_nanf("");
  if (!exists) return;
  if (J.a.splits > 1) {
    if (J.slot + J.part >= P.slots) return;
    const int64_t at = ((int64_t)(J.slot + J.part) * P.kv_heads + kvh) * P.part_rows + (row - g0);
    if (l != 0.f) store_rows<F32, DC>(reinterpret_cast<char*>(P.part + at * P.dim), acc, 1.f, P.dim, h);
    if (h == 0) {
      P.part_ml[at * 2] = m;
      P.part_ml[at * 2 + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
  const int64_t token = J.a.first + query;
  store_rows<T, DC>((char*)P.o + (token * P.o_t + (int64_t)head * P.o_h) * T::kBytes, acc, inv, P.dim, h);
  if (P.lse != nullptr && h == 0)
    P.lse[token * P.heads + head] = l == 0.f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T, int DP, int DC, bool WIDE>
__device__ __forceinline__ void paged_attention(const lm_paged_params& P, char* lds, float* ml, int* flag, Shared& S) {
  // Workgroups go to the eight XCDs in turn, each with an L2 of its own: where the key heads
  // divide by eight, each XCD takes an eighth of them, so that the tiles of a sequence's rows find
  // a head's keys in one L2.
  int w = (int)blockIdx.x, kvh;
  if ((P.kv_heads & 7) == 0) {
    const int hx = P.kv_heads >> 3, x = w & 7;
    w >>= 3;
    const int p = w / hx;
    kvh = x * hx + (w - p * hx);
    w = p;
  } else {
    const int p = w / P.kv_heads;
    kvh = w - p * P.kv_heads;
    w = p;
  }
  const int group = P.heads / P.kv_heads;
  if (threadIdx.x == 0) *flag = 0;
  Job J;
  if (!find_job(P, w, group, S, J)) return;
  if (!WIDE || J.a.narrow)
    paged_rows<T, DP, DC, 4>(P, J, kvh, group, lds, ml, flag);
  else
    paged_rows<T, DP, DC, 1>(P, J, kvh, group, lds, ml, flag);
}

// -------------------------------------------------------------------- join --

// Joins the parts of the split tiles: eight lane groups of 32 (four columns a lane)
// take a row's parts in turn, or, where a row has fewer than eight, several
// rows.  A workgroup walks over the rows of the split sequences.
template <typename T>
__device__ __forceinline__ void paged_join(const lm_paged_params& P, Shared& S, f32x4* red) {
  const int group = P.heads / P.kv_heads;
  const int most = most_blocks(P, group, S);
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int d = 4 * lane;
  int items = 0, slots = 0;  // before this stretch of sequences
  auto side_by_side = [](int splits) { return splits <= 2 ? 2 : splits <= 4 ? 4 : 8; };  // parts at a time
  for (int base = 0; base < P.seqs; base += kThreads) {
    const int s = base + (int)threadIdx.x;
    int mine = 0, held = 0;
    if (s < P.seqs) {
      Share a = share_of(P, s, group);
      split(a, most);
      if (a.splits > 1) {
        const int each = 8 / side_by_side(a.splits);  // rows at a time
        mine = (a.rows + each - 1) / each * P.kv_heads;
        held = a.tiles * a.splits;
      }
    }
    scan_all(mine, held, S);
    const int total = S.upto[kThreads - 1][0];
    // this workgroup's items of the stretch: those of all, counted from the first stretch on, that fall to it
    int i = ((int)blockIdx.x - items % (int)gridDim.x + (int)gridDim.x) % (int)gridDim.x;
    for (; i < total; i += gridDim.x) {
      int lo = 0;
#pragma unroll
      for (int step = kThreads / 2; step > 0; step >>= 1)
        if (S.upto[lo + step - 1][0] <= i) lo += step;
      Share a = share_of(P, base + lo, group);
      split(a, most);
      const int j = i - (lo > 0 ? S.upto[lo - 1][0] : 0);
      const int first = slots + (lo > 0 ? S.upto[lo - 1][1] : 0);
      const int pp = side_by_side(a.splits), each = 8 / pp;
      const int kvh = j % P.kv_heads;
      const int row = j / P.kv_heads * each + g / pp, phase = g % pp;
      const int size = a.narrow ? 32 : 128, tile = row / size;
      const int slot = first + (a.tiles - 1 - tile) * a.splits;
      const bool live = row < a.rows && slot + a.splits <= P.slots;
      const int64_t step = (int64_t)P.kv_heads * P.part_rows;
      const int64_t at = live ? ((int64_t)slot * P.kv_heads + kvh) * P.part_rows + (row - tile * size) : 0;
      // the common maximum and the sum: 32 lanes over the parts
      float m = kNegInf, l = 0.f;
      if (live) {
        for (int p = lane; p < a.splits; p += 32) m = fmaxf(m, P.part_ml[(at + p * step) * 2]);
      }
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
      if (live) {
        for (int p = lane; p < a.splits; p += 32) {
          const float pm = P.part_ml[(at + p * step) * 2], pl = P.part_ml[(at + p * step) * 2 + 1];
          l += pm == kNegInf ? pl : pl * exp2_fast(pm - m);  // no keys: zero, or the NaN of a bad page
        }
      }
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) l += __shfl_xor(l, x);
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      if (live && d < P.dim) {
#pragma unroll 4
        for (int p = phase; p < a.splits; p += pp) {
          const float pm = P.part_ml[(at + p * step) * 2], pl = P.part_ml[(at + p * step) * 2 + 1];
          const f32x4 v = *reinterpret_cast<const f32x4*>(P.part + (at + p * step) * P.dim + d);
          const float w = exp2_fast(pm - m);
          if (pl != 0.f && pm != kNegInf) {  // a part without keys has written none
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = __builtin_fmaf(v[c], w, sum[c]);
          }
        }
      }
      red[threadIdx.x] = sum;
      __syncthreads();
      if (phase == 0 && live && d < P.dim) {
        for (int p = 1; p < pp; ++p) {
          const f32x4 o = red[threadIdx.x + 32 * p];
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[c] += o[c];
        }
        const int query = row / group, head = kvh * group + (row - query * group);
        const int64_t token = a.first + query;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store4<T>((char*)P.o + (token * P.o_t + (int64_t)head * P.o_h + d) * T::kBytes, sum[0] * inv, sum[1] * inv,
                  sum[2] * inv, sum[3] * inv);
        if (P.lse != nullptr && d == 0)
          P.lse[token * P.heads + head] = l == 0.f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
      }
      __syncthreads();
    }
    items += total;
    slots += S.upto[kThreads - 1][1];
    __syncthreads();
  }
}

}  // namespace

// DP: elements of a tile's row in LDS; DC: columns worked on, the head size rounded up to 32.
#define LM_PAGED_KERNEL(NAME, T, DP, DC, WIDE, WPE)                                                              \
  extern "C" __global__ void __launch_bounds__(LM_PAGED_THREADS) __attribute__((amdgpu_waves_per_eu(WPE)))      \
      attnres_paged_attention_##NAME(lm_paged_params P) {                                                        \
    __shared__ __align__(16) char lds[2 * Tile<T, DP, 128>::kBytes];                                             \
    __shared__ float ml[128];                                                                                    \
    __shared__ int flag;                                                                                         \
    __shared__ Shared S;                                                                                         \
    paged_attention<T, DP, DC, WIDE>(P, lds, ml, &flag, S);                                                      \
  }
#define LM_PAGED_JOIN(NAME, T)                                                                                   \
  extern "C" __global__ void __launch_bounds__(LM_PAGED_THREADS) attnres_paged_join_##NAME(lm_paged_params P) {  \
    __shared__ Shared S;                                                                                         \
    __shared__ f32x4 red[LM_PAGED_THREADS];                                                                      \
    paged_join<T>(P, S, red);                                                                                    \
  }
#define LM_PAGED(NAME, T, DP, DC, WPE)                     \
  LM_PAGED_KERNEL(NAME##_d##DC##_n, T, DP, DC, false, WPE) \
  LM_PAGED_KERNEL(NAME##_d##DC##_w, T, DP, DC, true, WPE)

#if LM_PART == 15
LM_PAGED_JOIN(bf16, Bf16)
LM_PAGED(bf16, Bf16, 64, 32, 2)
LM_PAGED(bf16, Bf16, 64, 64, 2)
LM_PAGED(bf16, Bf16, 128, 96, 2)
LM_PAGED(bf16, Bf16, 128, 128, 2)
LM_PAGED_JOIN(f32, F32)
LM_PAGED(f32, F32, 64, 32, 1)
LM_PAGED(f32, F32, 64, 64, 1)
LM_PAGED(f32, F32, 128, 96, 1)
LM_PAGED(f32, F32, 128, 128, 1)
#endif
