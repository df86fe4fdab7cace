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
// call has, the device how long they are; so the grid is fixed or a bound, and every
// workgroup finds its own work in the lengths.  Sequences of up to 32 rows (single
// tokens, drafts) are narrow tiles: four waves share the 32 rows and each works
// on 32 keys of a block of 128.
//
// Calls of few rows (paged_stream): all tiles are narrow.  The blocks of all
// sequences' tiles lie one after another, and each of a key head's workgroups (two on
// every CU, over all heads) takes an equal stretch of them, whatever
// sequences it leads through; or, where no row of the table holds many blocks, a workgroup
// takes a whole tile.
//
// Calls with rows enough to fill the card 128 at a time (paged_tiles): the rows of
// longer sequences are taken so, each wave 32 of them over all keys, a workgroup
// a tile, the longest of a sequence first.  Where they are too few or too unequal for the card, long tiles are
// split, narrow ones beside them too (part_blocks).
//
// What a workgroup has of a tile that others share goes to the workspace, with a
// note of its parts, and paged_join adds them in order, so that
// results repeat bit for bit.
//
// Keys are found through the table: a wave-wide load covers at most 8 rows,
// which lie in one page, so the page's address is uniform and a lane's
// offset within it the same for every page.  A wave reads the
// table entries of a tile with one load, a tile ahead of its keys.  An entry outside
// the cache is read as page 0 and makes the rows that are worked on with it NaN.

#include "attention_tiles.h"
#include "paged_schedule.h"

namespace {

constexpr int kThreads = LM_PAGED_THREADS;

// ---------------------------------------------------------------- schedule --

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Element i of 32- or 64-bit whole numbers, taken into [0, most]; without a branch: the
// compiler makes one for each otherwise, and the schedule is a chain of such reads.
__device__ __forceinline__ int taken(const void* p, int i, int is64, int most) {
  const int32_t* w = (const int32_t*)p + ((int64_t)i << is64);
  const int lo = w[0], up = w[is64], hi = is64 ? up : lo >> 31;
  return hi < 0 ? 0 : hi > 0 || (uint32_t)lo > (uint32_t)most ? most : lo;
}

// The sequences' sizes are taken into what the call has, so that no length
// leads out of its tensors.  Behind the last sequence (s == seqs): the tokens that
// belong to none, as a sequence without keys.
__device__ __forceinline__ Share share_of(const lm_paged_params& P, int s) {
  Share a;
  const int in = s < P.seqs ? s : P.seqs - 1;  // where the last is read in place of none
  int lo = s, hi = s + 1;
  if (P.q_starts != nullptr) {
    lo = s == 0 ? 0 : taken(P.q_starts, s, P.starts64, P.tokens);
    hi = taken(P.q_starts, in + 1, P.starts64, P.tokens);
  }
  hi = s < P.seqs ? hi : P.tokens;
  int kv_len = 0;
  if (P.seqs > 0) kv_len = taken(P.kv_lens, in, P.lens64, P.capacity);
  a.set(lo, hi, s < P.seqs ? kv_len : 0, P.group, P.wide != 0);
  return a;
}

// A sequence's own token of row r, rows a group for each (r under 2^31).
__device__ __forceinline__ int query_of(const lm_paged_params& P, int r) {
  return (int)((__umulhi((uint32_t)r, P.group_mul) + (uint32_t)r) >> P.group_shift);
}

// The launch's arguments, read anew: values that the code before holds on to would
// crowd a loop's scalar registers.
typedef const __attribute__((address_space(4))) lm_paged_params* ParamsPtr;
__device__ __forceinline__ const lm_paged_params& anew() {
  ParamsPtr p = (ParamsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const lm_paged_params*)p;
}

// What a workgroup takes of a tile: its key blocks t0 .. t1-1 (of 128 keys, in a wide tile 64).
struct Piece {
  Share a;
  int seq, tile, t0, t1;
  int slot;  // where its sums go in the workspace; -1: it has all keys, and writes the result
};

struct Shared {
  float sum[LM_ATTN_WAVES];
  float most[LM_ATTN_WAVES];
  float cost[kCuts], shared[kCuts];
  int scan[LM_ATTN_WAVES][2];
  int upto[kThreads][2];
  Share share;
  int seq, before;
};

// Sums of numbers that are not negative stop at the largest: starts that do not rise name rows many times over, and
// a sum that wrapped would lead out of the sequences.
__device__ __forceinline__ int add_sat(int a, int b) { return __builtin_elementwise_add_sat(a, b); }

// Inclusive sums of N numbers over the workgroup's threads into S.upto.
template <int N>
__device__ __forceinline__ void scan_all(int (&v)[N], Shared& S) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = __shfl_up(v[i], m);
      v[i] = add_sat(v[i], lane >= m ? x : 0);
    }
  __syncthreads();  // what was there has been read
  if (lane == 63) {
#pragma unroll
    for (int i = 0; i < N; ++i) S.scan[wave][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int w = 0; w < LM_ATTN_WAVES - 1; ++w) v[i] = add_sat(v[i], w < wave ? S.scan[w][i] : 0);
    S.upto[threadIdx.x][i] = v[i];
  }
  __syncthreads();
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
// Sum of `v` and largest of `t` over the workgroup, to every thread, in a fixed order.
__device__ __forceinline__ void sum_and_most(float& v, float& t, Shared& S) {
  v = wave_sum(v);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) t = fmaxf(t, __shfl_xor(t, m));
  if ((threadIdx.x & 63) == 0) {
    S.sum[threadIdx.x >> 6] = v;
    S.most[threadIdx.x >> 6] = t;
  }
  __syncthreads();
  v = t = 0.f;
#pragma unroll
  for (int i = 0; i < LM_ATTN_WAVES; ++i) {
    v += S.sum[i];
    t = fmaxf(t, S.most[i]);
  }
}

// The thread whose inclusive sum is the first over `at`, which is under the last.
__device__ __forceinline__ int find_upto(const Shared& S, int at) {
  int lo = 0;
#pragma unroll
  for (int step = kThreads / 2; step > 0; step >>= 1)
    if (S.upto[lo + step - 1][0] <= at) lo += step;
  return uniform(lo);
}

// A tile whose keys several workgroups share, for the join; whole tiles have none (parts 0).
__device__ __forceinline__ void write_note(const lm_paged_params& P, int at, const Share& a, int row0, int head,
                                           int parts, int first, int next, int step) {
  lm_paged_note n;
  n.token = a.first;
  n.row0 = row0;
  n.rows = a.rows;
  n.head = head;
  n.parts = parts;
  n.first = first;
  n.next = next;
  n.step = step;
  P.notes[at] = n;
}

// ------------------------------------------------------------------- pages --

// Where a head's rows lie: its first page's, and the bytes from page to page and row to row.
struct Rows {
  const char* base;
  uint32_t page_bytes, row_bytes;
  __device__ __forceinline__ Rows(const void* p, const lm_strides& st, int kvh, int es)
      : base((const char*)p + (int64_t)kvh * st.h * es), page_bytes((uint32_t)(st.b * es)),
        row_bytes((uint32_t)(st.t * es)) {}
  __device__ __forceinline__ const char* at(uint32_t page, uint32_t row) const {
    return base + (uint64_t)page * page_bytes + row * row_bytes;  // a page's rows span under 2^31 bytes
  }
};

// A sequence's pages as one wave reads them, and its keys and values by them.
// Everything here is uniform, and is kept in scalar registers by reading the table
// through the scalar cache: with the lanes' own addresses, or pages
// handed on by v_readlane, the wide tiles' vector unit, which is what they wait for
// next to the matrix cores, had 18% more to do (2048 tokens behind 14336, 32/8 heads of 128: 575 against 510 us).
template <typename KT>
struct Keys {
  static constexpr int kPerWave = 64 / KT::kChunks;  // rows of a wave's load
  static_assert(kPerWave <= LM_PAGED_MIN_PAGE && LM_PAGED_MIN_PAGE == 16, "in one page");
  static constexpr int kWaves = KT::kRound / kPerWave;
  static constexpr int kLog = KT::kRows == 64 ? 6 : 5;
  // Pages that a wave asks for in a tile: of each round's first row, or of each 16 rows.
  static constexpr bool kByRound = KT::kRound >= 16;
  static constexpr int kPages = kByRound ? KT::kRounds : KT::kRows / 16;

  const __attribute__((address_space(4))) int32_t* table;
  Rows k, v;
  int shift, pages, last;  // last: the last key that exists
  int chunks, wave;
  bool one;                // a tile lies in one page
  bool bad;                // an entry outside the cache was met
  int page[kPages];        // of the tile that is requested next

  __device__ __forceinline__ Keys(const lm_paged_params& P, const Piece& J, int kvh, int es, int wave_)
      : table((const __attribute__((address_space(4))) int32_t*)(P.table + (int64_t)J.seq * P.table_ld)),
        k(P.k, P.sk, kvh, es), v(P.v, P.sv, kvh, es), shift(P.shift), pages(P.pages), last(J.a.kv_len - 1),
        chunks(P.dim * es / 16), wave(wave_), one(P.shift >= kLog), bad(false) {}

  // Reads the pages of the tile from key `row0` on (a multiple of 32); of the last key's behind it.
  __device__ __forceinline__ void find(int row0) {
    auto of = [&](int j) {
      const int r = row0 + (kByRound ? j * KT::kRound + wave * kPerWave : 16 * j);
      return table[(r < last ? r : last) >> shift];
    };
    page[0] = of(0);
    if (one) {
#pragma unroll
      for (int j = 1; j < kPages; ++j) page[j] = page[0];
    } else {
#pragma unroll
      for (int j = 1; j < kPages; ++j) page[j] = of(j);
    }
  }
  __device__ __forceinline__ uint32_t checked(int p) {
    const bool out = (uint32_t)p >= (uint32_t)pages;
    bad = bad || out;
    return out ? 0 : (uint32_t)p;
  }

  // Requests that tile, as KT::request does for contiguous keys.
  __device__ __forceinline__ void request(char* kl, char* vl, int row0, int lane) {
    const uint32_t mask = (1u << shift) - 1;
    const int mine = lane / KT::kChunks;
    const uint32_t ko = (uint32_t)mine * k.row_bytes, vo = (uint32_t)mine * v.row_bytes;
    auto load = [&](int i, const char* kb, const char* vb, uint32_t kr, uint32_t vr) {
      const uint32_t c = KT::chunk_offset(i, wave, lane, chunks);
      KT::load_lds(kl + (i * kWaves + wave) * 1024, kb, kr + c);
      KT::load_lds(vl + (i * kWaves + wave) * 1024, vb, vr + c);
    };
    if (row0 + KT::kRows - 1 <= last) {
      if (one) {
        const uint32_t p = checked(page[0]), r = ((uint32_t)row0 & mask) + (uint32_t)(wave * kPerWave);
        const char *kb = k.at(p, r), *vb = v.at(p, r);
#pragma unroll
        for (int i = 0; i < KT::kRounds; ++i) {
          load(i, kb, vb, ko, vo);
          kb += KT::kRound * k.row_bytes;
          vb += KT::kRound * v.row_bytes;
        }
      } else {
#pragma unroll
        for (int i = 0; i < KT::kRounds; ++i) {
          const uint32_t p = checked(page[kByRound ? i : i * KT::kRound / 16]);
          const uint32_t r = (uint32_t)(row0 + i * KT::kRound + wave * kPerWave) & mask;
          load(i, k.at(p, r), v.at(p, r), ko, vo);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < KT::kRounds; ++i) {  // rows behind the last repeat it
        const uint32_t p = checked(page[kByRound ? i : i * KT::kRound / 16]);
        const int r = row0 + i * KT::kRound + wave * kPerWave + mine;
        const uint32_t in = (uint32_t)(r < last ? r : last) & mask;
        load(i, k.at(p, 0), v.at(p, 0), in * k.row_bytes, in * v.row_bytes);
      }
    }
  }
};

// ------------------------------------------------------------------- tiles --

// A row of a tile: which it is, and the keys it sees.
struct Row {
  int row, query, head, lim;
  bool exists;
  __device__ __forceinline__ Row(const lm_paged_params& P, const Share& a, int r, int kvh) {
    row = r;
    query = query_of(P, r);
    head = kvh * P.group + (r - query * P.group);
    exists = r < a.rows;
    lim = a.kv_len == 0 ? 0 : a.kv_len - a.count + query + 1;
  }
};
// The keys that row r sees, if any.
__device__ __forceinline__ int sees(const lm_paged_params& P, const Share& a, int r) {
  return a.kv_len == 0 ? 0 : a.kv_len - a.count + query_of(P, r) + 1;
}

template <typename T>
__device__ __forceinline__ const char* q_row(const lm_paged_params& P, const Share& a, const Row& R) {
  return (const char*)P.q + ((int64_t)(a.first + R.query) * P.q_t + (int64_t)R.head * P.q_h) * T::kBytes;
}
template <typename T>
__device__ __forceinline__ char* o_row(const lm_paged_params& P, const Share& a, const Row& R) {
  return (char*)P.o + ((int64_t)(a.first + R.query) * P.o_t + (int64_t)R.head * P.o_h) * T::kBytes;
}
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// The workgroup's LDS, in four arrays of their own: the compiler lets a read of one pass a
// load into another that is under way; where both are in one array it waits for the
// load, and a wide tile's next block is no longer on its way while it works on one.
#define LDS_ARRAYS LM_LDS char *a, LM_LDS char *b, LM_LDS char *c, LM_LDS char *d
template <typename T, int DP>
constexpr int kLdsBytes = Tile<T, DP, 64>::kBytes;  // of each
__device__ __forceinline__ char* lds_of(int wave, LDS_ARRAYS) {
  LM_LDS char* lo = wave == 0 ? a : b;
  LM_LDS char* hi = wave == 2 ? c : d;
  return (char*)(wave < 2 ? lo : hi);
}

// 32 rows, four waves: each works on its own 32 keys of a block of 128, loads them itself
// and waits for no other; in the end every wave adds all four's sums of its 32 columns.
// ml: 4 x 128 floats.
template <typename T, int DP, int DC>
__device__ __forceinline__ void narrow_tile(const Piece& J, int kvh, LDS_ARRAYS, float* ml) {
  using KT = Tile<T, DP, 32, 1>;
  const lm_paged_params& P = anew();
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = uniform(threadIdx.x >> 6);
  const int r0 = J.tile * 32;
  const Row R(P, J.a, r0 + (lane & 31), kvh);
  // rows that are not there are not stored
  const int most = uniform(sees(P, J.a, (r0 + 32 < J.a.rows ? r0 + 32 : J.a.rows) - 1));
  const int all = uniform(sees(P, J.a, r0));
  const int own = 32 * wave;
  const int end = most < J.t1 * 128 ? most : J.t1 * 128;  // of the keys

  typename T::Frag qf[DC / 16];
  load_rows<T, DC>(qf, q_row<T>(P, J.a, R), P.dim, h, R.exists);
  f32x16 acc[DC / 32];
#pragma unroll
  for (int i = 0; i < DC / 32; ++i) acc[i] = zero16();
  float m = kNegInf, l = 0.f;
  const int row_at = KT::row_at(lane), col_at = KT::col_at(lane);
  Keys<KT> keys(P, J, kvh, T::kBytes, 0);
  char* kc = lds_of(wave, a, b, c, d);
  char* vc = kc + KT::kBytes;
  int key0 = J.t0 * 128 + own;
  if (key0 < end) keys.find(key0);
  for (; key0 < end; key0 += 128) {
    int ln = lane;  // opaque: offsets formed anew for each block instead of held in registers
    asm volatile("" : "+v"(ln));
    keys.request(kc, vc, key0, ln);
    if (key0 + 128 < end) keys.find(key0 + 128);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    attend<T, KT, DC, 1>(kc, vc, 0, key0, all, R.lim, qf, acc, m, l, P.scale_log2, row_at, col_at, lane, h);
  }
  l += other_half(l);
  if (keys.bad) l = __builtin_nanf("");
  static_assert(64 * DC / 2 * 4 <= kLdsBytes<T, DP>, "a wave's sums in its array");
  put<DC>(reinterpret_cast<float*>(kc), acc, lane);
  ml[wave * 128 + lane] = m;
  ml[wave * 128 + 64 + lane] = l;
  __syncthreads();
  m = kNegInf;
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w * 128 + lane]);
  float fade[4];
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float om = ml[w * 128 + lane];
    fade[w] = om == kNegInf ? 0.f : exp2_fast(om - m);
    l = __builtin_fmaf(ml[w * 128 + 64 + lane], fade[w], l);  // a NaN stays one
  }
  if (wave < DC / 32 && R.exists) {
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      sum[i] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        sum[i] = __builtin_fmaf(reinterpret_cast<const float*>(lds_of(w, a, b, c, d))[(wave * 16 + i) * 64 + lane],
                                fade[w], sum[i]);
    }
    const lm_paged_params& P = anew();
    const bool whole = J.slot < 0;
    const int64_t at = (int64_t)J.slot * P.part_rows + (R.row - r0);
    const float scale = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
    char* to = o_row<T>(P, J.a, R);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * wave + 8 * a + 4 * h;
      if (d >= P.dim) continue;
      if (whole)
        store4<T>(to + d * T::kBytes, sum[4 * a] * scale, sum[4 * a + 1] * scale, sum[4 * a + 2] * scale,
                  sum[4 * a + 3] * scale);
      else
        store4<F32>(reinterpret_cast<char*>(P.part + at * P.dim + d), sum[4 * a], sum[4 * a + 1], sum[4 * a + 2],
                    sum[4 * a + 3]);
    }
    if (wave == 0 && h == 0) {
      if (!whole) {
        P.part_ml[at * 2] = m;
        P.part_ml[at * 2 + 1] = l;
      } else if (P.lse != nullptr) {
        P.lse[(int64_t)(J.a.first + R.query) * P.heads + R.head] = lse_of(m, l);
      }
    }
  }
}

// 128 rows, each wave 32 of them over all keys: the waves share the blocks of 64, the next
// requested before one is worked on, its pages read a block before that.
template <typename T, int DP, int DC>
__device__ __forceinline__ void wide_tile(const Piece& J, int kvh, LDS_ARRAYS, int* flag) {
  using KT = Tile<T, DP, 64>;
  const lm_paged_params& P = anew();
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = uniform(threadIdx.x >> 6);
  const int g0 = J.tile * 128, r0 = g0 + wave * 32;
  const Row R(P, J.a, r0 + (lane & 31), kvh);
  auto last_of = [&](int r) { return (r < J.a.rows ? r : J.a.rows) - 1; };
  const int most = uniform(r0 < J.a.rows ? sees(P, J.a, last_of(r0 + 32)) : 0);
  const int all = uniform(sees(P, J.a, r0));
  const int any = uniform(sees(P, J.a, last_of(g0 + 128)));
  const int t1 = any < J.t1 * 64 ? (any + 63) >> 6 : J.t1;  // 0 or less where no row sees a key: the loop is empty

  typename T::Frag qf[DC / 16];
  load_rows<T, DC>(qf, q_row<T>(P, J.a, R), P.dim, h, R.exists);
  f32x16 acc[DC / 32];
#pragma unroll
  for (int i = 0; i < DC / 32; ++i) acc[i] = zero16();
  float m = kNegInf, l = 0.f;
  const int row_at = KT::row_at(lane), col_at = KT::col_at(lane);
  Keys<KT> keys(P, J, kvh, T::kBytes, wave);
  auto request = [&](int t, char* k, char* v) {
    keys.request(k, v, t * 64, lane);
    if (t + 1 < t1) keys.find((t + 1) * 64);
  };
  auto arrived = [] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  auto step = [&](int t, const char* kc, const char* vc) {
    if (t * 64 >= most) return;
    attend<T, KT, DC, 2>(kc, vc, 0, t * 64, all, R.lim, qf, acc, m, l, P.scale_log2, row_at, col_at, lane, h);
  };
  if (J.t0 < t1) {
    keys.find(J.t0 * 64);
    request(J.t0, (char*)a, (char*)b);
  }
  for (int t = J.t0; t < t1; t += 2) {
    arrived();
    if (t + 1 < t1) request(t + 1, (char*)c, (char*)d);
    step(t, (char*)a, (char*)b);
    if (t + 1 < t1) {
      arrived();
      if (t + 2 < t1) request(t + 2, (char*)a, (char*)b);
      step(t + 1, (char*)c, (char*)d);
    }
  }
  // a page outside the cache that any wave met
  if (keys.bad && lane == 0) *flag = 1;
  __syncthreads();
  l += other_half(l);
  if (*flag != 0) l = __builtin_nanf("");
  if (!R.exists) return;
  const lm_paged_params& E = anew();
  if (J.slot >= 0) {
    const int64_t at = (int64_t)J.slot * E.part_rows + (R.row - g0);
    store_rows<F32, DC>(reinterpret_cast<char*>(E.part + at * E.dim), acc, 1.f, E.dim, h);
    if (h == 0) {
      E.part_ml[at * 2] = m;
      E.part_ml[at * 2 + 1] = l;
    }
    return;
  }
  store_rows<T, DC>(o_row<T>(E, J.a, R), acc, l == 0.f ? 0.f : 1.f / l, E.dim, h);
  if (E.lse != nullptr && h == 0) E.lse[(int64_t)(J.a.first + R.query) * E.heads + R.head] = lse_of(m, l);
}

// ------------------------------------------------------------- few rows --

// Key blocks of a tile.
__device__ __forceinline__ int tile_blocks(const Share& a) { return (a.kv_len + 127) >> 7; }
// And what it counts for in the stretches: one where tiles are not split, and where it has no keys, as it is
// written too.
__device__ __forceinline__ int tile_units(const lm_paged_params& P, const Share& a) {
  return P.slots > 0 && a.kv_len > 128 ? tile_blocks(a) : 1;
}

template <typename T, int DP, int DC>
__device__ __forceinline__ void paged_stream(const lm_paged_params& P, LDS_ARRAYS, float* ml, Shared& S) {
  const int kvh = (int)blockIdx.x % P.kv_heads, w = (int)blockIdx.x / P.kv_heads;
  auto share = [&](int s) { return share_of(P, s < P.seqs ? s : P.seqs); };
  auto units = [&](const Share& x, int s) { return s > P.seqs ? 0 : x.tiles * tile_units(P, x); };
  // all units (under 2^31 where starts rise: the host sees to it), and this workgroup's stretch of them
  Share mine = share((int)threadIdx.x);
  int v[1] = {units(mine, (int)threadIdx.x)};
  scan_all<1>(v, S);
  int total = S.upto[kThreads - 1][0];
  for (int base = kThreads; base <= P.seqs; base += kThreads) {
    v[0] = units(share(base + (int)threadIdx.x), base + (int)threadIdx.x);
    scan_all<1>(v, S);
    total = add_sat(total, S.upto[kThreads - 1][0]);
  }
  const int each = (int)(((int64_t)total + P.target - 1) / P.target);
  const int64_t begin = (int64_t)w * each;
  int at = begin < total ? (int)begin : total;
  const int end = total - at > each ? at + each : total;
  const int note = w * P.kv_heads + kvh;          // this workgroup's note, and its slot of a tile that it begins
  const int cont = P.target * P.kv_heads + note;  // of one that it goes on with
  bool noted = false;
  if (at < end) {
    // the sequence in which the stretch begins: its thread hands it on
    int before = 0, base = 0;
    if (P.seqs >= kThreads) {
      for (;; base += kThreads) {
        mine = share(base + (int)threadIdx.x);
        v[0] = units(mine, base + (int)threadIdx.x);
        scan_all<1>(v, S);
        if (at - before < S.upto[kThreads - 1][0]) break;
        before += S.upto[kThreads - 1][0];
      }
    }
    const int front = threadIdx.x > 0 ? S.upto[threadIdx.x - 1][0] : 0;
    if (at - before < v[0] && at - before >= front) {
      S.share = mine;
      S.seq = base + (int)threadIdx.x;
      S.before = before + front;
    }
    __syncthreads();
    Piece J;
    J.a = S.share;
    J.seq = uniform(S.seq);
    before = uniform(S.before);
    int n = tile_units(P, J.a);
    J.tile = uniform((at - before) / n);
    J.t0 = uniform(at - before - J.tile * n);
    for (;;) {
      const int left = end - at;
      const bool ends = n - J.t0 <= left;  // with this tile's last block
      const int taken = ends ? n - J.t0 : left;
      J.t1 = uniform(ends ? tile_blocks(J.a) : J.t0 + left);
      J.slot = J.t0 > 0 ? cont : ends ? -1 : note;
      if (J.t0 == 0 && !ends) {
        noted = true;
        if (threadIdx.x == 0)
          write_note(P, note, J.a, J.tile * 32, kvh, 1 + (n - J.t1 + each - 1) / each, note, cont + P.kv_heads,
                     P.kv_heads);
      }
      narrow_tile<T, DP, DC>(J, kvh, a, b, c, d, ml);
      at += taken;
      if (at >= end) break;
      J.t0 = 0;
      if (++J.tile >= J.a.tiles) {
        J.tile = 0;
        do {  // there is one: units are left
          J.a = share_of(P, ++J.seq);
        } while (J.a.tiles == 0);
        n = tile_units(P, J.a);
      }
      __syncthreads();  // the sums have been read
    }
  }
  if (!noted && P.slots > 0 && threadIdx.x == 0) P.notes[note].parts = 0;
}

// ------------------------------------------------------------ many rows --

// The cut (Cuts) of the call's tiles.  `used`: how many parts of split tiles a head has with it.
template <bool TWO>  // workgroups of a CU
__device__ __forceinline__ int part_blocks(const lm_paged_params& P, int all, int* used, Shared& S) {
  float work = 0.f, top = 0.f;
  for (int s = threadIdx.x; s < P.seqs; s += kThreads) {
    const Share a = share_of(P, s);
    const float n = a.tiles > 0 ? (float)blocks_of(a) : 0.f;
    work += (float)a.tiles * n;
    top = fmaxf(top, n);
  }
  sum_and_most(work, top, S);
  const Cuts C(work, top, P.target, P.kv_heads);
  *used = 0;
  if (P.slots == 0 || C.many()) return uniform(C.longest);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
#pragma unroll
  for (int u = 0; u < kCuts / LM_ATTN_WAVES; ++u) {  // each wave its own
    const int j = wave * (kCuts / LM_ATTN_WAVES) + u, most = uniform(C.most(j));
    float parts = 0.f, shared = 0.f;
    for (int s = lane; s <= P.seqs; s += 64) {  // the rows behind the last too: whole tiles
      const Share a = share_of(P, s);
      const Split sp(a, most);
      const float n = (float)a.tiles * (float)sp.parts;
      parts += n;
      shared += sp.parts > 1 ? n : 0.f;
    }
    parts = wave_sum(parts);
    shared = wave_sum(shared);
    if (lane == 0) {
      S.cost[j] = C.cost(most, parts, shared, TWO, P.slots, all);
      S.shared[j] = shared;
    }
  }
  __syncthreads();
  int best = 0;
#pragma unroll
  for (int j = 1; j < kCuts; ++j) best = S.cost[j] < S.cost[best] ? j : best;
  *used = uniform((int)S.shared[best]);
  return uniform(C.most(best));
}

template <typename T, int DP, int DC>
__device__ __forceinline__ void paged_tiles(const lm_paged_params& P, LDS_ARRAYS, float* ml, int* flag, Shared& S) {
  // Workgroups go to the eight XCDs in turn, each with an L2 of its own: where the key heads
  // divide by eight, each XCD takes an eighth of them, so that the tiles of a sequence's rows find
  // a head's keys in one L2.
  int w = (int)blockIdx.x, kvh;
  const int all = (int)gridDim.x / P.kv_heads;  // workgroups of a head
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
  if (threadIdx.x == 0) *flag = 0;
  int used;
  const int most = part_blocks<!(T::kBytes == 4 && DC > 64)>(P, all, &used, S);
  if (threadIdx.x == 0)
    for_unused_notes(w, all, used, P.slots, [&](int i) { P.notes[(int64_t)i * P.kv_heads + kvh].parts = 0; });
  // the sequence of part w, all sequences' parts one after another, and the slots in front of its
  int parts = 0, slots = 0, base = 0;
  bool found = false;
  for (; base <= P.seqs; base += kThreads) {
    const int s = base + (int)threadIdx.x;
    const Share a = share_of(P, s < P.seqs ? s : P.seqs);
    const Split sp(a, most);
    int v[2];
    v[0] = s <= P.seqs ? a.tiles * sp.parts : 0;
    v[1] = sp.parts > 1 ? v[0] : 0;
    scan_all<2>(v, S);
    const int n = S.upto[kThreads - 1][0];
    found = w - parts < n;
    if (found) break;
    parts = add_sat(parts, n);
    slots = add_sat(slots, S.upto[kThreads - 1][1]);
  }
  if (!found) return;
  const int lo = find_upto(S, w - parts);
  Piece J;
  J.seq = base + lo;
  J.a = share_of(P, J.seq);
  const Split sp(J.a, most);
  const int i = uniform(w - parts - (lo > 0 ? S.upto[lo - 1][0] : 0));
  const int rank = i / sp.parts, part = i - rank * sp.parts;
  // The longest first; where all tiles run at once, those that share a CU with them the shortest first (prompts from
  // their start: 4 of 2048, 8/4 heads of 128, 61 us, all longest first 70; one of 8192, 190 and 208).
  const int early = P.turn > 0 && sp.parts == 1 ? P.turn - (w - i) : J.a.tiles;  // of this sequence
  J.tile = uniform(rank < early || early >= J.a.tiles ? J.a.tiles - 1 - rank : rank - (early > 0 ? early : 0));
  J.t0 = uniform(part * sp.per);
  J.t1 = uniform(J.t0 + sp.per < sp.n ? J.t0 + sp.per : sp.n);
  J.slot = -1;
  if (sp.parts > 1) {
    const int first = uniform(add_sat(add_sat(slots, lo > 0 ? S.upto[lo - 1][1] : 0), rank * sp.parts));
    if (first > P.slots - sp.parts) return;  // lengths that change under the launch
    J.slot = (first + part) * P.kv_heads + kvh;
    if (threadIdx.x == 0)
      write_note(P, J.slot, J.a, J.tile * (J.a.narrow ? 32 : 128), kvh, part == 0 ? sp.parts : 0, J.slot,
                 J.slot + P.kv_heads, P.kv_heads);
  }
  if (J.a.narrow)
    narrow_tile<T, DP, DC>(J, kvh, a, b, c, d, ml);
  else
    wide_tile<T, DP, DC>(J, kvh, a, b, c, d, flag);
}

// -------------------------------------------------------------------- join --

// Joins the parts of a tile that workgroups shared (blockIdx.x: its note).  Eight lane groups
// of 32, four columns a lane, take a row's parts in turn, or, where it has
// fewer than eight, several rows.  A row's maxima and sums are requested together with its
// first parts, so that up to 64 parts are one round trip.
template <typename T>
__device__ __forceinline__ void paged_join(const lm_paged_params& P, f32x4* red) {
  const lm_paged_note N = P.notes[blockIdx.x];
  if (N.parts < 2) return;
  // lengths that change under the launch can leave a note unwritten: what leads out of the call is none
  const int64_t slots = (int64_t)P.slots * P.kv_heads;
  if (N.first < 0 || N.first >= slots || N.next < 0 || N.step < 1 ||
      N.next + (N.parts - 2) * (int64_t)N.step >= slots || N.token < 0 || N.row0 < 0 || N.head < 0 ||
      N.head >= P.kv_heads || (int64_t)N.token * P.group + N.rows > (int64_t)P.tokens * P.group)
    return;
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, d = 4 * lane;
  const int pp = N.parts <= 2 ? 2 : N.parts <= 4 ? 4 : 8, each = 8 / pp;  // parts and rows side by side
  const int phase = g % pp;
  const int left = N.rows - N.row0, rows = left < P.part_rows ? left : P.part_rows;
  auto line = [&](int p, int r) {
    return (int64_t)(p == 0 ? N.first : N.next + (int64_t)(p - 1) * N.step) * P.part_rows + r;
  };
  constexpr int U = 8;
  for (int r0 = (int)blockIdx.y * each; r0 < rows; r0 += (int)gridDim.y * each) {
    const int r = r0 + g / pp;
    const bool live = r < rows;
    const int rr = live ? r : r0;
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = phase + pp * u < N.parts ? phase + pp * u : phase < N.parts ? phase : 0;
      v[u] = *reinterpret_cast<const f32x4*>(P.part + line(p, rr) * P.dim + (d < P.dim ? d : 0));
    }
    // the common maximum and the sum: 32 lanes over the parts
    float m = kNegInf, l = 0.f;
    for (int p = lane; p < N.parts; p += 32) m = fmaxf(m, P.part_ml[line(p, rr) * 2]);
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    auto weight = [&](float pm) { return pm == kNegInf ? 0.f : exp2_fast(pm - m); };
    for (int p = lane; p < N.parts; p += 32) {
      const int64_t at = line(p, rr) * 2;
      l = __builtin_fmaf(P.part_ml[at + 1], weight(P.part_ml[at]), l);  // a NaN stays one
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) l += __shfl_xor(l, x);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    auto take = [&](int p, const f32x4& x) {
      const float w = weight(P.part_ml[line(p, rr) * 2]);
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] = __builtin_fmaf(x[c], w, sum[c]);
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (phase + pp * u < N.parts) take(phase + pp * u, v[u]);
    for (int p = phase + pp * U; p < N.parts; p += pp)
      take(p, *reinterpret_cast<const f32x4*>(P.part + line(p, rr) * P.dim + (d < P.dim ? d : 0)));
    red[threadIdx.x] = sum;
    __syncthreads();
    if (phase == 0 && live && d < P.dim) {
      for (int p = 1; p < pp; ++p) {
        const f32x4 o = red[threadIdx.x + 32 * p];
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] += o[c];
      }
      const int row = N.row0 + r, query = query_of(P, row), head = N.head * P.group + (row - query * P.group);
      const int64_t token = N.token + query;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      store4<T>((char*)P.o + (token * P.o_t + (int64_t)head * P.o_h + d) * T::kBytes, sum[0] * inv, sum[1] * inv,
                sum[2] * inv, sum[3] * inv);
      if (P.lse != nullptr && d == 0) P.lse[token * P.heads + head] = lse_of(m, l);
    }
    __syncthreads();
  }
}

}  // namespace

// DP: elements of a tile's row in LDS; DC: columns worked on, the head size rounded up to 32.
#define LM_PAGED_LDS(T, DP)                                                                                      \
  __shared__ __align__(16) char a[kLdsBytes<T, DP>];                                                           \
  __shared__ __align__(16) char b[kLdsBytes<T, DP>];                                                           \
  __shared__ __align__(16) char c[kLdsBytes<T, DP>];                                                           \
  __shared__ __align__(16) char d[kLdsBytes<T, DP>];                                                           \
  __shared__ float ml[512];                                                                                      \
  __shared__ Shared S;
#define LM_PAGED(NAME, T, DP, DC, WPE)                                                                           \
  extern "C" __global__ void __launch_bounds__(LM_PAGED_THREADS) __attribute__((amdgpu_waves_per_eu(WPE)))      \
      attnres_paged_stream_##NAME##_d##DC(lm_paged_params P) {                                                   \
    LM_PAGED_LDS(T, DP)                                                                                          \
    paged_stream<T, DP, DC>(P, (LM_LDS char*)a, (LM_LDS char*)b, (LM_LDS char*)c, (LM_LDS char*)d, ml, S);       \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(LM_PAGED_THREADS) __attribute__((amdgpu_waves_per_eu(WPE)))      \
      attnres_paged_tiles_##NAME##_d##DC(lm_paged_params P) {                                                    \
    LM_PAGED_LDS(T, DP)                                                                                          \
    __shared__ int flag;                                                                                         \
    paged_tiles<T, DP, DC>(P, (LM_LDS char*)a, (LM_LDS char*)b, (LM_LDS char*)c, (LM_LDS char*)d, ml, &flag, S); \
  }
#define LM_PAGED_JOIN(NAME, T)                                                                                   \
  extern "C" __global__ void __launch_bounds__(LM_PAGED_THREADS) attnres_paged_join_##NAME(lm_paged_params P) {  \
    __shared__ f32x4 red[LM_PAGED_THREADS];                                                                      \
    paged_join<T>(P, red);                                                                                       \
  }

#if LM_PART == 15
LM_PAGED_JOIN(bf16, Bf16)
LM_PAGED(bf16, Bf16, 64, 32, 2)
LM_PAGED(bf16, Bf16, 64, 64, 2)
LM_PAGED(bf16, Bf16, 128, 96, 2)
LM_PAGED(bf16, Bf16, 128, 128, 2)
#endif
#if LM_PART == 16
LM_PAGED_JOIN(f32, F32)
LM_PAGED(f32, F32, 64, 32, 1)
LM_PAGED(f32, F32, 64, 64, 1)
LM_PAGED(f32, F32, 128, 96, 1)
LM_PAGED(f32, F32, 128, 128, 1)
#endif
