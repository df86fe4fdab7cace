// What a serving step needs around its attention over a paged cache, for gfx950:
// block tables and slot maps from the requests' lengths, the write of new keys
// and values into their slots, and the verification of drafted tokens.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lm_params.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

namespace {

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int is64) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// ------------------------------------------------------------------- slots --
//
//   have = ceil(held / page_size),  want = ceil((held + new) / page_size)
// A sequence that needs want - have pages gets them where the needs of all sequences
// up to it are at most the free pages, else none.  Every workgroup scans all lengths (a few
// thousand at most, in L2) and takes its share of the tokens, so that one
// launch does and no workgroup waits for another.  Tokens find their sequence by a
// search over 1024 ends in LDS.  Bound by latency: the lengths, their
// sums and the pages, each waiting for the one before.  The sums are 1024 threads' in 64 bits,
// over 16 waves, however few sequences there are.

constexpr int kSlotWaves = LM_SLOTS_THREADS / 64;
constexpr int kMaxTokens = 1 << 30;  // of one sequence
constexpr int kRefused = INT32_MIN;

struct SlotShared {
  int64_t scan[kSlotWaves][2];
  int32_t ends[LM_SLOTS_THREADS];
  int32_t first[LM_SLOTS_THREADS];
  int32_t held[LM_SLOTS_THREADS];
  int32_t taken;
};

// Inclusive sums of two numbers over the workgroup, from `before` on; `before` becomes the sum over all.
__device__ __forceinline__ void scan2(int64_t& a, int64_t& b, int64_t (&before)[2], SlotShared& S) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t x = __shfl_up(a, m), y = __shfl_up(b, m);
    a += lane >= m ? x : 0;
    b += lane >= m ? y : 0;
  }
  if (lane == 63) {
    S.scan[wave][0] = a;
    S.scan[wave][1] = b;
  }
  __syncthreads();
  a += before[0];
  b += before[1];
#pragma unroll
  for (int i = 0; i < kSlotWaves; ++i) {
    const int64_t x = S.scan[i][0], y = S.scan[i][1];
    a += i < wave ? x : 0;
    b += i < wave ? y : 0;
    before[0] += x;
    before[1] += y;
  }
}

// The first of the ends (in rising order) over `at`, which is under the last.
__device__ __forceinline__ int find_end(const int32_t* ends, int at) {
  int lo = 0;
#pragma unroll
  for (int step = LM_SLOTS_THREADS / 2; step > 0; step >>= 1)
    if (ends[lo + step - 1] <= at) lo += step;
  return lo;
}

__device__ __forceinline__ int32_t page_count(int64_t tokens, int shift) {
  return (int32_t)((tokens + ((1 << shift) - 1)) >> shift);
}
__device__ __forceinline__ int32_t clamp_to(int64_t v, int32_t most) {
  return v < 0 ? 0 : v > most ? most : (int32_t)v;
}

__device__ __forceinline__ void paged_slots(const lm_slots_params& P, SlotShared& S) {
  const int tid = threadIdx.x;
  const int32_t count = clamp_to(P.count[0], P.free_len);
  const int64_t stride = (int64_t)gridDim.x * LM_SLOTS_THREADS;
  const int64_t mine = (int64_t)blockIdx.x * LM_SLOTS_THREADS + tid;
  int64_t before[2] = {0, 0};  // tokens and pages asked for by the sequences in front of this stretch
  if (tid == 0) S.taken = 0;
  for (int base = 0; base < P.seqs; base += LM_SLOTS_THREADS) {
    const int s = base + tid;
    int64_t held = 0, tokens = 0, need = 0;
    bool sane = false;
    if (s < P.seqs) {
      held = index_at(P.held, s, P.held64);
      const int64_t n = index_at(P.change, s, P.change64);
      sane = held >= 0 && held <= kMaxTokens && n >= 0 && n <= kMaxTokens;
      tokens = clamp_to(n, kMaxTokens);
      held = sane ? held : 0;
      const int32_t want = page_count(held + tokens, P.shift);
      sane = sane && want <= P.table_width;
      need = sane ? want - page_count(held, P.shift) : 0;
    }
    const int begin = clamp_to(before[0], P.tokens);
    int64_t end = tokens, upto = need;
    scan2(end, upto, before, S);
    // (sequences behind one whose tokens the call has not are all refused: what they ask for does not show)
    const bool granted = sane && end <= P.tokens && (need == 0 || upto <= count);
    S.ends[tid] = clamp_to(end, P.tokens);
    // of the new pages in the free list
    S.first[tid] = !granted ? kRefused : need > 0 ? (int32_t)(count - 1 - (upto - need)) : 0;
    S.held[tid] = (int32_t)held;
    if (granted && need > 0) atomicMax(&S.taken, (int32_t)upto);  // those granted are the first that ask
    if (blockIdx.x == 0 && s < P.seqs) {
      P.q_starts[s + 1] = S.ends[tid];
      P.kv_lens[s] = granted ? (int32_t)(held + tokens) : 0;
    }
    __syncthreads();
    const int last = S.ends[LM_SLOTS_THREADS - 1];
    for (int64_t n = begin + mine; n < last; n += stride) {
      const int i = find_end(S.ends, (int)n);
      const int32_t at = S.held[i] + ((int)n - (i > 0 ? S.ends[i - 1] : begin));
      const int32_t first = S.first[i];
      int32_t slot = -1;
      if (first != kRefused) {
        const int32_t p = at >> P.shift, have = page_count(S.held[i], P.shift);
        int32_t* row = P.table + (int64_t)(base + i) * P.table_ld;
        const int32_t page = p < have ? row[p] : P.free[first - (p - have)];
        const int32_t in = at & ((1 << P.shift) - 1);
        if (in == 0) row[p] = page;  // a page's first row is that of a new token, and the page new
        if (page >= 0 && page < P.page_limit) slot = (page << P.shift) + in;
      }
      P.slots[n] = slot;
      P.positions[n] = at;
    }
    __syncthreads();
  }
  for (int64_t n = clamp_to(before[0], P.tokens) + mine; n < P.tokens; n += stride) {
    P.slots[n] = -1;
    P.positions[n] = 0;
  }
  if (blockIdx.x == 0 && tid == 0) {
    P.q_starts[0] = 0;
    P.count_out[0] = count - S.taken;
  }
}

// Gives back the pages behind the kept tokens: a sequence's last page first, so that
// the next to be taken is the one that continues it.
__device__ __forceinline__ void paged_release(const lm_slots_params& P, SlotShared& S) {
  const int tid = threadIdx.x;
  const int32_t count = clamp_to(P.count[0], P.free_len);
  const int64_t stride = (int64_t)gridDim.x * LM_SLOTS_THREADS;
  const int64_t mine = (int64_t)blockIdx.x * LM_SLOTS_THREADS + tid;
  int64_t before[2] = {0, 0};
  const int32_t room = P.free_len - count;
  for (int base = 0; base < P.seqs; base += LM_SLOTS_THREADS) {
    const int s = base + tid;
    int64_t back = 0, none = 0;
    int32_t have = 0;
    if (s < P.seqs) {
      int64_t held = index_at(P.held, s, P.held64);
      held = held > kMaxTokens ? 0 : held < 0 ? 0 : held;
      const int32_t kept = clamp_to(index_at(P.change, s, P.change64), (int32_t)held);
      have = page_count(held, P.shift);
      have = have < P.table_width ? have : P.table_width;
      const int32_t keep = page_count(kept, P.shift);
      back = have > keep ? have - keep : 0;
    }
    const int begin = clamp_to(before[0], room);
    scan2(back, none, before, S);
    S.ends[tid] = clamp_to(back, room);
    S.first[tid] = have;
    __syncthreads();
    const int last = S.ends[LM_SLOTS_THREADS - 1];
    for (int64_t n = begin + mine; n < last; n += stride) {
      const int i = find_end(S.ends, (int)n);
      const int32_t p = S.first[i] - 1 - ((int)n - (i > 0 ? S.ends[i - 1] : begin));
      P.free[count + n] = P.table[(int64_t)(base + i) * P.table_ld + p];
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) P.count_out[0] = count + clamp_to(before[0], room);
}

// ------------------------------------------------------------------- write --

// A thread per 16-byte piece of a token's keys, and the same of its values.
__device__ __forceinline__ void paged_write(const lm_write_params& P) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t n = i / P.per_token;
  if (n >= P.tokens) return;
  const int c = (int)(i - n * P.per_token), h = c / P.chunks, d = 16 * (c - h * P.chunks);
  const int64_t slot = index_at(P.slots, n, P.slots64);
  if (slot < 0 || slot >= P.limit) return;
  const int64_t page = slot >> P.shift, row = slot & ((1 << P.shift) - 1);
  const u32x4 k = *(const u32x4*)((const char*)P.k + n * P.k_t + h * P.k_h + d);
  const u32x4 v = *(const u32x4*)((const char*)P.v + n * P.v_t + h * P.v_h + d);
  *(u32x4*)((char*)P.k_cache + page * P.sk.b + h * P.sk.h + row * P.sk.t + d) = k;
  *(u32x4*)((char*)P.v_cache + page * P.sv.b + h * P.sv.h + row * P.sv.t + d) = v;
}

// ------------------------------------------------------------------ verify --
//
//   p = softmax(logits / temperature);  a draft d with probability q(d) stays if u0 q(d) < p(d)
//   the first that does not is replaced by a token from max(p - q, 0), and behind drafts
//   that all stay one comes from p: the first j whose sum up to j is over u1 of the whole sum
// Without draft probabilities q is 1 at the draft; greedily (temperature 0) p is 1 at the
// largest logit, the lowest index where several are.
//
// Which token a number falls to depends on sums over the whole vocabulary next to
// a border, of which there are as many as tokens: in 32 bits one choice in some
// hundreds would be another's.  So exponentials and sums are taken in 64.  Three launches:
//   rows   a wave per 2048 logits of each row: the largest, and the sum of exponentials
//          against it
//   pieces a workgroup per 4096 of the one row of each sequence that a token is taken
//          from (every one finds the first draft that falls for itself): the weights'
//          sum of each 512
//   pick   a wave per sequence: the piece, then the token in it
// (The last workgroup of a sequence to arrive could pick: one launch less, but the fence that
// shows it the others' sums writes back an L2 each time, 73 us more for 64 sequences.)
// Bound by the first launch: reading the logits once, and 64-bit arithmetic on them after
// that (one round of workgroups fills the card, so that one does not hide the other);
// for few rows by the launches' latencies.  64 sequences of up to 8 drafts, vocabulary
// 49152, bf16: 17 + 11 + 5 us (35 MB; 7 us at a copy's rate).

constexpr int kVerifyThreads = 256;
constexpr int kSide = kVerifyThreads / 16;  // drafts side by side
constexpr float kNegInf = -__builtin_inff();

// Eight consecutive values of a row from column j on (j a multiple of 8); `fill` behind its end.
__device__ __forceinline__ void get8(const void* row, int j, int n, int f32, int vec, float fill, float (&v)[8]) {
  if (vec && j + 8 <= n) {
    if (f32) {
      const u32x4 a = *(const u32x4*)((const float*)row + j), b = *(const u32x4*)((const float*)row + j + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = a[i], y = b[i];
        v[i] = __builtin_bit_cast(float, x);
        v[4 + i] = __builtin_bit_cast(float, y);
      }
    } else {
      const u32x4 a = *(const u32x4*)((const uint16_t*)row + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = a[i];
        v[2 * i] = __builtin_bit_cast(float, x << 16);
        v[2 * i + 1] = __builtin_bit_cast(float, x & 0xffff0000u);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at = j + i < n ? j + i : n - 1;
    const float x = f32 ? ((const float*)row)[at]
                        : __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[at] << 16);
    v[i] = j + i < n ? x : fill;
  }
}
__device__ __forceinline__ const char* row_of(const void* base, int64_t ld, int64_t r, int f32) {
  return (const char*)base + r * ld * (f32 ? 4 : 2);
}
__device__ __forceinline__ float get1(const void* row, int j, int f32) {
  return f32 ? ((const float*)row)[j] : __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[j] << 16);
}

template <typename N>
__device__ __forceinline__ N wave_sum(N v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// 2^t for t <= 0, to 1e-15 of itself: the polynomial that meets 2^f at the eleven Chebyshev points of
// [-1/2, 1/2].  Under 2^-1080 it is zero, and a NaN is taken for that.
__device__ __forceinline__ double exp2_neg(double t) {
  t = fmax(t, -1080.0);
  const double n = __builtin_rint(t), f = t - n;
  double p = 7.07258594926922339e-09;
  p = __builtin_fma(p, f, 1.02086902999583060e-07);
  p = __builtin_fma(p, f, 1.32154425879216893e-06);
  p = __builtin_fma(p, f, 1.52526572602008367e-05);
  p = __builtin_fma(p, f, 1.54035304417360499e-04);
  p = __builtin_fma(p, f, 1.33335582301649744e-03);
  p = __builtin_fma(p, f, 9.61812910760688825e-03);
  p = __builtin_fma(p, f, 5.55041086644477225e-02);
  p = __builtin_fma(p, f, 2.40226506959100972e-01);
  p = __builtin_fma(p, f, 6.93147180559949949e-01);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// (top, at) of the larger value, the lower index where both are the same.
__device__ __forceinline__ void larger(float& top, int& at, float t, int a) {
  const bool take = t > top || (t == top && a < at);
  top = take ? t : top;
  at = take ? a : at;
}

// The tokens' rows lie in the call: starts are taken into it.  Without a branch, so that several are requested
// together.
__device__ __forceinline__ int start_at(const lm_verify_params& P, int s) {
  const int32_t* w = (const int32_t*)P.q_starts + ((int64_t)s << P.starts64);
  const int lo = w[0], up = w[P.starts64], hi = P.starts64 ? up : lo >> 31;
  const int v = hi < 0 ? 0 : hi > 0 || (uint32_t)lo > (uint32_t)P.rows ? P.rows : lo;
  return s == 0 ? 0 : v;
}

// How many drafts sequence s has, from row r0 on; under 0: it has no row.  Rows from the last start on are padding,
// of which the first launch leaves nothing: where starts fall, no sequence reads there.
__device__ __forceinline__ int drafts_of(const lm_verify_params& P, int s, int r0) {
  const int end = start_at(P, s + 1), last = start_at(P, P.seqs);
  return (end < last ? end : last) - r0 - 1;
}

__device__ __forceinline__ void put_token(const lm_verify_params& P, int64_t r, int64_t token) {
  if (P.ids64)
    ((int64_t*)P.tokens)[r] = token;
  else
    ((int32_t*)P.tokens)[r] = (int32_t)token;
}

// N x 8 values of a row, from column j on and every `step` further; `fill` behind its end.
template <int N>
__device__ __forceinline__ void get_columns(const void* row, int j, int step, int n, int f32, int vec, float fill,
                                            float (&v)[N][8]) {
#pragma unroll
  for (int u = 0; u < N; ++u) {
    if (j + u * step < n) {
      get8(row, j + u * step, n, f32, vec, fill, v[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = fill;
    }
  }
}

// A wave's part of a row, 2048 logits: the largest and the sum of exponentials against it, a NaN
// where one is among them or the largest is infinite, zero where all are minus infinity.  Greedily
// where the largest is first, and one in place of the sum.  (Waves go their own ways: with the
// largest of a workgroup's 4096, two barriers and every row's place of the largest it took
// 19 us where it takes 16.)
constexpr int kPartEach = LM_VERIFY_PART / (8 * 64);
__device__ __forceinline__ void verify_rows(const lm_verify_params& P) {
  const int id = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (kVerifyThreads / 64) + (threadIdx.x >> 6)));
  const int r = id / P.parts, part = id - r * P.parts;
  if (r >= P.rows) return;
  const int lane = threadIdx.x & 63;
  if (r >= start_at(P, P.seqs)) {  // behind the last sequence
    if (part == 0 && lane == 0) put_token(P, r, -1);
    return;
  }
  const int base = part * LM_VERIFY_PART + 8 * lane;
  float v[kPartEach][8];
  get_columns(row_of(P.logits, P.logits_ld, r, P.logits_f32), base, 512, P.vocab, P.logits_f32, P.logits_vec, kNegInf,
              v);
  float top = kNegInf;
  bool odd = false;  // a NaN
#pragma unroll
  for (int u = 0; u < kPartEach; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      odd = odd || v[u][i] != v[u][i];
      top = fmaxf(top, v[u][i]);
    }
  int at = P.vocab;
  if (P.greedy) {
#pragma unroll
    for (int u = kPartEach - 1; u >= 0; --u)
#pragma unroll
      for (int i = 7; i >= 0; --i) at = v[u][i] == top ? base + 512 * u + i : at;
    at = top == kNegInf ? P.vocab : at;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) larger(top, at, __shfl_xor(top, m), __shfl_xor(at, m));
  } else {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
  }
  odd = __any(odd) || top == __builtin_inff();
  double sum = top == kNegInf ? 0.0 : 1.0;
  if (!P.greedy && top != kNegInf && !odd) {
    sum = 0;
#pragma unroll
    for (int u = 0; u < kPartEach; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += exp2_neg(((double)v[u][i] - (double)top) * P.scale_log2);
    sum = wave_sum(sum);
  }
  if (lane == 0) {
    P.part_top[id] = top;
    P.part_at[id] = at;
    P.part_sum[id] = odd ? (double)__builtin_nanf("") : sum;
  }
}

// A row's largest logit, where it is first, and its sum of exponentials, by 16 lanes side by side.
struct RowStats {
  float top;
  int at;
  double sum;
};
__device__ __forceinline__ RowStats row_stats(const lm_verify_params& P, int64_t r) {
  const int lane = threadIdx.x & 15;
  const int64_t o = r * P.parts;
  RowStats R = {kNegInf, P.vocab, 0};
  for (int i = lane; i < P.parts; i += 16) larger(R.top, R.at, P.part_top[o + i], P.part_at[o + i]);
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) larger(R.top, R.at, __shfl_xor(R.top, m), __shfl_xor(R.at, m));
  for (int i = lane; i < P.parts; i += 16) {
    const float t = P.part_top[o + i];
    // (of a part without a logit: zero, or a NaN)
    R.sum = __builtin_fma(P.part_sum[o + i], t == kNegInf ? 1.0 : exp2_neg(((double)t - (double)R.top) * P.scale_log2),
                          R.sum);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) R.sum += __shfl_xor(R.sum, m);
  return R;
}

__device__ __forceinline__ int64_t draft_of(const lm_verify_params& P, int r) {
  return index_at(P.ids, (int64_t)r + 1, P.ids64);
}

struct PickShared {
  RowStats stats[kSide];
  int first;
};

// How many of a sequence's drafts (rows from r0 on) stay, and the statistics of the row behind them, by the whole
// workgroup, 16 lanes a row.
__device__ __forceinline__ int accepted(const lm_verify_params& P, int r0, int drafts, RowStats* R, PickShared& S) {
  if (threadIdx.x == 0) S.first = drafts;
  __syncthreads();
  int base = 0;
  for (;; base += kSide) {
    const int i = base + (int)threadIdx.x / 16;
    if (i <= drafts) {
      // what the draft is compared by is requested with the statistics
      const int64_t d = i < drafts ? draft_of(P, r0 + i) : -1;
      const bool names = d >= 0 && d < P.vocab;
      float x = 0.f, q = 1.f, u = 0.f;
      if (names && !P.greedy) {
        x = get1(row_of(P.logits, P.logits_ld, r0 + i, P.logits_f32), (int)d, P.logits_f32);
        if (P.draft != nullptr) q = get1(row_of(P.draft, P.draft_ld, r0 + i, P.draft_f32), (int)d, P.draft_f32);
        u = P.uniforms[2 * (int64_t)(r0 + i)];
      }
      const RowStats mine = row_stats(P, r0 + i);
      bool stays = false;
      if (names)
        stays = P.greedy ? d == mine.at && mine.sum > 0  // a NaN is not
                         : (double)u * (double)q <
                               exp2_neg(((double)x - (double)mine.top) * P.scale_log2) / mine.sum;
      if ((threadIdx.x & 15) == 0) {
        S.stats[threadIdx.x / 16] = mine;
        if (!stays) atomicMin(&S.first, i);
      }
    }
    __syncthreads();
    if (S.first < base + kSide) break;  // at the latest behind the last draft
    __syncthreads();                    // the statistics have been passed over
  }
  *R = S.stats[S.first - base];
  return S.first;
}

// The weights that a token of row r is taken by: those of p - q times the row's sum of exponentials,
// or of p where `draft` is NULL, without the column `gone`.
struct Weights {
  const char *row, *draft;
  int gone;
  double top, sum;
};
__device__ __forceinline__ Weights weights_of(const lm_verify_params& P, int r, bool swapped, const RowStats& R) {
  Weights W;
  W.row = row_of(P.logits, P.logits_ld, r, P.logits_f32);
  W.draft = swapped && P.draft != nullptr ? row_of(P.draft, P.draft_ld, r, P.draft_f32) : nullptr;
  W.gone = -1;
  if (swapped && P.draft == nullptr) {
    const int64_t d = draft_of(P, r);
    W.gone = d >= 0 && d < P.vocab ? (int)d : -1;
  }
  W.top = (double)R.top;
  W.sum = R.sum;
  return W;
}
// e: the exponentials, w: the weights, of eight columns from j on
__device__ __forceinline__ void weights8(const lm_verify_params& P, const Weights& W, int j, const float (&v)[8],
                                         const float (&q)[8], double (&e)[8], double (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    e[i] = exp2_neg(((double)v[i] - W.top) * P.scale_log2);
    w[i] = W.draft != nullptr ? fmax(__builtin_fma(-W.sum, (double)q[i], e[i]), 0.0) : e[i];
    w[i] = j + i == W.gone ? 0.0 : w[i];
  }
}

constexpr int kPieces = LM_VERIFY_SLICE / LM_VERIFY_PIECE;  // of a workgroup
static_assert(LM_VERIFY_PIECE == 8 * 64, "a piece is a wave's values");

// A stretch of the row that a sequence's token is taken from: its pieces' sums.
__device__ __forceinline__ void verify_pieces(const lm_verify_params& P, PickShared& S) {
  const int s = blockIdx.x / P.slices, slice = blockIdx.x - s * P.slices;
  const int r0 = start_at(P, s), drafts = drafts_of(P, s, r0);
  if (drafts < 0) return;
  RowStats R;
  const int a = accepted(P, r0, drafts, &R, S);
  if (slice == 0 && threadIdx.x == 0) {
    P.chosen[s].sum = R.sum;
    P.chosen[s].top = R.top;
    P.chosen[s].accepted = a;
  }
  const Weights W = weights_of(P, r0 + a, a < drafts, R);
  constexpr int kEach = LM_VERIFY_SLICE / (8 * kVerifyThreads);
  const int j = slice * LM_VERIFY_SLICE + 8 * (int)threadIdx.x;
  float v[kEach][8], q[kEach][8];
  get_columns(W.row, j, 8 * kVerifyThreads, P.vocab, P.logits_f32, P.logits_vec, kNegInf, v);
  if (W.draft != nullptr) get_columns(W.draft, j, 8 * kVerifyThreads, P.vocab, P.draft_f32, P.draft_vec, 0.f, q);
  double* pieces = P.piece_sum + 2 * (int64_t)s * P.slices * kPieces;
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    double e[8], w[8], se = 0, sw = 0;
    weights8(P, W, j + u * 8 * kVerifyThreads, v[u], q[u], e, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      se += e[i];
      sw += w[i];
    }
    se = wave_sum(se);
    sw = wave_sum(sw);
    const int piece = slice * kPieces + u * (kVerifyThreads / 64) + (threadIdx.x >> 6);
    if ((threadIdx.x & 63) == 0) {
      pieces[2 * piece] = sw;
      pieces[2 * piece + 1] = se;
    }
  }
}

// A token by the number u from a sequence's pieces (which: their weights, or 1 their exponentials), by one wave; -1
// where they sum to nothing.
__device__ __forceinline__ int sample(const lm_verify_params& P, Weights W, const double* pieces, int which, double u) {
  const int lane = threadIdx.x & 63, n = P.slices * kPieces;
  if (which == 1) {
    W.draft = nullptr;
    W.gone = -1;
  }
  // every lane a stretch of pieces
  const int each = (n + 63) / 64;
  double mine = 0;
  for (int i = 0; i < each; ++i) {
    const int p = lane * each + i;
    if (p < n) mine += pieces[2 * p + which];
  }
  double upto = mine;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double x = __shfl_up(upto, m);
    upto += lane >= m ? x : 0;
  }
  const double goal = u * __shfl(upto, 63);
  // the first lane over the goal; what rounding leaves over is for the last with a weight
  const uint64_t heavy = __ballot(mine > 0), over = __ballot(mine > 0 && upto > goal);
  if (heavy == 0) return -1;
  const int who = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(heavy);
  double sum = __shfl(upto - mine, who), at = sum;
  int piece = -1;
  for (int i = 0; i < each; ++i) {  // every lane the same
    const int p = who * each + i;
    const double w = p < n ? pieces[2 * p + which] : 0;
    if (w > 0) {
      piece = p;
      at = sum;
      if (sum + w > goal) break;
    }
    sum += w;
  }
  const int j = piece * LM_VERIFY_PIECE + 8 * lane;
  double e[8], w[8], own = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 0;
  if (j < P.vocab) {
    float v[8], q[8];
    get8(W.row, j, P.vocab, P.logits_f32, P.logits_vec, kNegInf, v);
    if (W.draft != nullptr) get8(W.draft, j, P.vocab, P.draft_f32, P.draft_vec, 0.f, q);
    weights8(P, W, j, v, q, e, w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) own += w[i];
  double end = own;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double x = __shfl_up(end, m);
    end += lane >= m ? x : 0;
  }
  const uint64_t some = __ballot(own > 0), past = __ballot(own > 0 && at + end > goal);
  if (some == 0) return -1;
  const int in = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  double run = at + (end - own);
  int token = -1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (w[i] > 0 && (token < 0 || run <= goal)) token = j + i;  // the sum in front is not over the goal yet
    run += w[i];
  }
  return __shfl(token, in);
}

// The tokens of a sequence, by one wave; greedily by a workgroup, from the rows alone.
__device__ __forceinline__ void verify_pick(const lm_verify_params& P, PickShared& S) {
  const int s = blockIdx.x;
  const int r0 = start_at(P, s), drafts = drafts_of(P, s, r0);
  if (drafts < 0) {
    if (threadIdx.x == 0) P.counts[s] = 0;
    return;
  }
  RowStats R;
  int a, token = -1;
  if (P.greedy) {
    a = accepted(P, r0, drafts, &R, S);
    token = R.sum > 0 ? R.at : -1;  // a NaN is not
  } else {
    const lm_verify_choice C = P.chosen[s];
    a = C.accepted;
    R.top = C.top;
    R.sum = C.sum;
    if (R.sum > 0) {
      const Weights W = weights_of(P, r0 + a, a < drafts, R);
      const double goal = (double)P.uniforms[2 * (int64_t)(r0 + a) + 1];
      const double* pieces = P.piece_sum + 2 * (int64_t)s * P.slices * kPieces;
      token = sample(P, W, pieces, 0, goal);
      if (token < 0) token = sample(P, W, pieces, 1, goal);  // of p - q nothing is left
    }
  }
  for (int i = threadIdx.x; i <= drafts; i += blockDim.x)
    put_token(P, r0 + i, i < a ? draft_of(P, r0 + i) : i == a ? token : -1);
  if (threadIdx.x == 0) P.counts[s] = token < 0 ? a : a + 1;
}

}  // namespace

extern "C" __global__ void __launch_bounds__(LM_SLOTS_THREADS) attnres_paged_slots(lm_slots_params P) {
  __shared__ SlotShared S;
  paged_slots(P, S);
}
extern "C" __global__ void __launch_bounds__(LM_SLOTS_THREADS) attnres_paged_release(lm_slots_params P) {
  __shared__ SlotShared S;
  paged_release(P, S);
}
extern "C" __global__ void __launch_bounds__(256) attnres_paged_write(lm_write_params P) { paged_write(P); }
extern "C" __global__ void __launch_bounds__(kVerifyThreads) attnres_verify_rows(lm_verify_params P) { verify_rows(P); }
extern "C" __global__ void __launch_bounds__(kVerifyThreads) attnres_verify_pieces(lm_verify_params P) {
  __shared__ PickShared S;
  verify_pieces(P, S);
}
// 64 threads, or kVerifyThreads greedily
extern "C" __global__ void __launch_bounds__(kVerifyThreads) attnres_verify_pick(lm_verify_params P) {
  __shared__ PickShared S;
  verify_pick(P, S);
}
