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
// sums and the pages, each waiting for the one before.

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
    S.first[tid] = granted ? (int32_t)(count - 1 - (upto - need)) : kRefused;  // of the new pages in the free list
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
// Which token a number falls to depends on sums over the whole vocabulary
// next to a border, so the chosen row's are taken in 64 bits.  For the drafts' test one
// probability each is enough: 32-bit exponentials, whose sum errs by
// under 1e-5, and a row nearer to its border than that is summed again in 64 bits.

constexpr int kVerifyThreads = 256;
constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / 64;
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

// (top, at) of the larger value, the lower index where both are the same.
__device__ __forceinline__ void larger(float& top, int& at, float t, int a) {
  const bool take = t > top || (t == top && a < at);
  top = take ? t : top;
  at = take ? a : at;
}

// The tokens' rows lie in the call: starts are taken into it.
__device__ __forceinline__ int start_at(const lm_verify_params& P, int s) {
  const int64_t v = s == 0 ? 0 : index_at(P.q_starts, s, P.starts64);
  return v < 0 ? 0 : v > P.rows ? P.rows : (int)v;
}

// First pass: of LM_VERIFY_SLICE logits the largest, where it is first, and the sum of exponentials against it.
__device__ __forceinline__ void verify_rows(const lm_verify_params& P, float* tops, int* ats, double* sums) {
  const int r = blockIdx.x / P.slices, slice = blockIdx.x - r * P.slices;
  if (r >= start_at(P, P.seqs)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* row = row_of(P.logits, P.logits_ld, r, P.logits_f32);
  constexpr int U = LM_VERIFY_SLICE / (8 * kVerifyThreads);
  const int first = slice * LM_VERIFY_SLICE;
  float v[U][8];
  float top = kNegInf;
  int at = P.vocab;
  bool odd = false;  // a NaN
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int j = first + 8 * (u * kVerifyThreads + (int)threadIdx.x);
    if (j < P.vocab) {
      get8(row, j, P.vocab, P.logits_f32, P.logits_vec, kNegInf, v[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = kNegInf;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int j = first + 8 * (u * kVerifyThreads + (int)threadIdx.x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      odd = odd || v[u][i] != v[u][i];
      if (v[u][i] > top) {
        top = v[u][i];
        at = j + i;
      }
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) larger(top, at, __shfl_xor(top, m), __shfl_xor(at, m));
  if (lane == 0) {
    tops[wave] = top;
    ats[wave] = at;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerifyThreads / 64; ++w) larger(top, at, tops[w], ats[w]);
  const float ref = top == kNegInf ? 0.f : top;
  const float k = P.inv_temp * 1.44269504088896340736f;
  float part = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) part += __builtin_amdgcn_exp2f((v[u][i] - ref) * k);
  double sum = wave_sum((double)(odd ? __builtin_nanf("") : part));
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < kVerifyThreads / 64; ++w) sum += sums[w];
    const int64_t o = (int64_t)r * P.slices + slice;
    P.part_top[o] = top;
    P.part_at[o] = at;
    P.part_sum[o] = sum;
  }
}

struct PickShared {
  double sums[kPickWaves];
  double pieces[LM_VERIFY_MAX_PIECES];
  int first, token;
};

// Sum over the workgroup, to every thread, in a fixed order.
__device__ __forceinline__ double block_sum(double v, PickShared& S) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) S.sums[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0;
#pragma unroll
  for (int i = 0; i < kPickWaves; ++i) t += S.sums[i];
  return t;
}

// The sum of a row's exponentials against `top`, in 64 bits.
__device__ __forceinline__ double row_sum(const lm_verify_params& P, const char* row, float top, PickShared& S) {
  double t = 0;
  for (int j = 8 * (int)threadIdx.x; j < P.vocab; j += 8 * kPickThreads) {
    float v[8];
    get8(row, j, P.vocab, P.logits_f32, P.logits_vec, kNegInf, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) t += exp(((double)v[i] - (double)top) * P.inv_temp64);
  }
  return block_sum(t, S);
}

// A wave's 512 values from `j0`: each lane's eight weights.
__device__ __forceinline__ void weights8(const lm_verify_params& P, const char* row, const char* draft, int gone, int j,
                                         float top, double inv, double (&w)[8]) {
  float v[8], q[8];
  get8(row, j, P.vocab, P.logits_f32, P.logits_vec, kNegInf, v);
  if (draft != nullptr) get8(draft, j, P.vocab, P.draft_f32, P.draft_vec, 0.f, q);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    double p = exp(((double)v[i] - (double)top) * P.inv_temp64) * inv;
    if (draft != nullptr) {
      p -= (double)q[i];
      p = p < 0 ? 0 : p;  // a NaN stays one
    }
    w[i] = j + i == gone ? 0 : p;
  }
}

// A token from the row's weights by the number u; -1 where they have no sum, none where it is zero.
constexpr int kNoWeight = -2;
__device__ __forceinline__ int sample(const lm_verify_params& P, const char* row, const char* draft, int gone, float top,
                                      double inv, double u, PickShared& S) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int pieces = (P.vocab + LM_VERIFY_PIECE - 1) / LM_VERIFY_PIECE;
  for (int p = wave; p < pieces; p += kPickWaves) {
    const int j = p * LM_VERIFY_PIECE + 8 * lane;
    double t = 0;
    if (j < P.vocab) {
      double w[8];
      weights8(P, row, draft, gone, j, top, inv, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) t += w[i];
    }
    t = wave_sum(t);
    if (lane == 0) S.pieces[p] = t;
  }
  __syncthreads();
  if (wave == 0) {
    // every lane a stretch of pieces
    const int each = (pieces + 63) / 64;
    double mine = 0;
    for (int i = 0; i < each; ++i) {
      const int p = lane * each + i;
      if (p < pieces) mine += S.pieces[p];
    }
    double upto = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const double x = __shfl_up(upto, m);
      upto += lane >= m ? x : 0;
    }
    const double total = __shfl(upto, 63);
    const double goal = u * total;
    int token = !(total >= 0) || total > 1e300 ? -1 : total == 0 ? kNoWeight : -3;
    if (token == -3) {
      // the last lane with a weight takes what rounding leaves over
      const uint64_t heavy = __ballot(mine > 0), over = __ballot(mine > 0 && upto > goal);
      const int who = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(heavy);
      double sum = __shfl(upto - mine, who);
      int piece = -1;
      double at = sum;
      for (int i = 0; i < each; ++i) {  // every lane the same
        const int p = who * each + i;
        const double w = p < pieces ? S.pieces[p] : 0;
        if (w > 0) {
          piece = p;
          at = sum;
          if (sum + w > goal) break;
        }
        sum += w;
      }
      double w[8];
      const int j = piece * LM_VERIFY_PIECE + 8 * lane;
      double own = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 0;
      if (j < P.vocab) weights8(P, row, draft, gone, j, top, inv, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) own += w[i];
      double end = own;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const double x = __shfl_up(end, m);
        end += lane >= m ? x : 0;
      }
      const uint64_t some = __ballot(own > 0), past = __ballot(own > 0 && at + end > goal);
      const int lane2 = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
      double run = at + (end - own);
      int mineTok = -1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool before = mineTok < 0 || run <= goal;  // not past the goal yet
        if (w[i] > 0 && before) mineTok = j + i;
        run += w[i];
      }
      token = __shfl(mineTok, lane2);
    }
    if (lane == 0) S.token = token;
  }
  __syncthreads();
  const int t = S.token;
  __syncthreads();
  return t;
}

// A row's largest logit, where it is first, and the sum of its exponentials (the first pass's), to every lane.
struct RowStats {
  float top;
  int at;
  double sum;
};
__device__ __forceinline__ RowStats row_stats(const lm_verify_params& P, int64_t r) {
  const int lane = threadIdx.x & 63;
  RowStats R = {kNegInf, P.vocab, 0};
  for (int i = lane; i < P.slices; i += 64) larger(R.top, R.at, P.part_top[r * P.slices + i], P.part_at[r * P.slices + i]);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) larger(R.top, R.at, __shfl_xor(R.top, m), __shfl_xor(R.at, m));
  for (int i = lane; i < P.slices; i += 64) {
    const float t = P.part_top[r * P.slices + i];
    const double sum = P.part_sum[r * P.slices + i];
    R.sum += t == kNegInf ? sum : sum * exp(((double)t - (double)R.top) * P.inv_temp64);  // of none: zero, or a NaN
  }
  R.sum = wave_sum(R.sum);
  return R;
}

// Second pass: a workgroup per sequence, and one for the rows behind the last.
__device__ __forceinline__ void verify_pick(const lm_verify_params& P, PickShared& S) {
  const int tid = threadIdx.x, wave = tid >> 6, s = blockIdx.x;
  auto put = [&](int r, int64_t token) {
    if (P.ids64)
      ((int64_t*)P.tokens)[r] = token;
    else
      ((int32_t*)P.tokens)[r] = (int32_t)token;
  };
  const int r0 = start_at(P, s);
  if (s == P.seqs) {
    for (int64_t r = r0 + tid; r < P.rows; r += kPickThreads) put((int)r, -1);
    return;
  }
  const int next = start_at(P, s + 1), drafts = next - r0 - 1;
  if (drafts < 0) {
    if (tid == 0) P.counts[s] = 0;
    return;
  }
  auto draft_of = [&](int i) { return index_at(P.ids, r0 + i + 1, P.ids64); };
  auto weight_of = [&](int i, int64_t d) {  // the draft's own probability
    return P.draft == nullptr ? 1.0 : (double)get1(row_of(P.draft, P.draft_ld, r0 + i, P.draft_f32), (int)d, P.draft_f32);
  };
  // the first draft that does not stay
  int from = 0, a = drafts;
  while (from < drafts) {
    if (tid == 0) S.first = 2 * drafts;
    __syncthreads();
    for (int i = from + wave; i < drafts; i += kPickWaves) {
      const int64_t d = draft_of(i);
      bool stays = false, near = false;
      if (d >= 0 && d < P.vocab) {
        const RowStats R = row_stats(P, r0 + i);
        if (P.greedy) {
          stays = d == R.at && R.sum > 0;  // a NaN is not
        } else {
          const float x = get1(row_of(P.logits, P.logits_ld, r0 + i, P.logits_f32), (int)d, P.logits_f32);
          const double p = exp(((double)x - (double)R.top) * P.inv_temp64) / R.sum;
          const double need = (double)P.uniforms[2 * (int64_t)(r0 + i)] * weight_of(i, d);
          stays = need < p;
          near = fabs(need - p) <= 1e-4 * p;
        }
      }
      if (!stays || near) {
        if ((tid & 63) == 0) atomicMin(&S.first, 2 * i + (near ? 1 : 0));
        break;
      }
    }
    __syncthreads();
    const int found = S.first;
    __syncthreads();
    a = found >> 1;
    if (a == drafts || (found & 1) == 0) break;
    const char* row = row_of(P.logits, P.logits_ld, r0 + a, P.logits_f32);
    const RowStats R = row_stats(P, r0 + a);
    const double sum = row_sum(P, row, R.top, S);
    const int64_t d = draft_of(a);
    const double p = exp(((double)get1(row, (int)d, P.logits_f32) - (double)R.top) * P.inv_temp64) / sum;
    if (!((double)P.uniforms[2 * (int64_t)(r0 + a)] * weight_of(a, d) < p)) break;
    from = a + 1;
    a = drafts;
  }
  // the token in its place, or the one behind them all
  const RowStats R = row_stats(P, r0 + a);
  const char* row = row_of(P.logits, P.logits_ld, r0 + a, P.logits_f32);
  int token;
  if (P.greedy) {
    token = R.sum > 0 ? R.at : -1;  // a NaN is not
  } else {
    const double inv = 1.0 / row_sum(P, row, R.top, S), u = (double)P.uniforms[2 * (int64_t)(r0 + a) + 1];
    const bool swapped = a < drafts;
    const char* draft = swapped && P.draft != nullptr ? row_of(P.draft, P.draft_ld, r0 + a, P.draft_f32) : nullptr;
    const int64_t d = swapped ? draft_of(a) : -1;
    const int gone = swapped && P.draft == nullptr && d >= 0 && d < P.vocab ? (int)d : -1;
    token = sample(P, row, draft, gone, R.top, inv, u, S);
    if (token == kNoWeight) token = sample(P, row, nullptr, -1, R.top, inv, u, S);
  }
  for (int i = tid; i <= drafts; i += kPickThreads) put(r0 + i, i < a ? draft_of(i) : i == a ? token : -1);
  if (tid == 0) P.counts[s] = token < 0 ? a : a + 1;
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
extern "C" __global__ void __launch_bounds__(kVerifyThreads) attnres_verify_rows(lm_verify_params P) {
  __shared__ float tops[kVerifyThreads / 64];
  __shared__ int ats[kVerifyThreads / 64];
  __shared__ double sums[kVerifyThreads / 64];
  verify_rows(P, tops, ats, sums);
}
extern "C" __global__ void __launch_bounds__(kPickThreads) attnres_verify_pick(lm_verify_params P) {
  __shared__ PickShared S;
  verify_pick(P, S);
}
