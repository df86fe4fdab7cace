/*
 * How paged attention's work is dealt out, in what the host that sizes a launch (serving_capi.cpp) and
 * the kernels that find their own work in it (paged_attention_kernels.hip) have in common.
 *
 * Included by g++ (host) and by hipcc (device) alike.
 */
#ifndef KOTODAMA_AMD_PAGED_SCHEDULE_H
#define KOTODAMA_AMD_PAGED_SCHEDULE_H

#include <math.h>
#include <stdint.h>

#include "lm_params.h"

#ifdef __HIPCC__
#define LM_BOTH __host__ __device__ __forceinline__
#else
#define LM_BOTH inline
#endif

namespace {

// ---------------------------------------------------------------- launch --

// Keys that one workgroup takes of a tile without splitting it: a block of 128 costs it some 1.2 us, the
// launch that joins parts 4 to 5 (one token over 512 keys, 32/8 heads of 128: 11.7 us whole, 8.2 + 4.2 in
// parts; over 1024 keys 17.2 and 8.0 + 5.1).
constexpr int64_t kWholeKeys = 512;
// Waves of 32 rows per CU from which rows are taken 128 at a time; twice as many where a CU has room for one
// workgroup.  (bf16, heads of 128: 2 prompts of 2048, 8/4 heads, 54 us, 32 at a time 67; 1100 tokens, 32/8 heads,
// 38 and 59; half as many rows: 55 and 34, 18 and 14.  fp32: 1100 behind 7092, 32/8 heads, 1770 and 1490.)
constexpr int kWideWaves = 4;

// What the launches and the workspace of a call go by.
struct PagedPlan {
  bool wide = false, split = false;
  int target = 0, part_rows = 0, turn = 0;
  int64_t slots = 0, grid = 0, notes = 0;  // of all key heads
  int64_t at_ml = 0, at_notes = 0, bytes = 0;
};

// On a card of `cus`; false where the key blocks are too many for 32 bits.
inline bool paged_plan(int cus, int64_t tokens, int seqs, int heads, int kv_heads, int head_dim, bool f32,
                       int64_t capacity, PagedPlan* p) {
  const int64_t rows = tokens * (heads / kv_heads);
  // Workgroups to deal out to: two a CU, or one where the LDS has no room for two (64 ragged fp32 sequences of
  // up to 2048 keys, 8/4 heads of 128: 90 us, 97 with two rounds of them).  Heads of up to 64 in bf16 have room
  // for four, but shorter stretches cost more than they hide (64 sequences of up to 4096 keys: 39 us against 34).
  const int64_t at_once = (int64_t)cus * (head_dim > 64 && f32 ? 1 : 2);
  p->wide = rows / 32 * kv_heads >= (int64_t)cus * (at_once > cus ? kWideWaves : 2 * kWideWaves);
  p->split = capacity > kWholeKeys;
  if (p->wide) {
    p->target = (int)at_once;
    // where all tiles run at once, workgroups as many apart as there are CUs share one
    if (rows / 128 * kv_heads <= at_once && at_once > cus) p->turn = cus / kv_heads;
    // tiles: every sequence may end inside one; the rows behind the last sequence are one more
    const int64_t tiles = rows / 128 + seqs + 1, share = (p->target + kv_heads - 1) / kv_heads;
    // a split tile's parts are under twice its blocks over a part's most, and all those blocks at most the target's
    // share
    p->slots = p->split ? (2 * share + 8) * kv_heads : 0;
    p->grid = (tiles + (p->split ? share + 8 : 0)) * kv_heads;
    p->notes = p->slots;
    p->part_rows = 128;
  } else {
    if ((rows / 32 + seqs + 1) * ((capacity + 127) / 128) > INT32_MAX) return false;
    const int64_t tiles = rows / 32 + seqs + 1;
    p->target = !p->split ? (int)tiles : at_once > kv_heads ? (int)(at_once / kv_heads) : 1;
    p->grid = (int64_t)p->target * kv_heads;
    p->slots = p->split ? 2 * p->grid : 0;  // each workgroup goes on with a tile and begins one
    p->notes = p->split ? p->grid : 0;
    p->part_rows = rows < 32 ? (int)rows : 32;
  }
  const int64_t lines = p->slots * p->part_rows;
  p->at_ml = lines * head_dim * 4;
  p->at_notes = p->at_ml + (lines * 8 + 15) / 16 * 16;
  p->bytes = p->at_notes + p->notes * (int64_t)sizeof(lm_paged_note);
  return true;
}

// ----------------------------------------------------------------- tiles --

// One sequence's share of the call: its tokens, keys and tiles of rows.
struct Share {
  int first, count;  // new tokens
  int kv_len;
  int rows, tiles;
  bool narrow;
  // the tokens lo .. hi-1, over kv_len keys
  LM_BOTH void set(int lo, int hi, int keys, int group, bool wide) {
    first = lo;
    count = hi > lo ? hi - lo : 0;
    kv_len = keys;
    rows = count * group;
    narrow = !wide || rows <= 32;
    tiles = narrow ? (rows + 31) >> 5 : (rows + 127) >> 7;
  }
};

// A tile's work: blocks of 32 keys that a wave works on, as if its rows saw all keys of the sequence.  (A chunk's
// do but for the chunk itself; tiles of a prompt from its start work on half of them on the average, and count for
// twice their time in the cut.)
LM_BOTH int blocks_of(const Share& a) { return a.narrow ? (a.kv_len + 127) >> 7 : ((a.kv_len + 63) >> 6) * 2; }

// Its parts of at most `most` such blocks, and the key blocks of one.
struct Split {
  int n, parts, per;
  LM_BOTH Split(const Share& a, int most) {
    per = a.narrow ? most : (most + 1) >> 1;
    n = a.narrow ? (a.kv_len + 127) >> 7 : (a.kv_len + 63) >> 6;
    parts = n <= per ? 1 : (n + per - 1) / per;
  }
};

// The most blocks of a part.  Tried are the longest tile's, halves, thirds .. sevenths of them, and an equal share
// for `target` workgroups; of those whose parts the launch has room for (whole tiles always are) the one
// whose last workgroup should end first: rounds of the longest part, or all work and a part
// behind it; a workgroup that has its CU for itself takes 0.6 of the time.  A part costs some 8 blocks'
// time to begin and end, the join as much and 24 where it reads `target` parts' sums (2 prompts of 2048,
// 8/4 heads of 128: 55 us whole, 83 in halves; 1024 behind 15360, 32/8 heads: 309 in halves).  Every workgroup
// comes to the same.  (With the equal share alone, tiles a little fewer than workgroups were all cut in unequal
// halves: 1536 tokens behind 14848, 632 us where it takes 440; 3 prompts of 2048, 125 and 58.)
constexpr int kCuts = 8;
constexpr float kPartCost = 8.f, kAlone = 0.6f, kJoinCost = 24.f;
struct Cuts {
  float top, target, heads, each;  // the longest tile's blocks; all work over the target
  int longest;
  LM_BOTH Cuts(float work, float top_, int target_, int heads_)
      : top(top_), target((float)target_), heads((float)heads_), each(work * heads / target),
        longest(top < 1.f ? 1 : top < 0x1p24f ? (int)top : (int)top + 4) {}  // (a float's rounding)
  LM_BOTH bool many() const { return each >= 8.f * top; }  // tiles enough to even out: none is cut
  LM_BOTH int most(int j) const {
    const float c = ceilf(j + 1 < kCuts ? top / (float)(j + 1) : each);
    return c < 1.f ? 1 : c < top ? (int)c : longest;
  }
  // What the cut into parts of `most` costs that makes so many of a head, `shared` of them of split tiles; infinite
  // where a head's `slots` or `all` workgroups do not hold them.
  LM_BOTH float cost(int most, float parts, float shared, bool two, int slots, int all) const {
    const float n = parts * heads, part = (float)most + kPartCost;
    float c = fminf(ceilf(n / target) * part, each + part);
    if (two && 2.f * n <= target) c = kAlone * part;
    c += shared > 0.f ? kPartCost + kJoinCost * shared * heads / target : 0.f;
    const bool room = shared == 0.f || (shared <= (float)slots && parts <= (float)all);
    return room ? c : INFINITY;
  }
};

// Of the notes of a head's slots, its parts write the first `used`.  The others are cleared, or the join would take up
// what an earlier call has left there: by all of the head's workgroups in turn, as a cut may leave none without a
// part.
template <typename F>
LM_BOTH void for_unused_notes(int w, int all, int used, int slots, F clear) {
  for (int i = used + w; i < slots; i += all) clear(i);
}

}  // namespace

#endif  // KOTODAMA_AMD_PAGED_SCHEDULE_H
