// Which notes a paged-attention call of many rows writes, counted on the CPU (test infrastructure, like the
// rest of oracle/; nothing in the library links it): the launch, the cut and the tiles of
// kotodama_amd/csrc/paged_schedule.h, dealt out workgroup by workgroup as paged_tiles does in
// kotodama_amd/csrc/paged_attention_kernels.hip.

#include <cstdint>
#include <vector>

#include "paged_schedule.h"

namespace {

int clamped(int64_t v, int64_t most) { return (int)(v < 0 ? 0 : v > most ? most : v); }

}  // namespace

// starts (seqs + 1) and lens (seqs) as the call has them.  cut: which of the kCuts cuts, or -1: the one that the call
// takes.  written (room entries): how often each note of a head is written, cleared ones among them.
// info: a head's workgroups, its parts, its notes, how many of them parts write, the cut.
// Returns 0; 1 where the call has few rows or is too large, 2 where `cut` has no room, 3 where `room` is too
// small, 4 where a part's notes lie outside.
extern "C" int paged_notes(int cus, int64_t tokens, int seqs, int heads, int kv_heads, int head_dim, int f32,
                           int64_t capacity, const int64_t* starts, const int64_t* lens, int cut, int32_t* written,
                           int room, int64_t* info) {
  PagedPlan plan;
  if (!paged_plan(cus, tokens, seqs, heads, kv_heads, head_dim, f32 != 0, capacity, &plan) || !plan.wide) return 1;
  const int slots = (int)(plan.slots / kv_heads), all = (int)(plan.grid / kv_heads);
  if (slots > room || plan.slots != plan.notes || plan.grid % kv_heads != 0) return 3;
  std::vector<Share> a(seqs + 1);
  float work = 0.f, top = 0.f;
  for (int s = 0; s <= seqs; ++s) {  // the last: the rows behind all sequences
    const int lo = s == 0 ? 0 : clamped(starts[s], tokens);
    const int hi = s < seqs ? clamped(starts[s + 1], tokens) : (int)tokens;
    a[s].set(lo, hi, s < seqs ? clamped(lens[s], capacity) : 0, heads / kv_heads, true);
    if (s == seqs) continue;
    const float n = a[s].tiles > 0 ? (float)blocks_of(a[s]) : 0.f;
    work += (float)a[s].tiles * n;
    top = top > n ? top : n;
  }
  const Cuts C(work, top, plan.target, kv_heads);
  auto count = [&](int most, float* parts, float* shared) {
    *parts = *shared = 0.f;
    for (const Share& x : a) {
      const Split sp(x, most);
      const float n = (float)x.tiles * (float)sp.parts;
      *parts += n;
      *shared += sp.parts > 1 ? n : 0.f;
    }
  };
  float costs[kCuts], parts, shared;
  int best = 0;
  for (int j = 0; j < kCuts; ++j) {
    count(C.most(j), &parts, &shared);
    costs[j] = C.cost(C.most(j), parts, shared, !(f32 && head_dim > 64), slots, all);
    if (costs[j] < costs[best]) best = j;
  }
  if (slots == 0 || C.many()) best = 0;
  if (cut >= 0) best = cut;
  if (isinf(costs[best])) return 2;
  const int most = C.most(best);
  count(most, &parts, &shared);
  const int used = (int)shared;
  info[0] = all;
  info[1] = (int64_t)parts;
  info[2] = slots;
  info[3] = used;
  info[4] = best;
  for (int i = 0; i < slots; ++i) written[i] = 0;
  for (int w = 0; w < all; ++w) {
    for_unused_notes(w, all, used, slots, [&](int i) { ++written[i]; });
    int64_t before = 0, at = 0;
    for (const Share& x : a) {
      const Split sp(x, most);
      const int64_t n = (int64_t)x.tiles * sp.parts;
      if (w - before < n) {
        const int i = (int)(w - before), rank = i / sp.parts, part = i - rank * sp.parts;
        if (sp.parts > 1) {
          const int64_t slot = at + (int64_t)rank * sp.parts + part;
          if (slot < 0 || slot >= slots) return 4;
          ++written[slot];
        }
        break;
      }
      before += n;
      at += sp.parts > 1 ? n : 0;
    }
  }
  return 0;
}
