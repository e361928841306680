// What the plan of a ragged step (ragged_plan.cu) and the attention that runs it (ragged_attn.cu) agree on.
#pragma once

#include "common.cuh"

// Rows of one tensor-core tile and keys of one K/V tile; a CTA holds two row tiles.
constexpr int kRagTile = 128;

// One entry of the attention's work list: the new tokens [row0, row0 + n_tok) of sequence `seq`, whose first
// one stands at position pos0, against the K/V tiles [kt0, kt1) of 128 tokens each. slot < 0: the item covers all
// its keys and writes the output; otherwise its partial softmax state goes to workspace slot `slot`.
struct __align__(16) RagItem {
  int32_t seq, row0, n_tok, pos0, kt0, kt1, slot, kv_len;
};
// An item split over the key axis: its partials are slots [slot0, slot0 + parts).
struct __align__(16) RagMerge {
  int32_t row0, n_tok, slot0, parts;
};

// Sizes that follow from a plan's capacities alone, so that the host can size grids and workspaces without
// knowing the lengths.
struct RagShape {
  int group, tok_tile, tok_item;      // query heads per K/V head; tokens per row tile and per item
  int64_t max_items, max_list;        // items without splits; entries with splits
  int max_merges;                     // items that can be split
  int max_slots;                      // partial slots
  int64_t list_off, merge_off, total; // byte offsets in the plan's work area
};

// The first words of the work area. The list's places and items follow from the sizes that the plan was made for, so it
// leaves them here, and the attention runs no list that was made for others.
struct __align__(16) RagHead {
  int32_t n_list, n_merge, rows, max_blocks;
  int32_t max_rows, b, hq, hkv;
};
__device__ __forceinline__ bool rag_made_for(const RagHead& h, int64_t max_rows, int b, int hq, int hkv, int max_blocks) {
  return h.max_rows == max_rows && h.b == b && h.hq == hq && h.hkv == hkv && h.max_blocks == max_blocks;
}

// Splitting rule (see ragged_plan.cu): an item of n tiles gives at most ceil(n / share) entries, where share is at least
// ceil(all tiles / max_merges) (and at least 2; it is lengthened where the entries then fit one wave). So fewer than
// max_merges items are split, all items together give at most max_items + max_merges entries, and the split ones take
// fewer than 2 * max_merges slots.
static inline bool rag_shape(int64_t max_rows, int b, int hq, int hkv, int d, int sms, RagShape* s) {
  if (max_rows < 0 || max_rows > (1 << 26) || b < 0 || hq <= 0 || hkv <= 0 || hq % hkv || hq / hkv > 16) return false;
  if (d != 32 && d != 64 && d != 128) return false;
  s->group = hq / hkv;
  s->tok_tile = kRagTile / s->group;
  s->tok_item = 2 * s->tok_tile;
  s->max_items = max_rows / s->tok_item + b;
  if (s->max_items > max_rows) s->max_items = max_rows;
  s->max_merges = sms / hkv > 1 ? sms / hkv : 1;
  s->max_slots = 2 * s->max_merges;
  s->max_list = s->max_items + s->max_merges;
  s->list_off = 64;
  s->merge_off = s->list_off + s->max_list * (int64_t)sizeof(RagItem);
  s->total = s->merge_off + (int64_t)s->max_merges * (int64_t)sizeof(RagMerge);
  return true;
}

int mg_sm_count();  // multiprocessors of the current device (ragged_plan.cu)
