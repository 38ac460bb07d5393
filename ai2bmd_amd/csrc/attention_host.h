// Host side shared by the fragment attention's launchers.
#pragma once
#include "attention.h"

namespace vsn {

constexpr int kMaxSlots = 1024;          // partial results of one query block
constexpr int kFewSlots = 32;
constexpr size_t kLdsPerCu = 160 * 1024;

// the work lists of one pass: `small` items are fragments of one tile, `pair` items of two (backward), `lone` items a wave
// each with tiles of its own, `coop` items a workgroup of four
struct AttnBlock {
  int col0, cols;
};
struct AttnPlanView {
  const AttnWork *small_work, *pair_work, *lone_work, *coop_work;
  int small, pair, lone, coop;
  int long_rows;  // whether an item has more than one tile of rows
  const AttnBlock* block;  // runs of columns of the lone and coop items
  int blocks;
  const AttnJoin* join;
  int joins, few;  // the first `few` of them have at most kFewSlots pieces
};

// Waves per workgroup where every wave has its own tiles: four, as far as LDS allows.  One each instead: 8 read-out rows over
// up to 17 882 atoms bf16 34.9 us (four: 28.4), 4096 fragments of 33 ... 64 rows bf16, dim 32, forward 157 us (144), four
// proteins f32 and one of 746 atoms bf16 equal; only at dim 128, where LDS holds few, one is better (the 4096 fragments f32,
// forward 1202 and 1278 us, bf16 466 and 476).
inline int lone_waves(size_t bytes) {
  int waves = 4;
  while (waves > 1 && waves * bytes > kLdsPerCu / 2) waves /= 2;
  return waves;
}

inline bool allow_lds(const void* kernel, size_t bytes) {
  if (bytes <= 64 * 1024 || hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess)
    return true;
  (void)hipGetLastError();
  return false;
}

// Waves per small fragment: one that walks all heads, so distances are computed once and positions' gradients need no
// joining - or, where the fragments alone would leave half of the 1024 SIMDs idle, one per key head.  8 heads of 32, both
// directions, one wave and one per key head: 512 fragments f32 115 and 94 us, bf16 90 and 78; 1024 fragments f32 equal, bf16 99
// and 103 (forward alone 25 and 23).
inline int small_groups(int items, int kv_heads) { return items >= 512 ? 1 : kv_heads; }

// workers of the backward passes that add up slope and table gradients, per list
struct AttnWorkers {
  int lone, coop, small, pair;
};

int attn_small(int dtype, const AttnParams& p, int groups, bool backward, hipStream_t st);
// fragments of up to 64 queries and keys, heads of up to 64 columns, key heads that are not shared
int attn_pair_backward(int dtype, const AttnParams& p, hipStream_t st);
int attn_forward(int dtype, const AttnPlanView& plan, const AttnParams& p, hipStream_t st);
// dq pass (with delta, dslope, dtable and the queries' share of dpos), dk / dv pass, small fragments, then the joins
int attn_backward(int dtype, const AttnPlanView& by_query, const AttnPlanView& by_key, const AttnParams& p,
                  const AttnWorkers& n, hipStream_t st);

}  // namespace vsn
