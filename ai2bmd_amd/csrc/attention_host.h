// Host side shared by the fragment attention's launchers.
#pragma once
#include "attention.h"

namespace vsn {

constexpr int kMaxSlots = 1024;          // partial results of one query block
constexpr size_t kLdsPerCu = 160 * 1024;

// the work lists of one pass: `lone` items are a wave each with tiles of its own, `coop` items a workgroup of four
struct AttnPlanView {
  const AttnWork *lone_work, *coop_work;
  int lone, coop;
  const AttnJoin* join;
  int joins;
};

// waves per workgroup where every wave has its own tiles: one while there are fewer items than compute units can take
// one each, else four (as far as LDS allows)
inline int lone_waves(int64_t total, size_t bytes) {
  int waves = total <= 1024 ? 1 : 4;
  while (waves > 1 && waves * bytes > kLdsPerCu / 2) waves /= 2;
  return waves;
}

inline bool allow_lds(const void* kernel, size_t bytes) {
  return bytes <= 64 * 1024 ||
         hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess;
}

int attn_forward(int dtype, const AttnPlanView& plan, const AttnParams& p, hipStream_t st);
// dq pass (with delta, dslope, dtable and the queries' share of dpos), then the dk / dv pass, then the joins
int attn_backward(int dtype, const AttnPlanView& by_query, const AttnPlanView& by_key, const AttnParams& p,
                  int lone_workers, int coop_workers, hipStream_t st);

}  // namespace vsn
