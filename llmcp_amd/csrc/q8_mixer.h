// q8_mixer.h -- device helpers that the token mixers' kernels share: the
// sequences of a call and the slots of a paged cache.
#pragma once

#include "q8_device.h"
#include "q8_kernels.h"

namespace llmcp_q8 {

// Rows lo .. hi - 1 of a sequence, whatever row_starts holds.
struct RowRange {
  int32_t lo, hi;
};
__device__ __forceinline__ RowRange clamp_range(int32_t a, int32_t b, int32_t rows) {
  RowRange r;
  r.lo = min(max(a, 0), rows);
  r.hi = min(max(b, r.lo), rows);
  return r;
}
__device__ __forceinline__ RowRange row_range(const int32_t *starts, int32_t s, int32_t rows) {
  return clamp_range(starts[s], starts[s + 1], rows);
}

// The sequence that has `row` (the same in the whole wave), -1 for none: as
// many sequences as end at or before it, 64 looked at together.
__device__ __forceinline__ int32_t sequence_of(const int32_t *starts, int32_t sequences,
                                               int32_t row, int lane) {
  int32_t s = 0;
  for (int32_t at = 0; at < sequences; at += 64) {
    const bool before = at + lane < sequences && starts[at + lane + 1] <= row;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(before));
    s += n;
    if (n < 64) break;
  }
  if (s >= sequences) return -1;
  return __builtin_amdgcn_readfirstlane(s);
}

// The page of a position, -1 for none; an id that is none sets the flag.
__device__ __forceinline__ int32_t page_at(const KvBatch &b, const KvPages &c, int32_t s,
                                           int32_t index, int32_t *err_flag) {
  const int32_t page = b.table[(int64_t)s * b.max_pages + index];
  if ((uint32_t)page < (uint32_t)c.pages) return page;
  if (page != -1 && err_flag) *err_flag = 1;
  return -1;
}

}  // namespace llmcp_q8
