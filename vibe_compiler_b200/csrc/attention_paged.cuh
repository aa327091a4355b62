// What the paged attention kernels share: a sequence of the batch as the device arrays describe it, and where its keys lie.
#pragma once

#include "kernels.h"
#include "ptx_sm100.cuh"

namespace wb200 {

// Sequence s of a batch: its new tokens [begin, begin + count) and its keys. What does not fit the buffers leaves it empty and
// is reported (by one thread: `report`).
struct PagedSequence {
  int begin, count, keys;
};
__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatchArgs &b, const PagedCacheArgs &c, int s, int *refused, bool report) {
  const int begin = b.query_starts[s], end = b.query_starts[s + 1], keys = b.key_lengths[s];
  if (end <= begin) return {begin, 0, 0};
  if (begin < 0 || end > b.tokens || keys < 0 || keys > static_cast<long long>(b.table_width) * c.page_size) {
    if (report) raise_status(refused, kRefusedLength);
    return {0, 0, 0};
  }
  return {begin, end - begin, keys};
}
// Keys that new token `index` of a sequence sees: key j with j <= keys - count + index under the causal mask.
__device__ __forceinline__ int paged_visible(const PagedSequence &s, int index, int causal) {
  if (!causal) return s.keys;
  const int last = s.keys - s.count + index + 1;
  return last < 0 ? 0 : last;
}

// The first sequence from s on that brings tokens, or the number of sequences; by a whole warp, 32 sequences at a look.
__device__ __forceinline__ int next_with_tokens(const PagedBatchArgs &b, int s) {
  const int lane = threadIdx.x & 31;
  for (; s < b.sequences; s += 32) {
    const int i = s + lane;
    const unsigned int found = __ballot_sync(0xffffffffu, i < b.sequences && b.query_starts[i + 1] > b.query_starts[i]);
    if (found) return s + __ffs(found) - 1;
  }
  return b.sequences;
}

// The L2 policy of a sequence's keys: those that are read once give way first to what is read again.
__device__ __forceinline__ uint64_t l2_policy(bool read_again) {
  uint64_t normal, first;
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(normal));
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
  return read_again ? normal : first;
}

}  // namespace wb200
