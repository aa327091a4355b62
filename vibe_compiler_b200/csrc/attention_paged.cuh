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
  if (end - begin < b.least_count || end - begin > b.most_count) return {begin, 0, 0};
  return {begin, end - begin, keys};
}
// Keys that new token `index` of a sequence sees: key j with j <= keys - count + index under the causal mask.
__device__ __forceinline__ int paged_visible(const PagedSequence &s, int index, int causal) {
  if (!causal) return s.keys;
  const int last = s.keys - s.count + index + 1;
  return last < 0 ? 0 : last;
}

// Where the rows of tokens [first, first + count) of a block lie: for each that belongs to a sequence whose lengths fit and whose page
// is one of the cache's, place(index in the block, page, row of the page, position) is called by one thread, for the others nothing.
// `sequence_of`: count words of shared memory. Ends with a barrier.
template <typename Place>
__device__ __forceinline__ void place_tokens(const PagedBatchArgs &b, const PagedCacheArgs &c, int first, int count, int *refused, int *sequence_of, Place place) {
  // Every thread compares some sequences' token ranges with the block's tokens. A range that is not one of the rows' is reported
  // whether or not a token of the block lies in it.
  if (threadIdx.x < count) sequence_of[threadIdx.x] = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < b.sequences; s += blockDim.x) {
    const int begin = b.query_starts[s], end = b.query_starts[s + 1];
    if (begin < end && (begin < 0 || end > b.tokens)) {
      raise_status(refused, kRefusedLength);
      continue;
    }
    for (int t = max(begin, first); t < min(end, first + count); ++t) sequence_of[t - first] = s;
  }
  __syncthreads();
  if (threadIdx.x < count) {
    const int s = sequence_of[threadIdx.x], token = first + static_cast<int>(threadIdx.x);
    // What attention would leave out as a whole is not written here in part: its positions mean nothing.
    const PagedSequence sequence = s >= 0 ? paged_sequence(b, c, s, refused, true) : PagedSequence{0, 0, 0};
    if (sequence.count > 0) {
      const int position = sequence.keys - sequence.count + (token - sequence.begin);      // less than keys, which the table holds
      if (position < 0) {
        raise_status(refused, kRefusedLength);
      } else {
        const int slot = position / c.page_size, row = position - slot * c.page_size;
        const int page = b.page_table[s * b.table_stride + slot];
        if (page < 0 || page >= c.pages) raise_status(refused, kRefusedPage);
        else place(static_cast<int>(threadIdx.x), page, row, position);
      }
    }
  }
  __syncthreads();
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

// 16 bytes past L1, under an L2 policy. Keys that one tile of rows reads give way first: 100 sequences of up to 1000 keys 47 -> 44 us,
// 40 of 4000 at head_dim 64 72 -> 69, 64 of 2000 to 32000 652 -> 648.
__device__ __forceinline__ void cp_async16_hint(uint64_t policy, uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(src_bytes), "l"(policy)
               : "memory");
}

}  // namespace wb200
