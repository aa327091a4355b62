// The pages of a KV cache: taken for new tokens, shared and copied for forked sequences, given back, moved together.
//
// The book-keeping (reserve, fork, free, compact) is whole-number work on three small arrays, bound by latency: each call is
// ONE launch of one cluster of eight CTAs. A pass over the page counts is cut into eight parts; the CTAs exchange their
// parts' totals through distributed shared memory and meet at cluster barriers, so no call needs scratch, a second launch or
// a count the host knows. Sums over the sequences are made by every CTA for itself. Where an output array is the input
// itself nothing is copied, and everything that decides what a call does is read in front of the first barrier that a write
// stands behind.
//
// Pages are taken lowest index first in the order of the sequences, by ranks from prefix sums; counts change by integer
// atomics. No result depends on the order of threads.
//
// Measured back to back in a graph: room for the next token of 200 sequences (70 thousand pages, a table of 200 x 566) 10.6 us out
// of place and 5.5 in place with nothing to do; freeing and forking 24 of 64 sequences with the copies for 4 layers 21.5 us.
//
// pages_copy moves whole pages of many layers' caches in one launch, bound by HBM (each byte read and written once): 591 MB in 89 us,
// 6.6 TB/s.
#include "kernels.h"
#include "ptx_sm100.cuh"

namespace wb200 {
namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ int ld_cluster_i32(uint32_t cluster_addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Exclusive sum over the block's threads; *total is the sum of all. Ends with a barrier.
__device__ __forceinline__ int block_exclusive_sum(int value, int *warp_sums, int *total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int inclusive = value;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, inclusive, off);
    if (lane >= off) inclusive += other;
  }
  if (lane == 31) warp_sums[warp] = inclusive;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  __syncthreads();
  *total = all;
  return before + inclusive - value;
}

// prefix[i] = exclusive sum of value(i) over i < count, made by the whole block; returns the sum. prefix holds count + 1.
template <typename Value>
__device__ int block_prefix(int count, int *prefix, int *warp_sums, Value value) {
  int base = 0;
  for (int start = 0; start < count; start += kThreads) {
    const int i = start + static_cast<int>(threadIdx.x);
    int total;
    const int before = block_exclusive_sum(i < count ? value(i) : 0, warp_sums, &total);
    if (i < count) prefix[i] = base + before;
    base += total;
  }
  if (threadIdx.x == 0) prefix[count] = base;
  __syncthreads();
  return base;
}

// The pages of the cache are cut over the cluster's warps in order, in groups of 128: a lane looks at four neighbours at a time.
struct PagePart {
  int begin, end;
};
__device__ __forceinline__ PagePart page_part(int pages) {
  const int rank = static_cast<int>(cluster_cta_rank()) * kWarps + (threadIdx.x >> 5);
  const int groups = (pages - 1) / 128 + 1, workers = kCluster * kWarps;
  const int begin = static_cast<int>(static_cast<long long>(groups) * rank / workers), end = static_cast<int>(static_cast<long long>(groups) * (rank + 1) / workers);
  return {begin * 128, static_cast<int>(min(static_cast<long long>(end) * 128, static_cast<long long>(pages)))};
}
// The counts of pages page .. page + 3, `behind` for those from `end` on.
__device__ __forceinline__ void load_four(const int *refs, int page, int end, int behind, int (&v)[4]) {
  if (page + 3 < end && (reinterpret_cast<uintptr_t>(refs) & 15u) == 0) {
    const int4 w = *reinterpret_cast<const int4 *>(refs + page);
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = page + k < end ? refs[page + k] : behind;
  }
}
// Counts the pages for which flag(page, count) holds, each warp those of its part; *before is the number in front of the warp's
// part, the result that of all. `cta_total` is this CTA's word in the exchange. One cluster barrier.
template <typename Flag>
__device__ int cluster_count(const int *refs, int behind, PagePart part, int *warp_counts, int *cta_total, int *before, Flag flag) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int mine = 0;
#pragma unroll 2
  for (int start = part.begin; start < part.end; start += 128) {
    int v[4];
    load_four(refs, start + 4 * lane, part.end, behind, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) mine += start + 4 * lane + k < part.end && flag(start + 4 * lane + k, v[k]) ? 1 : 0;
  }
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) warp_counts[warp] = mine;
  __syncthreads();
  const int value = warp_counts[lane];               // kWarps == 32
  const int total = __reduce_add_sync(0xffffffffu, value);
  int in_front = __reduce_add_sync(0xffffffffu, lane < warp ? value : 0);
  if (threadIdx.x == 0) *cta_total = total;
  cluster_sync_all();
  const int rank = static_cast<int>(cluster_cta_rank());
  const uint32_t local = smem_u32(cta_total);
  int all = 0;
#pragma unroll
  for (int r = 0; r < kCluster; ++r) {
    const int theirs = ld_cluster_i32(cluster_map_shared(local, r));
    if (r < rank) in_front += theirs;
    all += theirs;
  }
  *before = in_front;
  return all;
}
static_assert(kWarps == 32, "a lane per warp's count");
// Walks a warp's part in order, as far as ranks below `limit` go, and calls take(page, count, is, rank) for every page: rank is
// the number of flagged pages in front of it, counted from `before`.
template <typename Flag, typename Take>
__device__ void for_each_ranked(const int *refs, int behind, PagePart part, int before, int limit, Flag flag, Take take) {
  const int lane = threadIdx.x & 31;
  for (int start = part.begin; start < part.end && before < limit; start += 128) {
    const int page = start + 4 * lane;
    int v[4], own = 0;
    load_four(refs, page, part.end, behind, v);
    bool is[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      is[k] = page + k < part.end && flag(page + k, v[k]);
      own += is[k] ? 1 : 0;
    }
    int inclusive = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, inclusive, off);
      if (lane >= off) inclusive += other;
    }
    int rank = before + inclusive - own;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (page + k < part.end) take(page + k, v[k], is[k], rank);
      rank += is[k] ? 1 : 0;
    }
    before += __shfl_sync(0xffffffffu, inclusive, 31);
  }
}
// The last i with prefix[i] <= rank (prefix ascending, prefix[0] = 0 <= rank < prefix[count]): the holder of a rank.
__device__ __forceinline__ int holder_of(const int *prefix, int count, int rank) {
  int low = 0, high = count;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (prefix[mid] <= rank) low = mid;
    else high = mid;
  }
  return low;
}
__device__ __forceinline__ int pages_of(int tokens, int page_size) { return tokens == 0 ? 0 : (tokens - 1) / page_size + 1; }
__device__ __forceinline__ int cluster_thread() { return static_cast<int>(cluster_cta_rank()) * kThreads + threadIdx.x; }
constexpr int kClusterThreads = kCluster * kThreads;

// Tokens held by a sequence; -1 for what the table cannot express.
__device__ __forceinline__ int held_tokens(const PageTablesArgs &p, int s) {
  const int tokens = p.lengths[s];
  if (tokens >= 0 && tokens <= static_cast<long long>(p.table_width) * p.page_size) return tokens;
  raise_status(p.refused, kRefusedLength);
  return -1;
}
// The output arrays as the inputs are, where they are not the inputs themselves.
__device__ void copy_ints(const int *from, int *to, int64_t count) {
  int64_t done = 0;
  if (((reinterpret_cast<uintptr_t>(from) | reinterpret_cast<uintptr_t>(to)) & 15u) == 0) {
    const int64_t quads = count / 4;
#pragma unroll 4
    for (int64_t i = cluster_thread(); i < quads; i += kClusterThreads) reinterpret_cast<int4 *>(to)[i] = reinterpret_cast<const int4 *>(from)[i];
    done = quads * 4;
  }
  for (int64_t i = done + cluster_thread(); i < count; i += kClusterThreads) to[i] = from[i];
}
__device__ void copy_tables(const PageTablesArgs &p) {
  if (p.refs_out != p.refs) copy_ints(p.refs, p.refs_out, p.pages);
  if (p.lengths_out != p.lengths) copy_ints(p.lengths, p.lengths_out, p.sequences);
  if (p.table_out == p.table) return;
  if (p.sequences == 1 || (p.table_stride == p.table_width && p.table_out_stride == p.table_width)) {
    copy_ints(p.table, p.table_out, static_cast<int64_t>(p.sequences) * p.table_width);
    return;
  }
  const int warp = cluster_thread() >> 5, lane = threadIdx.x & 31;
  for (int s = warp; s < p.sequences; s += kClusterThreads / 32) {
    const int *from = p.table + s * p.table_stride;
    int *to = p.table_out + s * p.table_out_stride;
#pragma unroll 8
    for (int j = lane; j < p.table_width; j += 32) to[j] = from[j];
  }
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) pages_reserve_kernel(const PageTablesArgs p, const int *wanted, int *result) {
  extern __shared__ int shared[];
  int *first = shared, *have = shared + p.sequences + 1;   // [sequences + 1]: rank of a sequence's first new page; [sequences]: pages it has
  __shared__ int warp_sums[kWarps], cta_total;
  __shared__ int too_wide;
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x == 0) too_wide = 0;
  __syncthreads();
  copy_tables(p);
  const int extra = block_prefix(p.sequences, first, warp_sums, [&](int s) {
    const int held = held_tokens(p, s), need = pages_of(max(max(held, wanted[s]), 0), p.page_size);
    have[s] = pages_of(max(held, 0), p.page_size);
    if (held < 0 || need > p.table_width) { too_wide = 1; return 0; }
    return need - have[s];
  });
  const PagePart part = page_part(p.pages);
  auto is_free = [](int, int count) { return count == 0; };
  int before;
  // The barrier of the count stands between everything that decides what is done, and the copies, and the changes.
  const int free_pages = cluster_count(p.refs, 1, part, warp_sums, &cta_total, &before, is_free);
  cluster_arrive();
  const int outcome = too_wide ? -1 : max(0, extra - free_pages);
  if (cluster_thread() == 0) *result = outcome;
  if (outcome == 0) {
    int s = -1;                                    // the sequence that the lane's last page went to
    for_each_ranked(p.refs, 1, part, before, extra, is_free, [&](int page, int, bool is, int rank) {
      if (!is || rank >= extra) return;
      if (s < 0 || rank >= first[s + 1]) s = holder_of(first, p.sequences, rank);
      p.table_out[s * p.table_out_stride + have[s] + rank - first[s]] = page;
      p.refs_out[page] = 1;
    });
    for (int i = cluster_thread(); i < p.sequences; i += kClusterThreads) {
      const int held = p.lengths[i], tokens = max(held, wanted[i]);
      if (tokens != held) p.lengths_out[i] = tokens;
    }
  }
  cluster_wait();   // every CTA has read the others' totals
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads)
pages_fork_kernel(const PageTablesArgs p, int count, const int *parents, const int *children, int *sources, int *destinations, int *result) {
  extern __shared__ int shared[];         // first[count + 1], then a bit per sequence: is a child
  int *first = shared;
  unsigned int *named = reinterpret_cast<unsigned int *>(shared + count + 1);
  __shared__ int warp_sums[kWarps], cta_total;
  __shared__ int wrong;
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x == 0) wrong = 0;
  for (int i = threadIdx.x; i < (p.sequences + 31) / 32; i += kThreads) named[i] = 0u;
  __syncthreads();
  copy_tables(p);
  auto in_table = [&](int s) { return s >= 0 && s < p.sequences; };
  const int extra = block_prefix(count, first, warp_sums, [&](int i) {
    const int parent = parents[i], child = children[i];
    if (!in_table(parent) || !in_table(child)) { wrong = 1; return 0; }
    if (p.lengths[child] != 0 || (atomicOr(&named[child >> 5], 1u << (child & 31)) >> (child & 31) & 1u)) { wrong = 1; return 0; }
    const int held = held_tokens(p, parent);
    if (held < 0) { wrong = 1; return 0; }
    return held % p.page_size != 0 ? 1 : 0;
  });
  for (int i = threadIdx.x; i < count; i += kThreads)
    if (in_table(parents[i]) && (named[parents[i] >> 5] >> (parents[i] & 31) & 1u)) wrong = 1;   // a parent that is a child
  const PagePart part = page_part(p.pages);
  auto is_free = [](int, int count) { return count == 0; };
  int before;
  const int free_pages = cluster_count(p.refs, 1, part, warp_sums, &cta_total, &before, is_free);
  cluster_arrive();
  const int outcome = wrong ? -1 : max(0, extra - free_pages);
  if (cluster_thread() == 0) *result = outcome;
  const int warp = cluster_thread() >> 5, lane = threadIdx.x & 31;
  if (outcome == 0) {
    // Parents are no children and children hold nothing, so what is read here is written by nobody; free pages and shared ones
    // are different pages, and a count that is raised meanwhile was not 0.
    for_each_ranked(p.refs, 1, part, before, extra, is_free, [&](int page, int, bool is, int rank) {
      if (!is || rank >= extra) return;
      const int i = holder_of(first, count, rank);
      p.table_out[children[i] * p.table_out_stride + p.lengths[parents[i]] / p.page_size] = page;
      p.refs_out[page] = 1;
      destinations[i] = page;
    });
    for (int i = warp; i < count; i += kClusterThreads / 32) {
      const int parent = parents[i], child = children[i], tokens = p.lengths[parent], full = tokens / p.page_size;
      const bool partial = tokens % p.page_size != 0;
      const int *from = p.table + parent * p.table_stride;
      int *to = p.table_out + child * p.table_out_stride;
#pragma unroll 4
      for (int j = lane; j < p.table_width; j += 32) {
        if (j < full) {
          const int page = from[j];
          to[j] = page;
          if (page >= 0 && page < p.pages) atomicAdd(p.refs_out + page, 1);
          else raise_status(p.refused, kRefusedPage);
        } else if (j != full || !partial) {
          to[j] = -1;
        }
      }
      if (lane == 0) {
        int source = partial ? from[full] : -1;
        if (partial && (source < 0 || source >= p.pages)) {        // nothing to copy the child's last rows from
          raise_status(p.refused, kRefusedPage);
          source = -1;
        }
        sources[i] = source;
        if (!partial) destinations[i] = -1;
        p.lengths_out[child] = tokens;
      }
    }
  } else {
    for (int i = cluster_thread(); i < count; i += kClusterThreads) sources[i] = destinations[i] = -1;
  }
  cluster_wait();   // every CTA has read the others' totals
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) pages_free_kernel(const PageTablesArgs p, int count, const int *sequences) {
  pdl_wait();
  pdl_launch_dependents();
  copy_tables(p);
  cluster_sync_all();
  const int warp = cluster_thread() >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < count; i += kClusterThreads / 32) {
    const int s = sequences[i];
    if (s < 0) continue;
    if (s >= p.sequences) {
      raise_status(p.refused, kRefusedSequence);
      continue;
    }
    // Whoever takes the length frees the sequence; one named twice has none left for the second.
    int tokens = 0;
    if (lane == 0) tokens = atomicExch(p.lengths_out + s, 0);
    tokens = __shfl_sync(0xffffffffu, tokens, 0);
    if (tokens == 0) continue;
    if (tokens < 0 || tokens > static_cast<long long>(p.table_width) * p.page_size) {
      raise_status(p.refused, kRefusedLength);
      if (lane == 0) p.lengths_out[s] = tokens;
      continue;
    }
    const int used = pages_of(tokens, p.page_size);
    int *row = p.table_out + s * p.table_out_stride;
    for (int j = lane; j < p.table_width; j += 32) {
      if (j < used) {
        const int page = row[j];
        if (page < 0 || page >= p.pages) {
          raise_status(p.refused, kRefusedPage);
        } else if (atomicSub(p.refs_out + page, 1) <= 0) {
          atomicAdd(p.refs_out + page, 1);
          raise_status(p.refused, kRefusedReference);
        }
      }
      row[j] = -1;
    }
  }
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) pages_compact_kernel(const PageTablesArgs p, int *sources, int *destinations) {
  __shared__ int warp_counts[kWarps], cta_totals[2];
  pdl_wait();
  pdl_launch_dependents();
  const PagePart part = page_part(p.pages);
  int before, front_before;
  const int live = cluster_count(p.refs, 0, part, warp_counts, &cta_totals[0], &before, [](int, int count) { return count > 0; });
  const int in_front = cluster_count(p.refs, 0, part, warp_counts, &cta_totals[1], &front_before, [&](int page, int count) { return page < live && count > 0; });
  const int moves = live - in_front;      // used pages behind the first `live`, and free ones among them
  for_each_ranked(p.refs, 0, part, before, live + 1, [](int, int count) { return count > 0; }, [&](int page, int, bool used, int rank) {
    if (used && page >= live) sources[rank - in_front] = page;
    if (!used && page < live) destinations[page - rank] = page;      // the pages in front of it less the used ones
  });
  for (int i = moves + cluster_thread(); i < p.pages / 2; i += kClusterThreads) sources[i] = destinations[i] = -1;
  if (p.refs_out != p.refs) copy_ints(p.refs, p.refs_out, p.pages);
  cluster_sync_all();
  // A moved page's count goes along, and in its place stands, until the table is done, where the page went.
  for (int i = cluster_thread(); i < moves; i += kClusterThreads) {
    const int from = sources[i], to = destinations[i];
    p.refs_out[to] = p.refs[from];
    p.refs_out[from] = -1 - to;
  }
  cluster_sync_all();
  const int warp = cluster_thread() >> 5, lane = threadIdx.x & 31;
  for (int s = warp; s < p.sequences; s += kClusterThreads / 32) {
    const int used = pages_of(max(held_tokens(p, s), 0), p.page_size);
    const int *from = p.table + s * p.table_stride;
    int *to = p.table_out + s * p.table_out_stride;
    const int width = p.table_out == p.table ? used : p.table_width;
#pragma unroll 4
    for (int j = lane; j < width; j += 32) {
      int page = from[j];
      if (j < used) {
        if (page < 0 || page >= p.pages) raise_status(p.refused, kRefusedPage);
        else if (page >= live && p.refs_out[page] < 0 && -1 - p.refs_out[page] < live) page = -1 - p.refs_out[page];
      }
      to[j] = page;
    }
  }
  if (p.lengths_out && p.lengths_out != p.lengths)
    for (int s = cluster_thread(); s < p.sequences; s += kClusterThreads) p.lengths_out[s] = p.lengths[s];
  cluster_sync_all();
  for (int i = cluster_thread(); i < moves; i += kClusterThreads) p.refs_out[sources[i]] = 0;
}

// ------------------------------------------------------------------ the pages' contents
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;

struct CopyParams {
  uint8_t *base[2 * kMaxCachesPerCopy];   // K and V of every cache
  int tensors, count, pages;
  const int *sources, *destinations;
  int *refused;
  // a page is `runs` runs of `run_units` units: outer * inner of them, outer and inner strides in units
  int64_t page_stride[2];                 // K, V
  int64_t outer_stride[2], inner_stride[2];
  int outer, inner, run_units, unit_bytes;
  int chunk_units, chunks;                // a page's units are cut into `chunks` chunks
};

// A block takes chunk blockIdx.y % chunks of tensor blockIdx.y / chunks, for every gridDim.x-th page. The page numbers are
// looked up 32 at a time, so entries that are passed over cost next to nothing.
template <typename Unit, bool kDense>
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const __grid_constant__ CopyParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int tensor = blockIdx.y / p.chunks, chunk = blockIdx.y - tensor * p.chunks, kind = tensor & 1;
  Unit *base = reinterpret_cast<Unit *>(p.base[tensor]);
  const int begin = chunk * p.chunk_units, end = min(begin + p.chunk_units, p.outer * p.inner * p.run_units);
  for (int64_t i0 = blockIdx.x; i0 < p.count; i0 += 32ll * gridDim.x) {
    const int64_t mine = i0 + static_cast<int64_t>(lane) * gridDim.x;
    int source = -1, destination = -1;
    if (mine < p.count) { source = p.sources[mine]; destination = p.destinations[mine]; }
    const bool wanted = source >= 0 && destination >= 0, inside = source < p.pages && destination < p.pages;
    if (wanted && !inside && threadIdx.x < 32) raise_status(p.refused, kRefusedPage);
    unsigned int todo = __ballot_sync(0xffffffffu, wanted && inside && source != destination);
    while (todo) {
      const int from_lane = __ffs(todo) - 1;
      todo &= todo - 1;
      const Unit *from = base + __shfl_sync(0xffffffffu, source, from_lane) * p.page_stride[kind];
      Unit *to = base + __shfl_sync(0xffffffffu, destination, from_lane) * p.page_stride[kind];
      auto place = [&](int u) -> int64_t {
        if constexpr (kDense) return u;
        const int run = u / p.run_units, outer = run / p.inner;
        return outer * p.outer_stride[kind] + (run - outer * p.inner) * p.inner_stride[kind] + (u - run * p.run_units);
      };
      int u = begin + threadIdx.x;
      for (; u + (kCopyUnroll - 1) * kCopyThreads < end; u += kCopyUnroll * kCopyThreads) {
        Unit held[kCopyUnroll];
#pragma unroll
        for (int k = 0; k < kCopyUnroll; ++k) held[k] = from[place(u + k * kCopyThreads)];
#pragma unroll
        for (int k = 0; k < kCopyUnroll; ++k) to[place(u + k * kCopyThreads)] = held[k];
      }
      for (; u < end; u += kCopyThreads) to[place(u)] = from[place(u)];
    }
  }
}

wb200_status check_launch(const char *what, cudaError_t error) {
  if (error != cudaSuccess) return fail(WB200_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(error));
  return WB200_OK;
}

constexpr size_t kMostShared = (2 * kMaxPagedSequences + 1) * sizeof(int);
wb200_status allow_shared() {
  static PerDeviceOnce attributes;
  return attributes.run([]() -> wb200_status {
    WB200_CUDA_CHECK(cudaFuncSetAttribute(pages_reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostShared)));
    WB200_CUDA_CHECK(cudaFuncSetAttribute(pages_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostShared)));
    return WB200_OK;
  });
}

}  // namespace

wb200_status launch_pages_reserve(const PageTablesArgs &args, const int *wanted, int *result, cudaStream_t stream) {
  wb200_status st = allow_shared();
  if (st != WB200_OK) return st;
  return check_launch("pages_reserve", launch_dependent(pages_reserve_kernel, kCluster, kThreads, (2 * static_cast<size_t>(args.sequences) + 1) * sizeof(int),
                                                        stream, args, wanted, result));
}

wb200_status launch_pages_fork(const PageTablesArgs &args, int count, const int *parents, const int *children, int *sources, int *destinations,
                               int *result, cudaStream_t stream) {
  wb200_status st = allow_shared();
  if (st != WB200_OK) return st;
  const size_t words = static_cast<size_t>(count) + 1 + (static_cast<size_t>(args.sequences) + 31) / 32;
  return check_launch("pages_fork", launch_dependent(pages_fork_kernel, kCluster, kThreads, words * sizeof(int), stream, args, count, parents, children,
                                                     sources, destinations, result));
}

wb200_status launch_pages_free(const PageTablesArgs &args, int count, const int *sequences, cudaStream_t stream) {
  return check_launch("pages_free", launch_dependent(pages_free_kernel, kCluster, kThreads, 0, stream, args, count, sequences));
}

wb200_status launch_pages_compact(const PageTablesArgs &args, int *sources, int *destinations, cudaStream_t stream) {
  return check_launch("pages_compact", launch_dependent(pages_compact_kernel, kCluster, kThreads, 0, stream, args, sources, destinations));
}

wb200_status launch_pages_copy(const PagedCacheArgs *caches, int cache_count, int count, const int *sources, const int *destinations, int *refused,
                               cudaStream_t stream) {
  const PagedCacheArgs &c = caches[0];
  const int element = c.format == WB200_F32 ? 4 : 2;
  CopyParams p{};
  p.tensors = 2 * cache_count;
  p.count = count;
  p.pages = c.pages;
  p.sources = sources;
  p.destinations = destinations;
  p.refused = refused;
  const int64_t strides[2][3] = {{c.k_page, c.k_row, c.k_head}, {c.v_page, c.v_row, c.v_head}};
  uint64_t bits = static_cast<uint64_t>(c.head_dim) * element;
  for (int t = 0; t < cache_count; ++t) {
    p.base[2 * t] = static_cast<uint8_t *>(caches[t].k);
    p.base[2 * t + 1] = static_cast<uint8_t *>(caches[t].v);
    bits |= reinterpret_cast<uintptr_t>(caches[t].k) | reinterpret_cast<uintptr_t>(caches[t].v);
  }
  bool dense = true;      // rows and heads of a page leave no gap, in either order
  for (int kind = 0; kind < 2; ++kind) {
    for (int i = 0; i < 3; ++i) bits |= static_cast<uint64_t>(strides[kind][i] * element);
    const int64_t row = strides[kind][1], head = strides[kind][2];
    const bool rows_outside = (c.kv_heads == 1 || head == c.head_dim) && (c.page_size == 1 || row == static_cast<int64_t>(c.kv_heads) * c.head_dim);
    const bool heads_outside = (c.page_size == 1 || row == c.head_dim) && (c.kv_heads == 1 || head == static_cast<int64_t>(c.page_size) * c.head_dim);
    dense = dense && (rows_outside || heads_outside);
  }
  p.unit_bytes = (bits & 15u) == 0 ? 16 : element;      // every run begins and ends on 16 bytes
  const int per_unit = p.unit_bytes / element;
  for (int kind = 0; kind < 2; ++kind) {
    p.page_stride[kind] = strides[kind][0] / per_unit;
    p.outer_stride[kind] = strides[kind][1] / per_unit;
    p.inner_stride[kind] = strides[kind][2] / per_unit;
  }
  p.outer = c.page_size;
  p.inner = c.kv_heads;
  p.run_units = c.head_dim / per_unit;
  // A chunk keeps a block busy for a while (16 units a thread); more blocks than fit at once take the pages in turn.
  const int64_t units = static_cast<int64_t>(p.outer) * p.inner * p.run_units;
  if (units > (1ll << 30)) return fail(WB200_ERR_LIMIT, "a page of more than 2^30 units");
  p.chunk_units = 16 * kCopyThreads;
  while ((units + p.chunk_units - 1) / p.chunk_units * p.tensors > 65535) p.chunk_units *= 2;
  p.chunks = static_cast<int>((units + p.chunk_units - 1) / p.chunk_units);
  const int64_t columns = static_cast<int64_t>(p.chunks) * p.tensors;
  int64_t rows = (148 * 8 * 4 + columns - 1) / columns;
  if (rows > count) rows = count;
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(columns));
  void (*kernel)(const CopyParams);
  if (p.unit_bytes == 16) kernel = dense ? pages_copy_kernel<uint4, true> : pages_copy_kernel<uint4, false>;
  else if (element == 4) kernel = dense ? pages_copy_kernel<uint32_t, true> : pages_copy_kernel<uint32_t, false>;
  else kernel = dense ? pages_copy_kernel<uint16_t, true> : pages_copy_kernel<uint16_t, false>;
  return check_launch("pages_copy", launch_dependent(kernel, grid, kCopyThreads, 0, stream, p));
}

}  // namespace wb200
