// Attention of few rows over a paged cache: how the work is dealt to the CTAs, and how a row's states are put together.
//
// The rows that share a KV head, (token, query head of its group), are packed into tiles of kRows: row r of a tile is token
// r / group, head r % group. A unit of work is one tile of rows of one KV head of one sequence; its keys are cut into steps. All
// units lie one behind the other on one axis of steps, which is cut into as many equal shares as there are CTAs. A share that ends
// inside a unit leaves an un-finalized record (m, l, acc) in the workspace, which a second kernel folds with the unit's others.
#pragma once

#include "attention_paged.cuh"

namespace wb200 {

constexpr int kRowsCluster = 8;     // the portable cluster size

// What the fold has to know about the unit that a CTA's share ends inside of; `records` 0: no such unit.
struct RowsSplit {
  int records, begin, count, tile, kv_head, reserved[3];
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// floor(a / b) for whole 0 <= a < 2^53 and 0 < b < 2^53: a quotient that is not whole is at least 1 / b away from the next whole
// number, more than the division's rounding.
__device__ __forceinline__ long long floor_ratio(long long a, long long b) { return static_cast<long long>(static_cast<double>(a) / static_cast<double>(b)); }

// The part of a unit that lies in a CTA's share: steps [step0, step1) of `steps`.
struct RowsPart {
  PagedSequence sequence;
  int s, kv_head, row_tile, row0, rows;  // the sequence; first packed row, rows there are
  int step0, step1, steps, left;         // left: work of the unit behind the share
  int keys;                              // that the tile's last token sees
  __device__ __forceinline__ bool whole() const { return step0 == 0 && step1 == steps; }
};

// kUnitSteps: what a unit costs by itself, in steps; a cut this near behind its beginning falls on it. kLeastSteps: no share is made
// smaller, as small batches are latency, and more CTAs shorten it. kClustered: a cluster of kRowsCluster CTAs takes all units of one
// KV head of one sequence (blockIdx.y), an equal part of a unit's keys each.
template <int kRows, int kStepKeys, int kUnitSteps, int kLeastSteps, int kWarps, bool kClustered>
struct RowsWalk {
  const AttentionPagedArgs &a;
  const int group;
  const unsigned long long by_grid;      // floor((2^64 - 1) / grid) + 1: n / grid = n * by_grid >> 64 for n < 2^55
  RowsPart part;
  int s, next_tile, shares, index, grid;
  long long total, at, share_end, prefix;   // the share: at .. share_end, from sequence s on, in front of which `prefix` steps lie

  __device__ __forceinline__ RowsWalk(const AttentionPagedArgs &args, int rows_group, unsigned long long reciprocal)
      : a(args), group(rows_group), by_grid(reciprocal), part(), s(-1), next_tile(0), shares(1), index(static_cast<int>(blockIdx.x)),
        grid(static_cast<int>(gridDim.x)), total(0), at(0), share_end(0), prefix(0) {}

  struct Units {
    int steps;
    long long weight;
  };
  // A sequence's units: tiles of rows x KV heads, each of `steps` steps of keys (at least one, so that rows without keys are written).
  __device__ __forceinline__ Units units_of(const PagedSequence &q) const {
    if (q.count == 0) return {1, 0};
    const int steps = q.keys == 0 ? 1 : (q.keys - 1) / kStepKeys + 1;
    const long long tiles = (static_cast<long long>(q.count) * group + kRows - 1) / kRows;
    return {steps, tiles * a.cache.kv_heads * (steps + kUnitSteps)};
  }
  // Where share i begins: total * i / shares. Totals of fewer shares than CTAs are small.
  __device__ __forceinline__ long long cut_at(int i) const {
    const unsigned long long n = static_cast<unsigned long long>(total) * static_cast<unsigned>(i);
    return static_cast<long long>(shares == grid ? __umul64hi(n, by_grid) : static_cast<unsigned>(n) / static_cast<unsigned>(shares));
  }

  // Finds the CTA's share; all threads. `totals`: kWarps words of shared memory, `start`, `start_prefix`: one each.
  __device__ __forceinline__ void find_share(long long *totals, int *start, long long *start_prefix) {
    if constexpr (kClustered) {
      s = static_cast<int>(blockIdx.y) / a.cache.kv_heads;
    } else {
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
      // A thread sums up a run of consecutive sequences.
      const int per_thread = (a.batch.sequences + kWarps * 32 - 1) / (kWarps * 32);
      const int first_mine = min(a.batch.sequences, static_cast<int>(threadIdx.x) * per_thread), end_mine = min(a.batch.sequences, first_mine + per_thread);
      long long mine = 0;
#pragma unroll 4
      for (int i = first_mine; i < end_mine; ++i) mine += units_of(paged_sequence(a.batch, a.cache, i, a.refused, false)).weight;
      if (blockIdx.x == 0)
        for (int i = first_mine; i < end_mine; ++i) paged_sequence(a.batch, a.cache, i, a.refused, true);
      long long before = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += other;
      }
      if (lane == 31) totals[warp] = before;
      if (threadIdx.x == 0) *start = -1;
      __syncthreads();
      before -= mine;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += totals[w];
        total += totals[w];
      }
      shares = total >= static_cast<long long>(kLeastSteps) * grid ? grid : max(1, static_cast<int>(total) / kLeastSteps);
      at = index < shares ? cut_at(index) : total;
      share_end = index < shares ? cut_at(index + 1) : total;
      if (at < share_end && before <= at && at < before + mine) {
        for (int i = first_mine; i < end_mine; ++i) {
          const long long weight = units_of(paged_sequence(a.batch, a.cache, i, a.refused, false)).weight;
          if (at < before + weight) {
            *start = i;
            *start_prefix = before;
            break;
          }
          before += weight;
        }
      }
      __syncthreads();
      s = *start;
      prefix = s >= 0 ? *start_prefix : 0;
    }
  }

  __device__ __forceinline__ void settle() {
    part.s = s;
    part.row0 = part.row_tile * kRows;
    part.rows = static_cast<int>(min(static_cast<long long>(part.sequence.count) * group - part.row0, static_cast<long long>(kRows)));
    // keys that the tile's last token sees bound what is read
    part.keys = min(part.sequence.keys, paged_visible(part.sequence, (part.row0 + part.rows - 1) / group, a.causal));
  }
  // The next part of the share; false: there is none. By whole warps, all alike.
  __device__ __forceinline__ bool next() {
    if constexpr (kClustered) {
      // The next tile of rows of the sequence; every CTA of the cluster has a part of it, be it empty.
      part.kv_head = static_cast<int>(blockIdx.y) - s * a.cache.kv_heads;
      part.sequence = paged_sequence(a.batch, a.cache, s, a.refused, blockIdx.x == 0 && part.kv_head == 0);
      if (static_cast<long long>(next_tile) * kRows >= static_cast<long long>(part.sequence.count) * group) return false;
      part.row_tile = next_tile++;
      part.steps = units_of(part.sequence).steps;
      part.step0 = static_cast<int>(static_cast<long long>(part.steps) * blockIdx.x / kRowsCluster);
      part.step1 = static_cast<int>(static_cast<long long>(part.steps) * (blockIdx.x + 1) / kRowsCluster);
      settle();
      return true;
    } else {
      while (s >= 0 && at < share_end) {
        part.sequence = paged_sequence(a.batch, a.cache, s, a.refused, false);
        const Units units = units_of(part.sequence);
        if (at >= prefix + units.weight) {               // on to the next sequence that has rows
          prefix += units.weight;
          s = next_with_tokens(a.batch, s + 1);
          if (s >= a.batch.sequences) return false;
          continue;
        }
        const long long into = at - prefix;
        const int all = units.steps + kUnitSteps;
        const int unit = into >> 32 ? static_cast<int>(floor_ratio(into, all)) : static_cast<int>(static_cast<unsigned>(into) / static_cast<unsigned>(all));
        const int begin = static_cast<int>(into - static_cast<long long>(unit) * all);
        const int end = static_cast<int>(min(static_cast<long long>(all), begin + (share_end - at)));
        at += end - begin;
        part.left = all - end;
        part.steps = units.steps;
        part.step0 = max(begin - kUnitSteps, 0);
        part.step1 = max(end - kUnitSteps, 0);
        if (part.step1 == part.step0) continue;
        part.row_tile = unit / a.cache.kv_heads;
        part.kv_head = unit - part.row_tile * a.cache.kv_heads;
        settle();
        return true;
      }
      return false;
    }
  }
  // Of a unit whose beginning ended the share: it goes on in the CTAs behind this one, up to the last share that begins in front of
  // its end.
  __device__ __forceinline__ RowsSplit split_of(const RowsPart &done) const {
    int behind = 0;
#pragma unroll 1
    for (int start = index + 1;; start += 32) {
      const int i = start + static_cast<int>(threadIdx.x & 31);
      const unsigned int inside = __ballot_sync(0xffffffffu, i < shares && cut_at(i) < share_end + done.left);
      behind += __popc(inside);
      if (inside != 0xffffffffu) break;
    }
    return {1 + behind, done.sequence.begin, done.sequence.count, done.row_tile, done.kv_head, {}};
  }
};

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&v);
  }
}
// A lane's elements of a row of kD floats.
template <int kD>
struct Slice {
  static constexpr int kPer = kD / 32;
  float v[kPer];
  __device__ __forceinline__ void load(const float *row, int lane) {
    if constexpr (kPer == 4) {
      const float4 w = *reinterpret_cast<const float4 *>(row + 4 * lane);
      v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
      const float2 w = *reinterpret_cast<const float2 *>(row + 2 * lane);
      v[0] = w.x; v[1] = w.y;
    }
  }
  __device__ __forceinline__ void load_cluster(uint32_t row, int lane) {     // of a CTA of the cluster
    if constexpr (kPer == 4) {
      const float4 w = ld_cluster_f32x4(row + 16 * lane);
      v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
      const float2 w = ld_cluster_f32x2(row + 8 * lane);
      v[0] = w.x; v[1] = w.y;
    }
  }
  __device__ __forceinline__ void store(float *row, int lane) const {
    if constexpr (kPer == 4) *reinterpret_cast<float4 *>(row + 4 * lane) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<float2 *>(row + 2 * lane) = make_float2(v[0], v[1]);
  }
};

// Writes a finished row (statistics in the log2 domain): out = acc / l, one rounding.
template <bool kBf16, int kD>
__device__ __forceinline__ void write_row(const AttentionPagedArgs &a, int token, int head, int lane, float m, float l, const Slice<kD> &acc) {
  constexpr uint32_t kNan = kBf16 ? 0x7fc07fc0u : 0x7e007e00u;
  const bool empty = l == 0.f;
  const float coefficient = empty ? 0.f : 1.0f / l;
  uint32_t bits[Slice<kD>::kPer / 2];
#pragma unroll
  for (int i = 0; i < Slice<kD>::kPer / 2; ++i) {
    bits[i] = pack2<kBf16>(acc.v[2 * i] * coefficient, acc.v[2 * i + 1] * coefficient);
    if (empty) bits[i] = a.zero_fully_masked ? 0u : kNan;
  }
  uint16_t *out = static_cast<uint16_t *>(a.out) + token * a.out_token + head * a.out_head + Slice<kD>::kPer * lane;
  if constexpr (kD == 128) *reinterpret_cast<uint2 *>(out) = make_uint2(bits[0], bits[1]);
  else *reinterpret_cast<uint32_t *>(out) = bits[0];
  if (a.lse && lane == 0) a.lse[static_cast<int64_t>(token) * a.q_heads + head] = empty ? -INFINITY : m * 0.69314718055994530942f + logf(l);
}

// A row's record: acc[kD], m, l (m in the log2 domain, a reference that need not be the maximum) and padding to 16 bytes.
template <int kD>
constexpr int kRowRecord = kD + 4;

// One row's states of the block's warps, kWarps records 8 rows apart, as one: a warp, with the largest m as the common exponent
// reference.
template <int kD, int kWarps>
__device__ __forceinline__ void fold_warps(const float *records, int r, int lane, float &top, float &l, Slice<kD> &sum) {
  float2 ml[kWarps];
  top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    ml[w] = *reinterpret_cast<const float2 *>(records + (w * 8 + r) * kRowRecord<kD> + kD);
    top = fmaxf(top, ml[w].x);
  }
  const float m_exp = top == -INFINITY ? 0.f : top;
  l = 0.f;
  sum = {};
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float weight = exp2_fast(ml[w].x - m_exp);
    Slice<kD> slice;
    slice.load(records + (w * 8 + r) * kRowRecord<kD>, lane);
    l = fmaf(ml[w].y, weight, l);
#pragma unroll
    for (int e = 0; e < Slice<kD>::kPer; ++e) sum.v[e] = fmaf(slice.v[e], weight, sum.v[e]);
  }
}
// The same over the CTAs of a cluster, each with the record at `record` of its shared memory.
template <int kD>
__device__ __forceinline__ void fold_cluster(const float *record, int lane, float &top, float &l, Slice<kD> &sum) {
  const uint32_t local = smem_u32(record);
  float2 ml = make_float2(-INFINITY, 0.f);             // of CTA `lane`
  if (lane < kRowsCluster) ml = ld_cluster_f32x2(cluster_map_shared(local + kD * 4, lane));
  top = ml.x;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  const float weight = exp2_fast(ml.x - (top == -INFINITY ? 0.f : top));
  l = ml.y * weight;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  sum = {};
#pragma unroll
  for (int c = 0; c < kRowsCluster; ++c) {
    Slice<kD> slice;
    slice.load_cluster(cluster_map_shared(local, c), lane);
    const float w = __shfl_sync(0xffffffffu, weight, c);
#pragma unroll
    for (int e = 0; e < Slice<kD>::kPer; ++e) sum.v[e] = fmaf(slice.v[e], w, sum.v[e]);
  }
}

struct RowsFold {
  AttentionPagedArgs a;
  int group;                        // query heads per KV head
  float *records;                   // [grid][2][kRows][kRowRecord]: a share's end of a unit (0), its start of one (1)
  RowsSplit *splits;                // [grid]
};

// Folds the records of the unit that starts in share blockIdx.x and goes on in the shares behind it: row blockIdx.y, a thread
// per element. Every warp weighs 32 records at a time with a lane each; the records' elements are loaded eight at a time.
template <bool kBf16, int kD, int kRows>
__global__ void __launch_bounds__(kD) attention_paged_fold_kernel(const __grid_constant__ RowsFold p) {
  constexpr int kRecord = kRowRecord<kD>;
  pdl_wait();
  pdl_launch_dependents();
  const RowsSplit split = p.splits[blockIdx.x];
  const int lane = threadIdx.x & 31, r = blockIdx.y;
  const int packed = split.tile * kRows + r, token = packed / p.group;
  if (split.records == 0 || token >= split.count) return;
  // record 0: the start (slot 1) of the first share; the others: the ends (slot 0) of the shares behind it
  const float *base = p.records + (static_cast<int64_t>(blockIdx.x) * 2 * kRows + r) * kRecord;
  auto record = [&](int i) { return base + (i == 0 ? kRows * kRecord : static_cast<int64_t>(i) * 2 * kRows * kRecord); };
  float top = -INFINITY, l = 0.f, sum = 0.f;          // l: this lane's share
  for (int first = 0; first < split.records; first += 32) {
    const int count = min(32, split.records - first);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < count) ml = *reinterpret_cast<const float2 *>(record(first + lane) + kD);
    float next = fmaxf(top, ml.x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, off));
    const float m_exp = next == -INFINITY ? 0.f : next, alpha = exp2_fast(top - m_exp), weight = exp2_fast(ml.x - m_exp);
    top = next;
    l = fmaf(l, alpha, ml.y * weight);
    sum *= alpha;
    for (int i = 0; i < count; i += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i + u < count ? record(first + i + u)[threadIdx.x] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = __shfl_sync(0xffffffffu, weight, (i + u) & 31);
        sum = i + u < count ? fmaf(v[u], w, sum) : sum;
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  const bool empty = l == 0.f;
  const int head = split.kv_head * p.group + packed - token * p.group;
  const int64_t row = static_cast<int64_t>(split.begin) + token;
  uint32_t bits = pack2<kBf16>(sum * (empty ? 0.f : 1.0f / l), 0.f);
  if (empty) bits = p.a.zero_fully_masked ? 0u : (kBf16 ? 0x7fc0u : 0x7e00u);
  static_cast<uint16_t *>(p.a.out)[row * p.a.out_token + head * p.a.out_head + threadIdx.x] = static_cast<uint16_t>(bits);
  if (p.a.lse && threadIdx.x == 0) p.a.lse[row * p.a.q_heads + head] = empty ? -INFINITY : top * 0.69314718055994530942f + logf(l);
}

}  // namespace wb200
