// Attention of few new tokens over a paged KV cache: decoding and drafted tokens (bf16 / f16, head_dim 64 and 128).
//
// The rows that share a KV head, (token, query head of its group), are packed into tiles of 16 (or 8) MMA rows: row r of a
// tile is token r / group, head r % group, so a step of one token per sequence reads every key once whatever the group. A
// unit of work is one tile of rows of one KV head of one sequence; its keys are cut into steps of 64. All units lie one
// behind the other on one axis of steps, which is cut into as many equal shares as there are CTAs: every CTA streams the
// same number of keys however ragged the lengths are, and the lengths are only read on the device (each CTA sums up the
// sequences' steps for itself, one load per thread for up to 128 sequences). A share that ends inside a unit leaves an
// un-finalized record (m, l, acc) in the workspace, which the second kernel folds with the unit's other records. Few units
// of short caches take a cluster of CTAs each instead, and one launch. Which CTA takes what, and the order of the folds,
// depend on the lengths and the number of SMs alone, so results repeat bit for bit.
//
// A CTA is four warps. Each streams every fourth 16-key tile of the share through a ring of its own (cp.async, 16-byte
// copies, rows XOR-swizzled), S = Q K^T and acc += P V by mma.sync m16n8k16, the running maximum and sum in f32; the first
// tiles of a share's next unit are on their way while the state of the one before is folded over the warps. With 8 rows the
// PV product runs transposed, rows on the 8-wide side: half the products. Matrix work is far from the bound (decoding does one
// flop per byte of cache and query head; the tensor pipe is 13 % busy), so the warp-level instructions do: a tcgen05 tile
// takes 128 rows whether they are there or not.
// Bound: HBM, the K and V bytes of the visible keys. 64 sequences of 2000 to 32000 keys, 32/8 heads, f16: 640 us, 6.7 TB/s;
// 40 of 4096 keys 110 us for 672 MB (DRAM reads equal the algorithmic bytes), of which the fold's launch is about 4.
#include "attention_paged.cuh"

namespace wb200 {
namespace {

constexpr int kWarps = 4;
constexpr int kTileKeys = 16;
constexpr int kStepKeys = kWarps * kTileKeys;
constexpr int kCluster = 8;         // the portable cluster size

template <int kD>
struct RowsShape {
  static constexpr int kRowBytes = kD * 2;
  static constexpr int kTileBytes = kTileKeys * kRowBytes;
  static constexpr int kStages = kD == 128 ? 3 : 6;          // 24 KiB of copies in flight per warp either way
  static constexpr int kRingBytes = kStages * 2 * kTileBytes;
  static constexpr int kRecord = kD + 4;                     // floats: acc[D], m, l and padding to 16 bytes
  static constexpr int kRecordsOff = kWarps * kRingBytes;    // the warps' records of eight rows
  static constexpr int kSmemBytes = kRecordsOff + kWarps * 8 * kRecord * 4;
  static_assert(2 * (kSmemBytes + 512 + 1024) <= 228 * 1024, "two CTAs to an SM");
};

// What the fold has to know about the unit that a CTA's share ends inside of; `records` 0: no such unit.
struct RowsSplit {
  int records, begin, count, tile, kv_head, reserved[3];
};

struct RowsParams {
  AttentionPagedArgs a;
  int group;                        // query heads per KV head
  float scale_log2;
  unsigned long long by_grid;       // floor((2^64 - 1) / grid) + 1: n / grid = n * by_grid >> 64 for n < 2^55
  float *records;                   // [grid][2][rows per tile][kRecord]: a share's end of a unit (0), its start of one (1)
  RowsSplit *splits;                // [grid]
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 bytes past L1, under an L2 policy. Keys that one tile of rows reads give way first: 100 sequences of up to 1000 keys 47 -> 44 us,
// 40 of 4000 at head_dim 64 72 -> 69, 64 of 2000 to 32000 652 -> 648.
__device__ __forceinline__ void cp_async16_hint(uint64_t policy, uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(src_bytes), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <bool kBf16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
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
// Byte offset of 16-byte chunk c of row r in a tile of rows of kRowBytes.
template <int kRowBytes>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) { return static_cast<uint32_t>(r * kRowBytes + ((c ^ (r & 7)) << 4)); }

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

// Work is counted in steps; a unit by itself (its queries, the first copies, the fold over the warps) counts as three, and a cut
// this near behind its beginning falls on it. 40 sequences of 50 to 8000 keys (107 us at the copy rate) with 0 / 1 / 2 / 3 / 5
// steps: 130 / 124 / 119 / 117 / 116 us, 100 sequences of 20 to 1000 keys (35 us) 60 / 52 / 47 / 47 / 47.
constexpr int kUnitSteps = 3;
constexpr int kLeastSteps = 3;      // no share is made smaller: small batches are latency, and more CTAs shorten it
// floor(a / b) for whole 0 <= a < 2^53 and 0 < b < 2^53: a quotient that is not whole is at least 1 / b away from the next whole
// number, more than the division's rounding.
__device__ __forceinline__ long long floor_ratio(long long a, long long b) { return static_cast<long long>(static_cast<double>(a) / static_cast<double>(b)); }
// A sequence's units: tiles of rows x KV heads, each of `steps` steps of keys (at least one, so that rows without keys are written).
struct RowsUnits {
  int steps;
  long long weight;
};
template <int kRows>
__device__ __forceinline__ RowsUnits rows_units(const RowsParams &p, const PagedSequence &s) {
  if (s.count == 0) return {1, 0};
  const int steps = s.keys == 0 ? 1 : (s.keys - 1) / kStepKeys + 1;
  const long long tiles = (static_cast<long long>(s.count) * p.group + kRows - 1) / kRows;
  return {steps, tiles * p.a.cache.kv_heads * (steps + kUnitSteps)};
}

// kClustered: a cluster of kCluster CTAs takes a whole unit (blockIdx.y), an equal part of its keys each, and its first CTA folds
// their states through distributed shared memory: one launch and no records, for batches of few units.
template <bool kBf16, int kD, bool kNarrow, bool kAligned, bool kClustered>
__global__ void __launch_bounds__(kWarps * 32, 2) attention_paged_rows_kernel(const __grid_constant__ RowsParams p) {
  using S = RowsShape<kD>;
  constexpr int kRows = kNarrow ? 8 : 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long warp_totals[kWarps], start_prefix;
  __shared__ int start_sequence;
  __shared__ int seen_keys[kWarps][S::kStages];       // bit i: key i of the tile in that slot takes part
  const AttentionPagedArgs &a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();

  // This CTA's share of all steps: at .. share_end, from sequence s on, in front of which `prefix` steps lie.
  int s = -1, next_tile = 0;
  long long total = 0, at = 0, share_end = 0, prefix = 0;
  const int index = static_cast<int>(blockIdx.x), grid = static_cast<int>(gridDim.x);
  int shares = 1;
  // Where share i begins: total * i / shares. Totals of fewer shares than CTAs are small.
  auto cut_at = [&](int i) {
    const unsigned long long n = static_cast<unsigned long long>(total) * static_cast<unsigned>(i);
    return static_cast<long long>(shares == grid ? __umul64hi(n, p.by_grid) : static_cast<unsigned>(n) / static_cast<unsigned>(shares));
  };
  if constexpr (!kClustered) {
    // A thread sums up a run of consecutive sequences.
    const int per_thread = (a.batch.sequences + kWarps * 32 - 1) / (kWarps * 32);
    const int first_mine = min(a.batch.sequences, static_cast<int>(threadIdx.x) * per_thread), end_mine = min(a.batch.sequences, first_mine + per_thread);
    long long mine = 0;
#pragma unroll 4
    for (int i = first_mine; i < end_mine; ++i) mine += rows_units<kRows>(p, paged_sequence(a.batch, a.cache, i, a.refused, false)).weight;
    if (blockIdx.x == 0)
      for (int i = first_mine; i < end_mine; ++i) paged_sequence(a.batch, a.cache, i, a.refused, true);
    long long before = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, before, off);
      if (lane >= off) before += other;
    }
    if (lane == 31) warp_totals[warp] = before;
    if (threadIdx.x == 0) start_sequence = -1;
    __syncthreads();
    before -= mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += warp_totals[w];
      total += warp_totals[w];
    }
    shares = total >= static_cast<long long>(kLeastSteps) * grid ? grid : max(1, static_cast<int>(total) / kLeastSteps);
    at = index < shares ? cut_at(index) : total;
    share_end = index < shares ? cut_at(index + 1) : total;
    if (at < share_end && before <= at && at < before + mine) {
      for (int i = first_mine; i < end_mine; ++i) {
        const PagedSequence sequence = paged_sequence(a.batch, a.cache, i, a.refused, false);
        const long long weight = rows_units<kRows>(p, sequence).weight;
        if (at < before + weight) {
          start_sequence = i;
          start_prefix = before;
          break;
        }
        before += weight;
      }
    }
    __syncthreads();
    s = start_sequence;
    prefix = s >= 0 ? start_prefix : 0;
  } else {
    s = static_cast<int>(blockIdx.y) / a.cache.kv_heads;
  }
  uint64_t policy = 0;
  RowsSplit split = {};

  const uint32_t ring_addr = smem_u32(smem + warp * S::kRingBytes);
  float *records = reinterpret_cast<float *>(smem + S::kRecordsOff);   // [warp][8][kRecord]

  // The part of a unit that lies in the share: steps [step0, step1) of `steps`, of which this warp takes every fourth tile.
  struct Part {
    PagedSequence sequence;
    int kv_head, row_tile, row0, rows;     // first packed row, rows there are
    int step0, step1, steps, left;         // left: work of the unit behind the share
    int first_key, key_end, tiles;         // this warp's
  } part = {};
  const int *pages = nullptr;
  const uint16_t *k_base = nullptr, *v_base = nullptr;
  auto settle_part = [&]() {
    part.row0 = part.row_tile * kRows;
    part.rows = static_cast<int>(min(static_cast<long long>(part.sequence.count) * p.group - part.row0, static_cast<long long>(kRows)));
    // keys that the tile's last token sees bound what is read
    const int tile_keys = min(part.sequence.keys, paged_visible(part.sequence, (part.row0 + part.rows - 1) / p.group, a.causal));
    part.key_end = min(tile_keys, part.step1 * kStepKeys);
    part.first_key = part.step0 * kStepKeys + warp * kTileKeys;
    part.tiles = part.key_end > part.first_key ? (part.key_end - part.first_key + kStepKeys - 1) / kStepKeys : 0;
    policy = l2_policy(static_cast<long long>(part.sequence.count) * p.group > kRows);
    pages = a.batch.page_table + s * a.batch.table_stride;
    k_base = static_cast<const uint16_t *>(a.cache.k) + part.kv_head * a.cache.k_head;
    v_base = static_cast<const uint16_t *>(a.cache.v) + part.kv_head * a.cache.v_head;
  };
  auto next_part = [&]() {
    if constexpr (kClustered) {
      // The next tile of rows of the sequence; every CTA of the cluster has a part of it, be it empty.
      part.kv_head = static_cast<int>(blockIdx.y) - s * a.cache.kv_heads;
      part.sequence = paged_sequence(a.batch, a.cache, s, a.refused, blockIdx.x == 0 && part.kv_head == 0);
      if (static_cast<long long>(next_tile) * kRows >= static_cast<long long>(part.sequence.count) * p.group) return false;
      part.row_tile = next_tile++;
      part.steps = rows_units<kRows>(p, part.sequence).steps;
      part.step0 = static_cast<int>(static_cast<long long>(part.steps) * blockIdx.x / kCluster);
      part.step1 = static_cast<int>(static_cast<long long>(part.steps) * (blockIdx.x + 1) / kCluster);
      settle_part();
      return true;
    } else {
      while (s >= 0 && at < share_end) {
        part.sequence = paged_sequence(a.batch, a.cache, s, a.refused, false);
        const RowsUnits units = rows_units<kRows>(p, part.sequence);
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
        settle_part();
        return true;
      }
      return false;
    }
  };
  // The page of a tile (kAligned: pages are whole tiles) or of the lane's key of it, looked up one tile ahead of its copies.
  auto look_up = [&](int tile) {
    const int key = part.first_key + tile * kStepKeys + (kAligned ? 0 : lane & 15);
    return tile < part.tiles && key < part.key_end ? pages[key / a.cache.page_size] : -1;
  };
  auto issue_tile = [&](int tile, int slot, int page) {
    if (tile < part.tiles) {
      const int key0 = part.first_key + tile * kStepKeys;
      const uint32_t k_dst = ring_addr + slot * (2 * S::kTileBytes), v_dst = k_dst + S::kTileBytes;
      const int own_key = key0 + (lane & 15);
      const bool inside = page >= 0 && page < a.cache.pages;
      if (!inside && own_key < part.key_end) raise_status(a.refused, kRefusedPage);
      const unsigned int seen = __ballot_sync(0xffffffffu, inside && own_key < part.key_end) & 0xffffu;
      if (lane == 0) seen_keys[warp][slot] = static_cast<int>(seen);
      const int in_page = (kAligned ? key0 : own_key) % a.cache.page_size;
      const int64_t k_row = (inside ? page : 0) * a.cache.k_page + in_page * a.cache.k_row;
      const int64_t v_row = (inside ? page : 0) * a.cache.v_page + in_page * a.cache.v_row;
      constexpr int kChunks = S::kRowBytes / 16, kRowsAtOnce = 32 / kChunks;
#pragma unroll
      for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
        const int r = i * kRowsAtOnce + lane / kChunks, c = lane % kChunks;
        int64_t k_at, v_at;
        if constexpr (kAligned) {
          k_at = k_row + r * a.cache.k_row;
          v_at = v_row + r * a.cache.v_row;
        } else {
          k_at = __shfl_sync(0xffffffffu, k_row, r);
          v_at = __shfl_sync(0xffffffffu, v_row, r);
        }
        const bool reads = (seen >> r) & 1u;         // other rows are zeros
        cp_async16_hint(policy, k_dst + tile_offset<S::kRowBytes>(r, c), k_base + (reads ? k_at + c * 8 : 0), reads ? 16u : 0u);
        cp_async16_hint(policy, v_dst + tile_offset<S::kRowBytes>(r, c), v_base + (reads ? v_at + c * 8 : 0), reads ? 16u : 0u);
      }
    }
    cp_async_commit();
  };
  int page = -1;                                       // of the next tile to be issued
  auto fill_ring = [&]() {
    page = look_up(0);
#pragma unroll 1
    for (int i = 0; i < S::kStages; ++i) {
      const int next = look_up(i + 1);
      issue_tile(i, i, page);
      page = next;
    }
  };

  bool more = next_part();
  if (more) fill_ring();
  while (more) {
    constexpr int kHalves = kNarrow ? 1 : 2;           // softmax rows per lane: g (and g + 8)
    constexpr int kAccs = kNarrow ? kD / 16 : kD / 8;  // fragments: 16 elements x 8 rows, or 16 rows x 8 elements
    float m_run[kHalves], l_run[kHalves], acc[kAccs][4];
    int last_key[kHalves];                             // last key the lane's row sees
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      m_run[h] = -INFINITY;
      l_run[h] = 0.f;
      last_key[h] = paged_visible(part.sequence, (part.row0 + g + 8 * h) / p.group, a.causal) - 1;
    }
#pragma unroll
    for (int j = 0; j < kAccs; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    // The tile's rows as A fragments (rows behind the last are zero).
    uint32_t q_frag[kD / 16][4];
    {
      const uint32_t *rows[2] = {nullptr, nullptr};
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const int packed = part.row0 + g + 8 * h, token = packed / p.group;
        if (g + 8 * h < part.rows)
          rows[h] = reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(a.q) + static_cast<int64_t>(part.sequence.begin + token) * a.q_token +
                                                       (part.kv_head * p.group + packed - token * p.group) * a.q_head) + t;
      }
#pragma unroll
      for (int ks = 0; ks < kD / 16; ++ks) {
        q_frag[ks][0] = rows[0] ? rows[0][ks * 8] : 0u;
        q_frag[ks][1] = rows[1] ? rows[1][ks * 8] : 0u;
        q_frag[ks][2] = rows[0] ? rows[0][ks * 8 + 4] : 0u;
        q_frag[ks][3] = rows[1] ? rows[1][ks * 8 + 4] : 0u;
      }
    }

    int slot = 0;
#pragma unroll 1
    for (int tile = 0; tile < part.tiles; ++tile) {
      const int next = look_up(tile + S::kStages + 1);
      cp_async_wait<S::kStages - 1>();
      __syncwarp();
      const uint32_t k_src = ring_addr + slot * (2 * S::kTileBytes), v_src = k_src + S::kTileBytes;
      const int key0 = part.first_key + tile * kStepKeys + 2 * t;
      const unsigned int seen = static_cast<unsigned int>(seen_keys[warp][slot]) >> (2 * t);
      float dot[2][2][4] = {};                         // even and odd k-steps apart: four short chains
#pragma unroll
      for (int ks = 0; ks < kD / 16; ++ks) {
        const int mi = lane >> 3;
        uint32_t bfrag[4];
        ldmatrix_x4(k_src + tile_offset<S::kRowBytes>((mi >> 1) * 8 + (lane & 7), 2 * ks + (mi & 1)), bfrag);
        mma_16816<kBf16>(dot[ks & 1][0], q_frag[ks], bfrag[0], bfrag[1]);
        mma_16816<kBf16>(dot[ks & 1][1], q_frag[ks], bfrag[2], bfrag[3]);
      }
      float alpha[kHalves], pr[kHalves][4];            // keys 2t, 2t + 1, 8 + 2t, 9 + 2t
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        float sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int offset = (i >> 1) * 8 + (i & 1);
          sc[i] = (dot[0][i >> 1][2 * h + (i & 1)] + dot[1][i >> 1][2 * h + (i & 1)]) * p.scale_log2;
          if (!((seen >> offset) & 1u) || key0 + offset > last_key[h]) sc[i] = -INFINITY;
        }
        float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = fmaxf(top, m_run[h]), m_exp = m_new == -INFINITY ? 0.f : m_new;
        alpha[h] = exp2_fast(m_run[h] - m_exp);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pr[h][i] = exp2_fast(sc[i] - m_exp);
          sum += pr[h][i];
        }
        l_run[h] = l_run[h] * alpha[h] + sum;
        m_run[h] = m_new;
      }
      // Probabilities are rounded to the storage type for the product with V, whose MMA takes both operands in one type; the sum
      // keeps them in f32. Error against 64 bits (2-norm, the result's own rounding in it): f16 2.8e-4 where f32 ones have 2.1e-4.
      if constexpr (kNarrow) {
        const uint32_t p_lo = pack2<kBf16>(pr[0][0], pr[0][1]), p_hi = pack2<kBf16>(pr[0][2], pr[0][3]);
        const float alpha0 = __shfl_sync(0xffffffffu, alpha[0], 8 * t), alpha1 = __shfl_sync(0xffffffffu, alpha[0], 8 * t + 4);   // rows 2t, 2t + 1
#pragma unroll
        for (int j = 0; j < kAccs; ++j) {
          const int mi = lane >> 3;
          uint32_t vfrag[4];
          ldmatrix_x4_trans(v_src + tile_offset<S::kRowBytes>((mi >> 1) * 8 + (lane & 7), 2 * j + (mi & 1)), vfrag);
          acc[j][0] *= alpha0; acc[j][1] *= alpha1; acc[j][2] *= alpha0; acc[j][3] *= alpha1;
          mma_16816<kBf16>(acc[j], vfrag, p_lo, p_hi);
        }
      } else {
        const uint32_t p_frag[4] = {pack2<kBf16>(pr[0][0], pr[0][1]), pack2<kBf16>(pr[kHalves - 1][0], pr[kHalves - 1][1]),
                                    pack2<kBf16>(pr[0][2], pr[0][3]), pack2<kBf16>(pr[kHalves - 1][2], pr[kHalves - 1][3])};
#pragma unroll
        for (int j = 0; j < kAccs; ++j) {
          acc[j][0] *= alpha[0]; acc[j][1] *= alpha[0];
          acc[j][2] *= alpha[kHalves - 1]; acc[j][3] *= alpha[kHalves - 1];
        }
#pragma unroll
        for (int j = 0; j < kAccs; j += 2) {
          const int mi = lane >> 3;
          uint32_t vfrag[4];
          ldmatrix_x4_trans(v_src + tile_offset<S::kRowBytes>((mi & 1) * 8 + (lane & 7), j + (mi >> 1)), vfrag);
          mma_16816<kBf16>(acc[j], p_frag, vfrag[0], vfrag[1]);
          mma_16816<kBf16>(acc[j + 1], p_frag, vfrag[2], vfrag[3]);
        }
      }
      __syncwarp();   // every lane has read the slot
      issue_tile(tile + S::kStages, slot, page);
      page = next;
      if (++slot == S::kStages) slot = 0;
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
    }
    // The next part's first tiles are on their way while this one's state is put together. (The ring's groups of copies have all
    // been waited for but the empty ones behind the last tile.)
    const Part done = part;
    more = next_part();
    if (more) fill_ring();
    const bool whole = done.step0 == 0 && done.step1 == done.steps;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {                // eight rows at a time
      __syncthreads();                                 // the records of the rows before have been read
      float *mine_records = records + warp * (8 * S::kRecord);
      if constexpr (kNarrow) {
#pragma unroll
        for (int j = 0; j < kAccs; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) mine_records[(2 * t + (i & 1)) * S::kRecord + j * 16 + g + 8 * (i >> 1)] = acc[j][i];
      } else {
#pragma unroll
        for (int j = 0; j < kAccs; ++j) *reinterpret_cast<float2 *>(mine_records + g * S::kRecord + j * 8 + 2 * t) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
      }
      if (t == 0) *reinterpret_cast<float2 *>(mine_records + g * S::kRecord + kD) = make_float2(m_run[h], l_run[h]);
      __syncthreads();
      // Fold over the warps, a warp per row, with the row's maximum as the common exponent reference.
      for (int r = warp; r < 8 && r + 8 * h < done.rows; r += kWarps) {
        float2 ml[kWarps];
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          ml[w] = *reinterpret_cast<const float2 *>(records + (w * 8 + r) * S::kRecord + kD);
          top = fmaxf(top, ml[w].x);
        }
        const float m_exp = top == -INFINITY ? 0.f : top;
        float l = 0.f;
        Slice<kD> sum = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float weight = exp2_fast(ml[w].x - m_exp);
          Slice<kD> slice;
          slice.load(records + (w * 8 + r) * S::kRecord, lane);
          l = fmaf(ml[w].y, weight, l);
#pragma unroll
          for (int e = 0; e < Slice<kD>::kPer; ++e) sum.v[e] = fmaf(slice.v[e], weight, sum.v[e]);
        }
        const int row = r + 8 * h;
        if constexpr (kClustered) {                    // over the first warp's record, which this warp has read
          sum.store(records + r * S::kRecord, lane);
          if (lane == 0) *reinterpret_cast<float2 *>(records + r * S::kRecord + kD) = make_float2(top, l);
        } else if (whole) {
          const int packed = done.row0 + row, token = packed / p.group;
          write_row<kBf16, kD>(a, done.sequence.begin + token, done.kv_head * p.group + packed - token * p.group, lane, top, l, sum);
        } else {
          float *record = p.records + ((static_cast<int64_t>(blockIdx.x) * 2 + (done.step0 == 0 ? 1 : 0)) * kRows + row) * S::kRecord;
          sum.store(record, lane);
          if (lane == 0) *reinterpret_cast<float2 *>(record + kD) = make_float2(top, l);
        }
      }
      if constexpr (kClustered) {
        cluster_sync_all();                            // the CTAs' states are in their shared memory
        if (blockIdx.x == 0) {
          for (int r = warp; r < 8 && r + 8 * h < done.rows; r += kWarps) {
            const uint32_t local = smem_u32(records + r * S::kRecord);
            float2 ml = make_float2(-INFINITY, 0.f);   // of CTA `lane`
            if (lane < kCluster) ml = ld_cluster_f32x2(cluster_map_shared(local + kD * 4, lane));
            float top = ml.x;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float weight = exp2_fast(ml.x - (top == -INFINITY ? 0.f : top));
            float l = ml.y * weight;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
            Slice<kD> sum = {};
#pragma unroll
            for (int c = 0; c < kCluster; ++c) {
              Slice<kD> slice;
              slice.load_cluster(cluster_map_shared(local, c), lane);
              const float w = __shfl_sync(0xffffffffu, weight, c);
#pragma unroll
              for (int e = 0; e < Slice<kD>::kPer; ++e) sum.v[e] = fmaf(slice.v[e], w, sum.v[e]);
            }
            const int packed = done.row0 + r + 8 * h, token = packed / p.group;
            write_row<kBf16, kD>(a, done.sequence.begin + token, done.kv_head * p.group + packed - token * p.group, lane, top, l, sum);
          }
        }
        cluster_sync_all();                            // and are kept until they have been read
      }
    }
    if (!kClustered && done.step0 == 0 && !whole) {
      // The unit ends the share and goes on in the CTAs behind this one, up to the last share that begins in front of its end.
      int behind = 0;
#pragma unroll 1
      for (int start = index + 1;; start += 32) {
        const unsigned int inside = __ballot_sync(0xffffffffu, start + lane < shares && cut_at(start + lane) < share_end + done.left);
        behind += __popc(inside);
        if (inside != 0xffffffffu) break;
      }
      split = {1 + behind, done.sequence.begin, done.sequence.count, done.row_tile, done.kv_head, {}};
    }
  }
  cp_async_wait<0>();
  if (!kClustered && threadIdx.x == 0) p.splits[blockIdx.x] = split;
}

// Folds the records of the unit that starts in share blockIdx.x and goes on in the shares behind it: row blockIdx.y, a thread
// per element. Every warp weighs 32 records at a time with a lane each; the records' elements are loaded eight at a time.
template <bool kBf16, int kD, bool kNarrow>
__global__ void __launch_bounds__(kD) attention_paged_fold_kernel(const __grid_constant__ RowsParams p) {
  using S = RowsShape<kD>;
  constexpr int kRows = kNarrow ? 8 : 16;
  pdl_wait();
  pdl_launch_dependents();
  const RowsSplit split = p.splits[blockIdx.x];
  const int lane = threadIdx.x & 31, r = blockIdx.y;
  const int packed = split.tile * kRows + r, token = packed / p.group;
  if (split.records == 0 || token >= split.count) return;
  // record 0: the start (slot 1) of the first share; the others: the ends (slot 0) of the shares behind it
  const float *base = p.records + (static_cast<int64_t>(blockIdx.x) * 2 * kRows + r) * S::kRecord;
  auto record = [&](int i) { return base + (i == 0 ? kRows * S::kRecord : static_cast<int64_t>(i) * 2 * kRows * S::kRecord); };
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

using RowsKernel = void (*)(const RowsParams);
template <bool kBf16, int kD, bool kNarrow, bool kClustered>
constexpr RowsKernel rows_kernel(bool aligned) {
  return aligned ? attention_paged_rows_kernel<kBf16, kD, kNarrow, true, kClustered> : attention_paged_rows_kernel<kBf16, kD, kNarrow, false, kClustered>;
}
#define WB200_ROWS_KERNELS(D, NARROW, CLUSTERED)                                                                          \
  {{rows_kernel<false, D, NARROW, CLUSTERED>(false), rows_kernel<false, D, NARROW, CLUSTERED>(true)},                     \
   {rows_kernel<true, D, NARROW, CLUSTERED>(false), rows_kernel<true, D, NARROW, CLUSTERED>(true)}}
const RowsKernel kRowsKernels[2][2][2][2][2] = {   // [clustered][head_dim 128][narrow][bf16][aligned]
    {{WB200_ROWS_KERNELS(64, false, false), WB200_ROWS_KERNELS(64, true, false)}, {WB200_ROWS_KERNELS(128, false, false), WB200_ROWS_KERNELS(128, true, false)}},
    {{WB200_ROWS_KERNELS(64, false, true), WB200_ROWS_KERNELS(64, true, true)}, {WB200_ROWS_KERNELS(128, false, true), WB200_ROWS_KERNELS(128, true, true)}}};
const RowsKernel kFoldKernels[2][2][2] = {      // [head_dim 128][narrow][bf16]
    {{attention_paged_fold_kernel<false, 64, false>, attention_paged_fold_kernel<true, 64, false>},
     {attention_paged_fold_kernel<false, 64, true>, attention_paged_fold_kernel<true, 64, true>}},
    {{attention_paged_fold_kernel<false, 128, false>, attention_paged_fold_kernel<true, 128, false>},
     {attention_paged_fold_kernel<false, 128, true>, attention_paged_fold_kernel<true, 128, true>}}};

constexpr int kCtasPerSm = 2;
size_t rows_record_bytes(int sm_count) { return static_cast<size_t>(sm_count) * kCtasPerSm * 2 * 16 * (128 + 4) * sizeof(float); }

}  // namespace

bool attention_paged_rows_supports(const AttentionPagedArgs &a) {
  if (a.cache.head_dim != 64 && a.cache.head_dim != 128) return false;
  const uint64_t bits = reinterpret_cast<uintptr_t>(a.cache.k) | reinterpret_cast<uintptr_t>(a.cache.v) | reinterpret_cast<uintptr_t>(a.q) |
                        reinterpret_cast<uintptr_t>(a.out) |
                        static_cast<uint64_t>((a.cache.k_page | a.cache.k_row | a.cache.k_head | a.cache.v_page | a.cache.v_row | a.cache.v_head |
                                               a.q_token | a.q_head | a.out_token | a.out_head) * 2);
  return (bits & 15u) == 0;     // rows begin on 16 bytes
}

// Clusters where all units' are resident at once (clusters of eight leave a part of every GPC unused) and, at the longest the
// page table can hold, an eighth of a unit's keys through one CTA (39 bytes / ns) does not take longer than all keys through the
// whole GPU (6500 bytes / ns) and the second launch (4 us). One launch and two, head_dim 128, 16-row pages, per call in a graph:
// 1 x 8 KV heads, 500 / 2000 / 4000 / 16000 keys 5.6 / 7.7 / 11.0 / 31.8 and 10.0 / 9.7 / 11.0 / 20.5 us; 4 x 8, 1000 / 4000 / 32000
// keys 7.2 / 16.4 / 84.7 and 11.0 / 19.2 / 87.0 us. Those sequences are equally long: the host does not know the lengths, and one long
// sequence among short ones is worse off in clusters, eight CTAs to its KV head (4 x 8, one of 32000 keys and three of 500: 68.7 and
// 26.8 us). Nor does a table wider than the longest sequence say so (3 x 4 of up to 2000 keys, room for 4800 / 6400: 8.1 / 10.0 us).
bool attention_paged_rows_clustered(const AttentionPagedArgs &a, int sm_count) {
  const int64_t units = static_cast<int64_t>(a.batch.sequences) * a.cache.kv_heads;
  if (units * kCluster > sm_count * kCtasPerSm * 7 / 8) return false;
  const double unit_bytes = 4.0 * a.cache.head_dim * a.cache.page_size * a.batch.table_width;
  return unit_bytes / kCluster / 39.0 <= static_cast<double>(units) * unit_bytes / 6500.0 + 4000.0;
}

size_t attention_paged_rows_workspace(int sm_count) { return rows_record_bytes(sm_count) + static_cast<size_t>(sm_count) * kCtasPerSm * sizeof(RowsSplit); }

wb200_status launch_attention_paged_rows(const AttentionPagedArgs &a, int sm_count, cudaStream_t stream) {
  RowsParams p{};
  p.a = a;
  p.group = a.q_heads / a.cache.kv_heads;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.by_grid = ~0ull / static_cast<unsigned>(sm_count * kCtasPerSm) + 1;
  p.records = static_cast<float *>(a.workspace);
  p.splits = reinterpret_cast<RowsSplit *>(static_cast<uint8_t *>(a.workspace) + rows_record_bytes(sm_count));
  // Tiles of 8 rows where a sequence's rows fit one, as far as the caller says.
  const bool narrow = static_cast<int64_t>(p.group) * (a.batch.max_query > 0 ? a.batch.max_query : 1) <= 8;
  const int wide = a.cache.head_dim == 128 ? 1 : 0, bf16 = a.cache.format == WB200_BF16 ? 1 : 0;
  static PerDeviceOnce attributes;
  const wb200_status st = attributes.run([]() -> wb200_status {
    for (int d = 0; d < 2; ++d)
      for (int n = 0; n < 2; ++n)
        for (int b = 0; b < 2; ++b)
          for (int al = 0; al < 2; ++al)
            for (int c = 0; c < 2; ++c)
              WB200_CUDA_CHECK(cudaFuncSetAttribute(kRowsKernels[c][d][n][b][al], cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                    d ? RowsShape<128>::kSmemBytes : RowsShape<64>::kSmemBytes));
    return WB200_OK;
  });
  if (st != WB200_OK) return st;
  const size_t smem = wide ? RowsShape<128>::kSmemBytes : RowsShape<64>::kSmemBytes;
  const bool aligned = a.cache.page_size % kTileKeys == 0;
  if (attention_paged_rows_clustered(a, sm_count)) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(kCluster, static_cast<unsigned>(a.batch.sequences) * a.cache.kv_heads);
    config.blockDim = dim3(kWarps * 32);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes_of[2];
    attributes_of[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes_of[0].val.programmaticStreamSerializationAllowed = 1;
    attributes_of[1].id = cudaLaunchAttributeClusterDimension;
    attributes_of[1].val.clusterDim.x = kCluster; attributes_of[1].val.clusterDim.y = 1; attributes_of[1].val.clusterDim.z = 1;
    config.attrs = attributes_of;
    config.numAttrs = 2;
    WB200_CUDA_CHECK(cudaLaunchKernelEx(&config, kRowsKernels[1][wide][narrow][bf16][aligned], p));
    return WB200_OK;
  }
  const unsigned grid = static_cast<unsigned>(sm_count * kCtasPerSm);
  WB200_CUDA_CHECK(launch_dependent(kRowsKernels[0][wide][narrow][bf16][aligned], grid, kWarps * 32, smem, stream, p));
  WB200_CUDA_CHECK(launch_dependent(kFoldKernels[wide][narrow][bf16], dim3(grid, narrow ? 8 : 16), a.cache.head_dim, 0, stream, p));
  return WB200_OK;
}

}  // namespace wb200
