// Attention of chunks of new tokens over a paged KV cache on tcgen05 tensor cores (bf16 / f16, head_dim 64 and 128): the kernel and its
// fold. Two launches take it, one for caches of the type itself and one for caches held in four bits.
//
// The arithmetic of a tile is that of the prefill kernel (attention_fa.cu): S = Q K^T in TMEM, a thread per row for the
// softmax with a lagging exponent reference, the rounded P back into TMEM as the A operand of P V. What differs is what the
// rows and the tiles are:
//   rows     The rows that share a KV head, (token, query head of its group), are packed: row r of a tile is token r / group,
//            head r % group, 128 / group tokens to a tile. A chunk of 64 tokens of a group of 4 fills the two tiles of an item,
//            which then reads its keys once instead of four times; Q comes in by one TMA box per tile and half.
//   keys     A 128-key tile is one TMA box per page part of 2^n rows that divides both (whole tiles of 128-row pages, sixteen
//            boxes at 8). K and V have a loader warp each, whose lanes look up a page each, one tile ahead.
//   tails    Rows behind a sequence's last key are not masked by TMA's fill, as the page goes on, and 0 * v is not 0 for what a
//            stale row may hold. The V loader zeroes those rows in shared memory before the products see them.
//   halves   An item is two row tiles of one KV head of one sequence, so that one tile's products run under the other's softmax.
//            Where the sequence has rows for one tile only, its odd key tiles take the second tile's place, and the two halves
//            of the state are joined at the end, by both tiles' warps, half of the columns each: a step of one row tile takes
//            1820 clocks instead of nearly the 3250 of two.
//   codes    Of a cache held in four bits (kQuantized) eight decoder warps, four for K and four for V, take the loaders' place: they
//            read codes, and write their values, rounded to the type as the products want them, where TMA would write the rows.
//   shares   All items lie one behind the other on one axis of work, cut into equal shares for the CTAs, so ragged batches and
//            few long items fill the GPU alike. Each CTA finds its share from the lengths on the device. A cut near the end of
//            an item moves to it; others leave f32 records of the item's parts, folded by a second kernel.
// Results depend on the lengths and the number of SMs only: repeats give the same bits.
// With codes a step of two row tiles takes 4500 clocks, of one 3050: the decoders share the schedulers with the softmax (their work left
// out, 3900). All loops together have to stay in the instruction cache: decoders with code of their own for V, which needs fewer
// instructions in another order of the columns, took 6200 clocks, unrolled twice 8700.
// Bound: the chain S -> softmax -> P V of a step (see attention_fa.cu), 4 * head_dim flop per visible (row, key) pair. A step of two
// row tiles takes 3250 clocks, of which its products are 2048. 4096 tokens behind 32768 cached ones, 32/8 heads: 1.9 ms back to
// back in a graph (1.2 PFLOP/s), 2.2 ms among other work (the clock gives way to the power cap); 8 chunks of 256 tokens at 4096 keys
// 132 us, the tensor pipe 54 % busy, of which about 9 us are the start, the cuts' records and their fold.
#pragma once

#include <type_traits>

#include "attention_paged.cuh"
#include "quantized_rows.cuh"

namespace wb200 {
namespace {

constexpr int kTileM = 128;                     // packed rows per Q tile (TMEM lanes)
constexpr int kTileN = 128;                     // keys per tile
constexpr int kBlockBytes = 128 * 128;          // [128 rows][128 B], swizzled
constexpr int kOutStageBytes = 32 * 128;        // a softmax warp's 32 rows x 64 columns of output
// Warps: Q and K loader, MMA, V loader, scheduler, 2 x 4 softmax; behind them, for codes, four decoders of K and four of V.
template <bool kQuantized>
constexpr int kChunkThreads = kQuantized ? 640 : 384;
constexpr int kDecoders = 4;                    // warps to an operand
constexpr int kSegments = 4;                    // segments handed out and not yet taken in by every warp
template <bool kQuantized>
constexpr int kReaders = kQuantized ? 10 + 2 * kDecoders : 11;   // warps that take them
constexpr int kPParts = 2;
constexpr int kFirstChunks = 3;                 // 32-key chunks of the first part of P, of 4
constexpr uint32_t kColS0 = 0, kColO0 = 256;    // S_t at 128 t, O_t at 256 + 128 t
constexpr int kMaxSequences = 4096;             // staged in shared memory
// Work, in twelfths of a step of two row tiles (3250 clocks; 4500 with codes to decode): a key tile of two row tiles, of one (1820
// clocks; 3050), and what an item costs by itself (its Q, the first scores, the write-out: 4700). With codes the clocks say 8 twelfths for
// one row tile and 13 for an item; of weights 6 to 9 and 14 to 32 tried, 7 and 24 were the shortest over seven mixed batches (40 decoding
// sequences beside 8 chunks: 8 and 14 438 us, 7 and 24 425).
constexpr int kPairWork = 12, kSingleWork = 7;
template <bool kQuantized>
constexpr int kItemWork = kQuantized ? 24 : 18;
constexpr int kLeastWork = 24;                  // no share is made smaller
constexpr int kLeastCut = 12;                   // a cut this near to an end of an item moves there
// What cutting items costs a launch: the records' write-out, one more item to begin in each CTA, and the fold behind the last
// CTA, about 11 us or six steps of two tiles (four and a half of the longer ones).
template <bool kQuantized>
constexpr int kCutWork = kQuantized ? 54 : 72;

template <int kHd>
struct Shape {
  static constexpr int kHalves = kHd / 64;                   // 64-element column blocks
  static constexpr int kTileBytes = kHalves * kBlockBytes;
  static constexpr int kSlots = 8 / kHalves;                 // 128 KiB of K and V tiles
  static constexpr int kQOff = 0;
  static constexpr int kRingOff = 2 * kTileBytes;
  static constexpr int kOutOff = kRingOff + kSlots * kTileBytes;
  static constexpr int kBarOff = kOutOff + 8 * kOutStageBytes;
  static constexpr int kSegmentOff = kBarOff + 512;
  static constexpr size_t kBytes = kSegmentOff + kSegments * 64 + 1024;
  static_assert(kBytes <= 227 * 1024, "a CTA's shared memory");
  static constexpr int kRecordFloats = kTileM * kHd + 2 * kTileM;   // acc as [kHd / 4][128 rows][4], then (m, l) per row
  static_assert(kMaxSequences * 24 <= kSlots * kTileBytes, "the staged lengths must fit the ring");
};

// What the fold has to know about the item that a CTA's share ends inside of; `records` 0: none.
struct ChunkSplit {
  int records, begin, count, pair, kv_head, halved, reserved[2];
};

struct ChunkParams {
  AttentionPagedArgs a;
  int group, tile_tokens;          // query heads per KV head; tokens per Q tile
  unsigned long long by_group;     // 2^32 / group + 1: row / group = row * by_group >> 32 for the rows of a tile
  unsigned long long by_grid;      // floor((2^64 - 1) / grid) + 1: n / grid = n * by_grid >> 64 for n < 2^56
  int box_rows;                    // keys per TMA box
  int rows_inside;                 // the cache's tensor maps have rows inside heads
  float scale_log2;
  float *records;                  // [grid][2][2 tiles][kRecordFloats]: a share's end of an item (0), its start of one (1)
  ChunkSplit *splits;              // [grid]
};

struct QuantizedChunkParams : ChunkParams {
  QuantizedRowsArgs rows;
};

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <int kRegs>
__device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
__device__ __forceinline__ unsigned long long pack_f32x2(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(unsigned long long v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "setp.ne.b32 P, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, P;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z, int w, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void ld_shared_v4(uint32_t src, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src) : "memory");
}

// Token of a packed row, within its tile.
__device__ __forceinline__ int token_of(const ChunkParams &p, int row) { return static_cast<int>(row * p.by_group >> 32); }
// 128-key tiles that Q tile (or pair) whose last token is `last` visits.
__device__ __forceinline__ int tiles_to(int keys, int count, int causal, int last) {
  int visible = keys;
  if (causal) visible = keys - count + min(last, count - 1) + 1;
  return visible <= 0 ? 0 : (visible + kTileN - 1) / kTileN;
}

// An item: the key tiles that Q tile 0 / 1 visits. A single row tile is halved: tile t takes every second key tile, from t on.
struct Item {
  int n0, n1, steps, halved;
};
__device__ __forceinline__ Item make_item(const ChunkParams &p, int count, int keys, int pair) {
  Item item;
  const int first = pair * 2 * p.tile_tokens;
  item.halved = first + p.tile_tokens >= count;
  item.n0 = tiles_to(keys, count, p.a.causal, first + p.tile_tokens - 1);
  item.n1 = item.halved ? 0 : tiles_to(keys, count, p.a.causal, first + 2 * p.tile_tokens - 1);
  item.steps = max(1, max(item.n0, item.n1));
  return item;
}
template <bool kQuantized>
__device__ __forceinline__ int item_work(const Item &item) {
  return kItemWork<kQuantized> + item.steps * (item.halved ? kSingleWork : kPairWork);
}
// The key tile that a cut at work `x` of an item falls on; 0 and `steps` are the item's ends.
template <bool kQuantized>
__device__ __forceinline__ int cut_tile(const Item &item, int x, int least_cut) {
  const int all = item_work<kQuantized>(item), each = item.halved ? kSingleWork : kPairWork;
  if (x < kItemWork<kQuantized> + least_cut) return 0;
  if (x + least_cut > all) return item.steps;
  return min(max((x - kItemWork<kQuantized> + each / 2) / each, 1), item.steps - 1);
}

// A place between two key tiles: in front of tile `tile` of the item.
struct Place {
  int sequence, kv_head, pair, tile;
};
// One CTA's part of an item: key tiles [t0, t1) of its steps; t1 0 behind the last.
struct Segment {
  int begin, count, keys;          // the sequence
  int sequence, kv_head, pair;
  int n0, n1, halved;
  int whole;
  int t0, t1;
  __device__ __forceinline__ int of(int t) const {            // key tiles of this segment for Q tile t
    if (halved) return (max(0, min(n0, t1) - t0) + 1 - t) >> 1;
    return max(0, min(t ? n1 : n0, t1) - t0);
  }
  __device__ __forceinline__ int tiles() const { return halved ? max(0, min(n0, t1) - t0) : max(of(0), of(1)); }
};
static_assert(sizeof(Segment) <= 64, "the segments' area");
// The scheduler's walk through its CTA's share.
struct ShareWalk {
  Place at, end;                   // at.sequence == the batch's: done
  int begin, count, keys, pairs;   // of the current sequence

  __device__ __forceinline__ void look_up(const ChunkParams &p) {
    const PagedSequence s = paged_sequence(p.a.batch, p.a.cache, at.sequence, p.a.refused, false);
    enter(p, s.begin, s.count, s.keys);
  }
  __device__ __forceinline__ void enter(const ChunkParams &p, int sequence_begin, int sequence_count, int sequence_keys) {
    begin = sequence_begin; count = sequence_count; keys = sequence_keys;
    pairs = (count + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
  }
  __device__ __forceinline__ bool next(const ChunkParams &p, Segment &out) {
    while (at.sequence < p.a.batch.sequences) {
      if (count == 0 || at.kv_head == p.a.cache.kv_heads) {
        at = {next_with_tokens(p.a.batch, at.sequence + 1), 0, 0, 0};
        if (at.sequence < p.a.batch.sequences) look_up(p);
        continue;
      }
      const Item item = make_item(p, count, keys, at.pair);
      const bool last = at.sequence == end.sequence && at.kv_head == end.kv_head && at.pair == end.pair;
      out.begin = begin; out.count = count; out.keys = keys;
      out.sequence = at.sequence; out.kv_head = at.kv_head; out.pair = at.pair;
      out.n0 = item.n0; out.n1 = item.n1; out.halved = item.halved;
      out.t0 = at.tile;
      out.t1 = last ? min(end.tile, item.steps) : item.steps;
      out.whole = out.t0 == 0 && out.t1 == item.steps;
      if (last) at.sequence = p.a.batch.sequences;
      at.tile = 0;
      if (++at.pair == pairs) { at.pair = 0; ++at.kv_head; }
      if (out.t1 > out.t0) return true;
    }
    return false;
  }
};
// With codes, tmap_k and tmap_v are not looked at.
template <bool kBf16, int kHd, bool kQuantized>
__global__ void __launch_bounds__(kChunkThreads<kQuantized>, 1)
attention_paged_chunk_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                             const __grid_constant__ std::conditional_t<kQuantized, QuantizedChunkParams, ChunkParams> p) {
  using L = Shape<kHd>;
  constexpr int kThreads = kChunkThreads<kQuantized>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t *smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem);

  const uint32_t bar_base = smem_base + L::kBarOff;
  auto kv_full = [&](int s) { return bar_base + 8u * s; };
  auto kv_empty = [&](int s) { return bar_base + 8u * (L::kSlots + s); };
  auto tail_full = [&](int s) { return bar_base + 8u * (2 * L::kSlots + s); };   // a V tile whose tail is still to be zeroed
  constexpr int kFixed = 3 * L::kSlots;
  const uint32_t q_full = bar_base + 8u * kFixed;
  auto s_full = [&](int t) { return bar_base + 8u * (kFixed + 1 + t); };
  auto p_part = [&](int t, int part) { return bar_base + 8u * (kFixed + 3 + kPParts * t + part); };
  auto o_done = [&](int t) { return bar_base + 8u * (kFixed + 3 + 2 * kPParts + t); };
  const uint32_t q_empty = bar_base + 8u * (kFixed + 5 + 2 * kPParts);
  auto paired = [&](int quarter) { return bar_base + 8u * (kFixed + 6 + 2 * kPParts + quarter); };   // the two tiles' warps of the same TMEM lanes
  auto segment_full = [&](int i) { return bar_base + 8u * (kFixed + 10 + 2 * kPParts + i); };
  auto segment_empty = [&](int i) { return bar_base + 8u * (kFixed + 10 + 2 * kPParts + kSegments + i); };
  uint8_t *bar_ptr = smem + L::kBarOff;
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bar_ptr + 8 * (kFixed + 10 + 2 * kPParts + 2 * kSegments));
  volatile int *abort_word = reinterpret_cast<volatile int *>(bar_ptr + 8 * (kFixed + 11 + 2 * kPParts + 2 * kSegments));
  Segment *const segments = reinterpret_cast<Segment *>(smem + L::kSegmentOff);
  static_assert(8 * (kFixed + 12 + 2 * kPParts + 2 * kSegments) <= 512, "the barriers must fit their area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kSlots; ++s) {
      mbar_init(kv_full(s), kQuantized ? kDecoders : 1);
      mbar_init(kv_empty(s), 1);
      mbar_init(tail_full(s), 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      for (int part = 0; part < kPParts; ++part) mbar_init(p_part(t, part), kTileM / 32);
      mbar_init(o_done(t), 1);
    }
    for (int quarter = 0; quarter < 4; ++quarter) mbar_init(paired(quarter), 2);
    for (int i = 0; i < kSegments; ++i) {
      mbar_init(segment_full(i), 1);
      mbar_init(segment_empty(i), kReaders<kQuantized>);
    }
    *abort_word = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_q);
    if constexpr (!kQuantized) {
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  // ---- this CTA's share of all work; the lengths are staged in the ring's memory
  __shared__ Place cuts[2];
  __shared__ int last_share, item_count, most_work;
  __shared__ int4 first_staged;
  {
    int4 *staged = reinterpret_cast<int4 *>(smem + L::kRingOff);                                       // begin, count, keys
    long long *prefix = reinterpret_cast<long long *>(smem + L::kRingOff + kMaxSequences * sizeof(int4));   // inclusive sums of a head's work
    const int sequences = p.a.batch.sequences;
    if (threadIdx.x == 0) item_count = most_work = 0;
    __syncthreads();
    auto pairs_of = [&](int count) { return (count + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens); };
    auto pair_work = [&](int count, int keys, int pair) { return item_work<kQuantized>(make_item(p, count, keys, pair)); };
    // A lane per sequence; those of more than four items by the whole warp.
#pragma unroll 1
    for (int start = warp * 32; start < sequences; start += kThreads) {
      const int s = start + lane;
      PagedSequence q = {0, 0, 0};
      if (s < sequences) {
        q = paged_sequence(p.a.batch, p.a.cache, s, p.a.refused, blockIdx.x == 0);
        staged[s] = make_int4(q.begin, q.count, q.keys, 0);
      }
      const int pairs = pairs_of(q.count);
      long long work = 0;
      int most = 0;
      if (pairs <= 4) {
#pragma unroll 1
        for (int pair = 0; pair < pairs; ++pair) {
          const int mine = pair_work(q.count, q.keys, pair);
          work += mine;
          most = max(most, mine);
        }
      }
      unsigned int long_ones = __ballot_sync(0xffffffffu, pairs > 4);
      while (long_ones) {
        const int from = __ffs(long_ones) - 1;
        long_ones &= long_ones - 1;
        const int count = __shfl_sync(0xffffffffu, q.count, from), keys = __shfl_sync(0xffffffffu, q.keys, from), all = pairs_of(count);
        long long sum = 0;
#pragma unroll 1
        for (int pair = lane; pair < all; pair += 32) {
          const int mine = pair_work(count, keys, pair);
          sum += mine;
          most = max(most, mine);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane == from) work = sum;
      }
      if (s < sequences) prefix[s] = work;
      const int items = __reduce_add_sync(0xffffffffu, pairs) * p.a.cache.kv_heads;
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0 && items > 0) {
        atomicAdd(&item_count, items);
        atomicMax(&most_work, most);
      }
    }
    __syncthreads();
    if (warp == 0) {
      long long base = 0;
#pragma unroll 1
      for (int start = 0; start < sequences; start += 32) {
        long long value = start + lane < sequences ? prefix[start + lane] : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const long long other = __shfl_up_sync(0xffffffffu, value, off);
          if (lane >= off) value += other;
        }
        if (start + lane < sequences) prefix[start + lane] = base + value;
        base += __shfl_sync(0xffffffffu, value, 31);
      }
    }
    __syncthreads();
    // Warp 0 places the cut in front of the CTA's share, warp 1 the one behind it. Code that runs once costs what its fetch costs:
    // with whole-number divisions by way of f64 and a search by halves this took 1.7 to 2.6 us of a launch.
    if (warp < 2) {
      const int heads = p.a.cache.kv_heads, grid = static_cast<int>(gridDim.x);
      const long long total = sequences > 0 ? prefix[sequences - 1] * heads : 0;
      const int shares = total >= static_cast<long long>(kLeastWork) * grid ? grid : max(1, static_cast<int>(total) / kLeastWork);
      // Where share i begins: total * i / shares. Totals of fewer shares than CTAs are small.
      auto cut_at = [&](int i) {
        const unsigned long long n = static_cast<unsigned long long>(total) * static_cast<unsigned>(i);
        return static_cast<long long>(shares == grid ? __umul64hi(n, p.by_grid) : static_cast<unsigned>(n) / static_cast<unsigned>(shares));
      };
      // Items are left whole where the CTA with the most of them ends before one with an equal share and the cost of cuts: items
      // much alike by counting, others by what a share can grow by.
      const long long counted = static_cast<long long>(__umul64hi(item_count + grid - 1, p.by_grid)) * most_work;
      const bool alike = 10ll * most_work * item_count <= 13ll * total;
      const bool whole = alike ? (counted - kCutWork<kQuantized>) * shares <= total : most_work <= kCutWork<kQuantized>;
      const int least_cut = static_cast<int>(max(static_cast<long long>(kLeastCut), min(cut_at(1) >> 6, 1ll << 20)));
      const int index = static_cast<int>(blockIdx.x) + warp;
      const long long x = cut_at(index);
      Place place = {sequences, 0, 0, 0};
      int last = 0;
      if (index <= shares && x < total) {
        int low = 0, span = sequences;                 // the first sequence whose sum is beyond x lies in [low, low + span)
#pragma unroll 1
        while (span > 1) {
          const int step = (span + 31) >> 5;
          const int found = __ffs(__ballot_sync(0xffffffffu, prefix[low + min((lane + 1) * step, span) - 1] * heads > x)) - 1;
          low += found * step;
          span = min(step, span - found * step);
        }
        const long long before = low > 0 ? prefix[low - 1] : 0, per_head = prefix[low] - before;
        const int4 q = staged[low];
        const int pairs = pairs_of(q.y);
        place.sequence = low;
        long long rest = x - before * heads;
#pragma unroll 1
        for (int start = 1;; start += 32) {            // how many whole heads lie in front
          const unsigned int whole_heads = __ballot_sync(0xffffffffu, start + lane < heads && (start + lane) * per_head <= rest);
          place.kv_head += __popc(whole_heads);
          if (whole_heads != 0xffffffffu) break;
        }
        rest -= place.kv_head * per_head;
#pragma unroll 1
        for (int start = 0; pairs > 1; start += 32) {  // the pair of row tiles that work `rest` of the head lies in
          const int pair = start + lane;
          long long sum = pair < pairs ? pair_work(q.y, q.z, pair) : 0;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += other;
          }
          const unsigned int beyond = __ballot_sync(0xffffffffu, sum > rest);
          if (beyond || start + 32 >= pairs) {
            const int found = beyond ? __ffs(beyond) - 1 : 31;
            const long long in_front = __shfl_sync(0xffffffffu, sum, max(found - 1, 0));
            place.pair = start + found;
            if (found > 0) rest -= in_front;
            break;
          }
          rest -= __shfl_sync(0xffffffffu, sum, 31);
        }
        const Item item = make_item(p, q.y, q.z, place.pair);
        const int all = item_work<kQuantized>(item);
        place.tile = whole ? (2 * rest < all ? 0 : item.steps) : cut_tile<kQuantized>(item, static_cast<int>(rest), least_cut);
        if (warp == 0) {
          if (lane == 0) first_staged = q;
        } else if (place.tile > 0 && place.tile < item.steps) {
          // The item goes on in the shares behind this cut, up to the last whose cut does not move to its end.
          const long long end = x - rest + all - least_cut;
          last = index;
#pragma unroll 1
          for (int start = index + 1;; start += 32) {
            const unsigned int inside = __ballot_sync(0xffffffffu, start + lane < shares && cut_at(start + lane) <= end);
            last += __popc(inside);
            if (inside != 0xffffffffu) break;
          }
        }
      }
      if (lane == 0) {
        cuts[warp] = place;
        if (warp == 1) last_share = last;
      }
    }
  }
  fence_proxy_async_smem();      // the staged lengths give way to tiles
  __syncthreads();

  // The segments as the scheduler hands them out: every other warp takes them in turn.
  int segment_at = 0;
  uint32_t segment_phase = 0;
  auto take = [&](Segment &seg) {              // false behind the last, or when a wait gave up
    if (!__all_sync(0xffffffffu, mbar_wait(segment_full(segment_at), segment_phase, abort_word, 103))) return false;
    seg = segments[segment_at];
    return seg.t1 > 0;
  };
  auto give_back = [&]() {                     // this warp has no more need of the segment in shared memory
    __syncwarp();
    if (lane == 0) mbar_arrive(segment_empty(segment_at));
    if (++segment_at == kSegments) { segment_at = 0; segment_phase ^= 1u; }
  };
  auto take_working = [&](Segment &seg) {      // the next one with keys to visit, given back
    while (take(seg)) {
      give_back();
      if (seg.tiles() > 0) return true;
    }
    return false;
  };

  auto load_queries = [&](const Segment &seg, int q_bytes) {
    const int token0 = seg.begin + seg.pair * 2 * p.tile_tokens, token1 = token0 + p.tile_tokens;
    if (elect_one_sync()) {
      mbar_arrive_expect_tx(q_full, seg.halved ? q_bytes : 2 * q_bytes);
      for (int c = 0; c < L::kHalves; ++c) {
        tma_load_3d(smem_base + L::kQOff + c * kBlockBytes, &tmap_q, q_full, c * 64, seg.kv_head * p.group, token0);
        if (!seg.halved) tma_load_3d(smem_base + L::kQOff + L::kTileBytes + c * kBlockBytes, &tmap_q, q_full, c * 64, seg.kv_head * p.group, token1);
      }
    }
    __syncwarp();
  };
  // The place of the segment's tile j in the ring's order, from its first: the order in which the MMA warp takes the tiles, K and V in
  // turn, or, halved, K of the first two tiles, then V of a tile and K of the next one of its half in turn.
  auto ring_place = [](const Segment &seg, int j, int tiles, bool is_v) {
    if (!seg.halved) return 2 * j + (is_v ? 1 : 0);
    if (is_v) return j < tiles - 1 ? 2 * j + 2 : 2 * tiles - 1;
    return j < 2 ? j : 2 * j - 1;
  };

  // setmaxnreg.inc waits until the CTA's own register pool can supply the request: the totals must fit the launch's.
  constexpr int kBaseRegs = kQuantized ? 80 : 104, kSoftmaxRegs = kQuantized ? 104 : 200, kDecoderRegs = 96;
  static_assert(128 * kBaseRegs + 256 * kSoftmaxRegs + (kQuantized ? 256 * kDecoderRegs : 0) <= kThreads * (kQuantized ? 96 : 168),
                "setmaxnreg totals exceed the launch allocation");
  if (warp < 4) {
  setmaxnreg_dec<kBaseRegs>();
  if (kQuantized && (warp == 0 || warp == 2)) {
    // ------------------------------------------------------------ Q loader (warp 0)
    uint32_t q_loads = 0;
    const int q_bytes = p.tile_tokens * p.group * 128 * L::kHalves;
    Segment seg;
    while (warp == 0 && take_working(seg)) {
      if (q_loads > 0 && !__all_sync(0xffffffffu, mbar_wait(q_empty, (q_loads - 1) & 1u, abort_word, 101))) break;
      ++q_loads;
      load_queries(seg, q_bytes);
    }
  } else if (!kQuantized && (warp == 0 || warp == 2)) {
    // ------------------------------------------------------------ loaders: Q and K by warp 0, V by warp 2. Either walks as a whole
    // warp and one elected lane issues; a box costs its issuer more than 100 clocks, so two warps share them.
    const bool is_v = warp == 2;
    const CUtensorMap *map = is_v ? &tmap_v : &tmap_k;
    uint32_t position = 0;                           // of the segment's first tile in the ring's order: slot position % kSlots
    uint32_t q_loads = 0, tail_phases = 0;           // bit s: parity of the next tail in slot s
    bool ok = true;
    Segment seg;
    const int boxes = kTileN / p.box_rows;           // per tile, of 64 columns each
    const int page_size = p.a.cache.page_size;
    const int box_slot = lane * p.box_rows / page_size, box_row = lane * p.box_rows % page_size;   // lane i: box i of a tile
    const int tile_slots = kTileN / page_size, tile_rows = kTileN % page_size;
    const uint32_t box_bytes = p.box_rows * 128;
    const int q_bytes = p.tile_tokens * p.group * 128 * L::kHalves;
    while (ok && take_working(seg)) {
      const int tiles = seg.tiles();
      if (!is_v) {
        if (q_loads > 0 && !__all_sync(0xffffffffu, mbar_wait(q_empty, (q_loads - 1) & 1u, abort_word, 101))) break;
        ++q_loads;
        load_queries(seg, q_bytes);
      }
      // Keys of one pair of row tiles: 40 sequences of 5 tokens 131 -> 125 us, beside chunks 271 -> 268.
      const uint64_t policy = l2_policy(seg.count > 2 * p.tile_tokens);
      const int *pages = p.a.batch.page_table + seg.sequence * p.a.batch.table_stride;
      // Where the keys of lane i's box of a tile lie: entry of the page table, row in the page. The page is looked up a tile ahead.
      int at_slot, at_row, page;
      {
        const int first = seg.t0 * kTileN / page_size;
        at_slot = first + box_slot;
        at_row = seg.t0 * kTileN - first * page_size + box_row;
        if (at_row >= page_size) { at_row -= page_size; ++at_slot; }
      }
      int keys_left = seg.keys - seg.t0 * kTileN;
      auto look_up = [&](int left, int entry) { return lane < boxes && lane * p.box_rows < left ? pages[entry] : -1; };
      page = look_up(keys_left, at_slot);
      for (int j = 0; j < tiles && ok; ++j, keys_left -= kTileN) {
        const int row = at_row;
        at_slot += tile_slots;
        at_row += tile_rows;
        if (at_row >= page_size) { at_row -= page_size; ++at_slot; }
        const int next_page = j + 1 < tiles ? look_up(keys_left - kTileN, at_slot) : -1;
        const int count = min(boxes, (keys_left + p.box_rows - 1) / p.box_rows);    // boxes that hold a key
        if (!is_v && lane < count && (page < 0 || page >= p.a.cache.pages)) raise_status(p.a.refused, kRefusedPage);   // zeros come in for it
        const uint32_t at = position + ring_place(seg, j, tiles, is_v);
        const int slot = at % L::kSlots;
        if (!__all_sync(0xffffffffu, mbar_wait(kv_empty(slot), ((at / L::kSlots) & 1u) ^ 1u, abort_word, 102))) { ok = false; break; }
        const bool tail = is_v && keys_left < kTileN;
        const uint32_t bar = tail ? tail_full(slot) : kv_full(slot);
        uint32_t dst = smem_base + L::kRingOff + slot * L::kTileBytes;
        if (elect_one_sync()) mbar_arrive_expect_tx(bar, count * box_bytes * L::kHalves);
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < count; i += 4, dst += 4 * box_bytes) {     // the operands of four boxes first, then their copies in one go
          int box_page[4], box_at[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            box_page[u] = __shfl_sync(0xffffffffu, page, (i + u) & 31);
            box_at[u] = __shfl_sync(0xffffffffu, row, (i + u) & 31);
          }
          if (elect_one_sync()) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if (i + u >= count) break;
              const int y = p.rows_inside ? box_at[u] : seg.kv_head, z = p.rows_inside ? seg.kv_head : box_at[u];
#pragma unroll
              for (int c = 0; c < L::kHalves; ++c) tma_load_4d(dst + u * box_bytes + c * kBlockBytes, map, bar, c * 64, y, z, box_page[u], policy);
            }
          }
          __syncwarp();
        }
        if (tail) {
          // V rows behind the sequence's last key give way to zeros before the products see them.
          if (!__all_sync(0xffffffffu, mbar_wait(bar, (tail_phases >> slot) & 1u, abort_word, 105))) { ok = false; break; }
          tail_phases ^= 1u << slot;
          const uint32_t zero[4] = {0u, 0u, 0u, 0u};
          const uint32_t from = smem_base + L::kRingOff + slot * L::kTileBytes + keys_left * 128;
#pragma unroll 1
          for (int i = lane; i < (kTileN - keys_left) * 8; i += 32) {
#pragma unroll
            for (int c = 0; c < L::kHalves; ++c) st_shared_v4(from + c * kBlockBytes + i * 16, zero);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(kv_full(slot));
        }
        page = next_page;
      }
      position += 2 * tiles;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (the whole warp walks, one elected lane issues)
    {
      constexpr uint32_t idesc_s = umma_idesc_f16(kTileM, kTileN, kBf16, false, false);
      constexpr uint32_t idesc_o = umma_idesc_f16(kTileM, kHd, kBf16, false, true);
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto advance = [&]() { if (++slot == L::kSlots) { slot = 0; phase ^= 1u; } };
      const uint64_t q_desc0 = umma_desc_kmajor(smem_base + L::kQOff);
      const uint64_t q_desc1 = umma_desc_kmajor(smem_base + L::kQOff + L::kTileBytes);
      const uint64_t ring_k_desc = umma_desc_kmajor(smem_base + L::kRingOff);
      const uint64_t ring_v_desc = umma_desc_mnmajor(smem_base + L::kRingOff, kBlockBytes);
      constexpr uint32_t kSlotStep = L::kTileBytes >> 4;
      auto issue_s = [&](auto tile_tag, int k_slot, uint64_t q_desc) {
        constexpr int t = decltype(tile_tag)::value;
        const uint64_t k_desc = ring_k_desc + static_cast<uint32_t>(k_slot) * kSlotStep;
        const uint32_t d_tmem = tmem_base + kColS0 + t * 128;
        if (elect_one_sync()) {
#pragma unroll
          for (int ks = 0; ks < kHd / 16; ++ks) {
            constexpr uint32_t kBlockStep = kBlockBytes >> 4;
            const uint32_t off = (ks >> 2) * kBlockStep + (ks & 3) * 2;
            umma_f16_ss(d_tmem, q_desc + off, k_desc + off, idesc_s, ks != 0 ? 1u : 0u);
          }
          umma_commit(s_full(t));
        }
        __syncwarp();
      };
      auto issue_pv_part = [&](auto tile_tag, auto part_tag, int v_slot, bool accumulate, bool last) {
        constexpr int t = decltype(tile_tag)::value;
        constexpr int part = decltype(part_tag)::value;
        const uint64_t v_desc = ring_v_desc + static_cast<uint32_t>(v_slot) * kSlotStep;
        const uint32_t d_tmem = tmem_base + kColO0 + t * 128;
        if (elect_one_sync()) {
#pragma unroll
          for (int ks = part ? 2 * kFirstChunks : 0; ks < (part ? 8 : 2 * kFirstChunks); ++ks) {
            const uint64_t bdesc = v_desc + static_cast<uint32_t>((ks * 2048) >> 4);
            const uint32_t acc = (accumulate || ks != 0) ? 1u : 0u;
            umma_f16_ts(d_tmem, tmem_base + kColS0 + t * 128 + ks * 8, bdesc, idesc_o, acc);
          }
          if (part == kPParts - 1 && last) umma_commit(o_done(t));
        }
        __syncwarp();
      };
      auto commit = [&](uint32_t bar) {
        if (elect_one_sync()) umma_commit(bar);
        __syncwarp();
      };

      uint32_t base0 = 0, base1 = 0;
      uint32_t q_count = 0;
      Segment seg;
      using Tile0 = std::integral_constant<int, 0>;
      using Tile1 = std::integral_constant<int, 1>;
      while (ok && take_working(seg)) {
        const int n0 = seg.of(0), n1 = seg.of(1);
        const int n_max = max(n0, n1);
        ok = mbar_wait(q_full, q_count & 1u, abort_word);
        ++q_count;
        if (!seg.halved) {
          if (ok) ok = mbar_wait(kv_full(slot), phase, abort_word);
          if (ok) {
            tc_fence_after();
            if (n0 > 0) issue_s(Tile0{}, slot, q_desc0);
            if (n1 > 0) issue_s(Tile1{}, slot, q_desc1);
            commit(kv_empty(slot));
            if (n_max == 1) commit(q_empty);
            advance();
          }
          for (int j = 0; ok && j < n_max; ++j) {
            const int v_slot = slot;
            const uint32_t v_phase = phase;
            advance();
            const int k_slot = slot;
            const uint32_t k_phase = phase;
            const bool has_next = j + 1 < n_max;
            if (has_next) advance();
            if (!mbar_wait(kv_full(v_slot), v_phase, abort_word)) { ok = false; break; }
            bool k_ready = false;
            auto tile_step = [&](auto tile_tag, int n_tiles, uint32_t tile_base, uint64_t q_desc) {
              constexpr int t = decltype(tile_tag)::value;
              if (j < n_tiles) {
                if (!mbar_wait_spin(p_part(t, 0), (tile_base + j) & 1u, abort_word)) { ok = false; return; }
                tc_fence_after();
                issue_pv_part(tile_tag, Tile0{}, v_slot, j > 0, false);
                if (!mbar_wait_spin(p_part(t, 1), (tile_base + j) & 1u, abort_word)) { ok = false; return; }
                tc_fence_after();
                issue_pv_part(tile_tag, Tile1{}, v_slot, j > 0, j + 1 == n_tiles);
              }
              if (j + 1 < n_tiles) {
                if (!k_ready) {
                  if (!mbar_wait(kv_full(k_slot), k_phase, abort_word)) { ok = false; return; }
                  tc_fence_after();
                  k_ready = true;
                }
                issue_s(tile_tag, k_slot, q_desc);
              }
            };
            tile_step(Tile0{}, n0, base0, q_desc0);
            if (ok) tile_step(Tile1{}, n1, base1, q_desc1);
            if (!ok) break;
            commit(kv_empty(v_slot));
            if (has_next) commit(kv_empty(k_slot));
            if (j + 2 == n_max) commit(q_empty);
          }
        } else {
          // Both tiles' scores come from the one row tile; each has K and V tiles of its own.
          auto scores = [&](auto tile_tag) {
            if (!mbar_wait(kv_full(slot), phase, abort_word)) { ok = false; return; }
            tc_fence_after();
            issue_s(tile_tag, slot, q_desc0);
            commit(kv_empty(slot));
            advance();
          };
          auto half_step = [&](auto tile_tag, int j, int n_tiles, uint32_t tile_base) {
            constexpr int t = decltype(tile_tag)::value;
            if (!mbar_wait(kv_full(slot), phase, abort_word)) { ok = false; return; }
            if (!mbar_wait_spin(p_part(t, 0), (tile_base + j) & 1u, abort_word)) { ok = false; return; }
            tc_fence_after();
            issue_pv_part(tile_tag, Tile0{}, slot, j > 0, false);
            if (!mbar_wait_spin(p_part(t, 1), (tile_base + j) & 1u, abort_word)) { ok = false; return; }
            tc_fence_after();
            issue_pv_part(tile_tag, Tile1{}, slot, j > 0, j + 1 == n_tiles);
            commit(kv_empty(slot));
            advance();
            if (j + 1 < n_tiles) scores(tile_tag);
          };
          if (ok) scores(Tile0{});
          if (ok && n1 > 0) scores(Tile1{});
          if (ok && n0 == 1) commit(q_empty);
          for (int j = 0; ok && j < n0; ++j) {
            half_step(Tile0{}, j, n0, base0);
            if (ok && j < n1) half_step(Tile1{}, j, n1, base1);
            if (ok && j + 2 == n0) commit(q_empty);
          }
        }
        base0 += n0;
        base1 += n1;
      }
    }
  } else {
    // ------------------------------------------------------------ scheduler
    ShareWalk walk;
    walk.at = cuts[0];
    walk.end = cuts[1];
    walk.begin = walk.count = walk.keys = walk.pairs = 0;
    if (walk.at.sequence < p.a.batch.sequences) walk.enter(p, first_staged.x, first_staged.y, first_staged.z);
    ChunkSplit split = {};
    bool more = true;
    while (more) {
      Segment seg;
      more = walk.next(p, seg);
      if (!more) seg = {};
      // The share ends inside an item that it begins: the fold will want the records of the shares behind it.
      if (more && seg.t0 == 0 && !seg.whole) split = {last_share - static_cast<int>(blockIdx.x) + 1, seg.begin, seg.count, seg.pair, seg.kv_head, seg.halved, {}};
      if (!__all_sync(0xffffffffu, mbar_wait(segment_empty(segment_at), segment_phase ^ 1u, abort_word, 104))) break;
      if (lane == 0) {
        segments[segment_at] = seg;
        mbar_arrive(segment_full(segment_at));
      }
      if (++segment_at == kSegments) { segment_at = 0; segment_phase ^= 1u; }
    }
    if (lane == 0) p.splits[blockIdx.x] = split;
  }
  } else if (kQuantized && warp >= 12) {
    setmaxnreg_dec<kDecoderRegs>();
    if constexpr (kQuantized) {
      // ------------------------------------------------------------ decoders: K by the first kDecoders warps, V by the others, 32 rows of
      // a tile each. A lane takes 16 bytes of codes, 32 elements of a row, of every kRowsAtOnce-th row. The next tile's codes are on
      // their way while this one's are decoded, and its pages while those are asked for. The code is the same for K and V, and in one
      // loop, as all warps' loops together have to stay in the instruction cache.
      constexpr int kLanes = kHd / 32, kRowsAtOnce = 32 / kLanes, kAtOnce = 32 / kRowsAtOnce;       // lanes to a row
      static_assert(kDecoders * 32 == kTileN, "32 rows to a decoder");
      const bool is_v = warp >= 12 + kDecoders;
      const int row0 = ((warp - 12) & (kDecoders - 1)) * 32, chunk = lane % kLanes, lane_row = lane / kLanes;
      const QuantizedRows &rows = is_v ? p.rows.v : p.rows.k;
      const int page_size = p.a.cache.page_size, tile_slots = kTileN / page_size, tile_rows = kTileN % page_size;
      // Where the lane's 16 bytes go in a row: 64-column block, and chunks of it. Lanes of the two blocks take their words in another
      // order, so that eight lanes' stores fall into different banks.
      const int turned = kHd == 128 ? (chunk >> 1) * 2 : 0;
      const uint32_t dst = smem_base + L::kRingOff + (kHd == 128 ? (chunk >> 1) * kBlockBytes : 0) + (row0 + lane_row) * 128;
      const uint32_t dst_chunk = (((chunk & 1) * 4 + turned) ^ (lane_row & 7)) << 4;                // of the first word; rows 8 apart are swizzled alike
      uint32_t position = 0;
      bool ok = true;
      Segment seg;
      while (ok && take_working(seg)) {
        const int tiles = seg.tiles();
        const int *pages = p.a.batch.page_table + seg.sequence * p.a.batch.table_stride;
        const uint8_t *codes = rows.codes + seg.kv_head * rows.codes_head + chunk * 16;
        const uint32_t *steps = rows.steps + seg.kv_head * rows.steps_head + (kHd == 128 ? chunk >> 1 : 0);
        // The lane's key of the tile that is looked up next, and its place.
        int key = seg.t0 * kTileN + row0 + lane, left = tiles;
        int slot_of = key / page_size, row_of = key - slot_of * page_size;
        int page = -1, in_page = 0;
        bool wanted = false;
        auto look_up = [&]() {
          wanted = left > 0 && key < seg.keys;
          page = wanted ? pages[slot_of] : -1;
          in_page = row_of;
          --left;
          key += kTileN;
          slot_of += tile_slots;
          row_of += tile_rows;
          if (row_of >= page_size) { row_of -= page_size; ++slot_of; }
        };
        uint4 word[kAtOnce];
        uint32_t pair[kAtOnce];
        auto load = [&]() {                              // of what was looked up
          const bool inside = page >= 0 && page < p.a.cache.pages;
          if (wanted && !inside) raise_status(p.a.refused, kRefusedPage);
          const int place = inside ? page : -1;
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int from = u * kRowsAtOnce + lane_row, row_page = __shfl_sync(0xffffffffu, place, from), row = __shfl_sync(0xffffffffu, in_page, from);
            word[u] = make_uint4(0u, 0u, 0u, 0u);        // rows without a key, or without a page, are zeros
            pair[u] = 0u;
            if (row_page >= 0) {
              word[u] = __ldcg(reinterpret_cast<const uint4 *>(codes + row_page * rows.codes_page + row * rows.codes_row));
              pair[u] = __ldcg(steps + row_page * rows.steps_page + row * rows.steps_row);
            }
          }
        };
        look_up();
        load();
        look_up();
#pragma unroll 1
        for (int j = 0; ok && j < tiles; ++j) {
          const uint32_t at = position + ring_place(seg, j, tiles, is_v);
          const int slot = at % L::kSlots;
          uint4 word_now[kAtOnce];
          uint32_t pair_now[kAtOnce];
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) { word_now[u] = word[u]; pair_now[u] = pair[u]; }
          load();
          look_up();
          if (!__all_sync(0xffffffffu, mbar_wait(kv_empty(slot), ((at / L::kSlots) & 1u) ^ 1u, abort_word, 102))) { ok = false; break; }
          const uint32_t tile = dst + slot * L::kTileBytes;
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const uint32_t step2 = __byte_perm(pair_now[u], 0u, 0x1010), low2 = __byte_perm(pair_now[u], 0u, 0x3232);
            const uint4 w = word_now[u];
            const uint32_t words[4] = {turned ? w.z : w.x, turned ? w.w : w.y, turned ? w.x : w.z, turned ? w.y : w.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t v[4];
              decode_word<kBf16>(words[c], step2, low2, v);
              st_shared_v4(tile + u * (kRowsAtOnce * 128) + (dst_chunk ^ (c << 4)), v);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(kv_full(slot));
        }
        position += 2 * tiles;
      }
    }
  } else {
    setmaxnreg_inc<kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax / rescale / epilogue
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row_in_tile = quarter * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_sel + kColS0 + t * 128;
    const uint32_t o_addr = tmem_base + lane_sel + kColO0 + t * 128;
    uint32_t tiles_done = 0, items_done = 0, meets = 0;
    bool ok = true;
    const uint32_t out_stage = smem_base + L::kOutOff + (warp - 4) * kOutStageBytes;
    while (ok) {
      int my_tiles, row_limit, masked_from, key_base, key_step;     // keys from masked_from on are hidden from some row of the tile
      {
        Segment seg;
        if (!take(seg)) break;
        my_tiles = seg.of(t);
        key_base = (seg.t0 + (seg.halved ? t : 0)) * kTileN;
        key_step = (seg.halved ? 2 : 1) * kTileN;
        row_limit = seg.keys - 1;
        masked_from = seg.keys;
        if (p.a.causal) {                                   // token i sees keys up to keys - count + i
          const int first = seg.keys - seg.count + (2 * seg.pair + (seg.halved ? 0 : t)) * p.tile_tokens;
          row_limit = min(row_limit, first + token_of(p, row_in_tile));
          masked_from = min(masked_from, first + 1);
        }
      }
      constexpr float kRescaleThreshold = 8.0f;
      float m_ref = -INFINITY, m_true = -INFINITY, l_run = 0.f;

      for (int j = 0; ok && j < my_tiles; ++j, ++tiles_done) {
        if (!mbar_wait(s_full(t), tiles_done & 1u, abort_word, 110 + t)) { ok = false; break; }
        tc_fence_after();
        const int key0 = key_base + j * key_step;
        // With eight more warps a thread has no room for its row's 128 scores: the last 64 are read for the maximum, and again once the
        // first 64 have given way to P.
        uint32_t r[kQuantized ? 64 : 128];
        const bool masked = key0 + kTileN > masked_from;
        const int visible_in_tile = row_limit - key0;
        auto read_half = [&](int half) {
#pragma unroll
          for (int c = 0; c < 2; ++c) tmem_ld_32x32(s_addr + (2 * half + c) * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32 * c]));
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (64 * half + i > visible_in_tile) r[i] = 0xff800000u;
          }
        };
        float raw_max;
        if constexpr (kQuantized) {
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int half = 1; half >= 0; --half) {
            read_half(half);
#pragma unroll
            for (int i = 0; i < 64; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
          }
          raw_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32 * c]));
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (i > visible_in_tile) r[i] = 0xff800000u;   // -inf
          }
          float mx[4];
#pragma unroll
          for (int a = 0; a < 4; ++a) mx[a] = fmax3(__uint_as_float(r[32 * a]), __uint_as_float(r[32 * a + 1]), __uint_as_float(r[32 * a + 2]));
#pragma unroll
          for (int i = 3; i + 1 < 32; i += 2) {
#pragma unroll
            for (int a = 0; a < 4; ++a) mx[a] = fmax3(mx[a], __uint_as_float(r[32 * a + i]), __uint_as_float(r[32 * a + i + 1]));
          }
#pragma unroll
          for (int a = 0; a < 4; ++a) mx[a] = fmaxf(mx[a], __uint_as_float(r[32 * a + 31]));
          raw_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        }
        m_true = fmaxf(m_true, raw_max * p.scale_log2);
        float alpha = 1.0f;
        const bool moves = m_true - m_ref > kRescaleThreshold, any_moves = __any_sync(0xffffffffu, moves);
        if (moves) {
          alpha = exp2f(m_ref - m_true);
          m_ref = m_true;
        }
        const float m_exp = (m_ref == -INFINITY) ? 0.f : m_ref;
        const unsigned long long scale2 = pack_f32x2(p.scale_log2, p.scale_log2), neg_m2 = pack_f32x2(-m_exp, -m_exp);
        unsigned long long sum2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t packed[16];
          const int base = kQuantized ? 32 * (c & 1) : 32 * c;
          if (kQuantized && c == 2) read_half(1);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const unsigned long long x2 = fma_f32x2(pack_f32x2(__uint_as_float(r[base + i]), __uint_as_float(r[base + i + 1])), scale2, neg_m2);
            float x0, x1;
            unpack_f32x2(x2, x0, x1);
            const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
            sum2[(i >> 1) & 3] = add_f32x2(sum2[(i >> 1) & 3], pack_f32x2(e0, e1));
            // P is rounded to the storage type for the product with V (one type for both operands); the sum is not. Error against
            // 64 bits in bf16: 2.3e-3 where an f32 P has 1.7e-3 (2-norm, the result's own rounding in it).
            packed[i >> 1] = pack2<kBf16>(e0, e1);
          }
          tmem_st_32x16(s_addr + c * 16, packed);    // P lies over the first 64 columns of S
          if (c == kFirstChunks - 1 && j > 0 && any_moves) {
#pragma unroll 1
            for (int oc = 0; oc < kHd / 32; ++oc) {
              uint32_t o[32];
              tmem_ld_32x32(o_addr + oc * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x32(o_addr + oc * 32, o);
            }
          }
          if (c == kFirstChunks - 1 || c == 3) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_part(t, c == 3 ? 1 : 0));
          }
        }
        float s0, s1, s2, s3, s4, s5, s6, s7;
        unpack_f32x2(sum2[0], s0, s1); unpack_f32x2(sum2[1], s2, s3); unpack_f32x2(sum2[2], s4, s5); unpack_f32x2(sum2[3], s6, s7);
        l_run = l_run * alpha + (((s0 + s1) + (s2 + s3)) + ((s4 + s5) + (s6 + s7)));
      }

      if (ok && my_tiles > 0) ok = mbar_wait(o_done(t), items_done++ & 1u, abort_word, 114 + t);
      const Segment seg = segments[segment_at];
      const int first_token = (2 * seg.pair + (seg.halved ? 0 : t)) * p.tile_tokens;       // of the tile, within the sequence
      const bool joined = seg.halved && seg.whole;
      if (ok && seg.whole) {
        // Of a halved item the two tiles' warps of the same TMEM lanes join their states and write half of the columns each.
        const int columns = joined ? kHd / 2 : kHd, c0 = joined ? t * columns : 0;
        const uint32_t other_addr = o_addr + (t ? -128 : 128);
        auto arrive_pair = [&]() {
          __syncwarp();
          if (lane == 0) mbar_arrive(paired(quarter));
        };
        auto wait_pair = [&]() { return mbar_wait(paired(quarter), meets++ & 1u, abort_word, 116); };
        float scale0 = 1.f, scale1 = 0.f;              // of this warp's state and the other's
        bool other_half = false;
        if (joined) {
          float2 *const states = reinterpret_cast<float2 *>(smem + L::kOutOff);
          states[(warp - 4) * (kOutStageBytes / 8) + lane] = make_float2(m_ref, l_run);
          tc_fence_before();
          arrive_pair();
          if (!(ok = wait_pair())) break;
          const float2 other = states[((warp - 4) ^ 4) * (kOutStageBytes / 8) + lane];
          arrive_pair();
          other_half = seg.of(1 - t) > 0;
          const float top = fmaxf(l_run > 0.f ? m_ref : -INFINITY, other.y > 0.f ? other.x : -INFINITY);
          scale0 = l_run > 0.f ? ex2_approx(m_ref - top) : 0.f;
          scale1 = other.y > 0.f ? ex2_approx(other.x - top) : 0.f;
          l_run = l_run * scale0 + other.y * scale1;
          m_ref = top;
          if (!(ok = wait_pair())) break;              // the stages' states have been read
        }
        tc_fence_after();
        const bool empty = l_run == 0.f;
        const float coefficient = empty ? 0.f : 1.0f / l_run;
        scale0 *= coefficient;
        scale1 *= coefficient;
        const uint32_t filled = p.a.zero_fully_masked ? 0u : (kBf16 ? 0x7fc07fc0u : 0x7e007e00u);
        const int at = token_of(p, row_in_tile), token = first_token + at, head = seg.kv_head * p.group + row_in_tile - at * p.group;
        const bool used = at < p.tile_tokens && token < seg.count;
        // Where the lane's row of the output begins; -1: not a row.
        const long long row_at = used ? static_cast<int64_t>(seg.begin + token) * p.a.out_token + head * p.a.out_head : -1;
        // Through shared memory, 32 rows x 64 columns at a time (32 columns of a half at head_dim 64), so that a store instruction
        // covers rows' 128 (64) bytes. The loops stay rolled: code that runs once per item comes from L2, eight instructions a line.
        const int by_row = columns < 64 ? 2 : 3;       // 2^n lanes store a row
#pragma unroll 1
        for (int pass = c0; pass < c0 + columns; pass += 64) {
          __syncwarp();                              // the stage's previous contents have been read
#pragma unroll 1
          for (int c = 0; c < min(columns, 64); c += 16) {
            uint32_t r[16];
            if (my_tiles > 0) {
              tmem_ld_32x16(o_addr + pass + c, r);
              tmem_wait_ld();
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * scale0);
            if (other_half) {
              uint32_t o[16];
              tmem_ld_32x16(other_addr + pass + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(fmaf(__uint_as_float(o[i]), scale1, __uint_as_float(r[i])));
            }
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                w[k] = pack2<kBf16>(__uint_as_float(r[i + 2 * k]), __uint_as_float(r[i + 2 * k + 1]));
                if (empty) w[k] = filled;
              }
              st_shared_v4(out_stage + lane * 128 + ((((c + i) >> 3) ^ (lane & 7)) << 4), w);
            }
          }
          if (joined) {                              // one pass: both accumulators have been read
            tc_fence_before();
            arrive_pair();
          } else {
            __syncwarp();
          }
          const int chunk = lane & ((1 << by_row) - 1);
#pragma unroll 1
          for (int i = lane >> by_row; i < 32; i += 128 >> by_row) {         // four loads on their way together
            uint32_t w[4][4];
            long long to[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int r_out = i + u * (32 >> by_row);
              to[u] = __shfl_sync(0xffffffffu, row_at, r_out);
              ld_shared_v4(out_stage + r_out * 128 + (((chunk ^ r_out) & 7) << 4), w[u]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (to[u] >= 0)
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.a.out) + to[u] + pass + chunk * 8) = make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
          }
        }
        if (p.a.lse && used && !(joined && t))
          p.a.lse[static_cast<int64_t>(seg.begin + token) * p.a.q_heads + head] =
              empty ? -INFINITY : m_ref * 0.69314718055994530942f + logf(l_run);
        if (joined) ok = wait_pair();
      } else if (ok && first_token < seg.count) {
        // A part of an item: the state as it is, four columns of 32 rows to a store.
        tc_fence_after();
        float *record = p.records + ((static_cast<int64_t>(blockIdx.x) * 2 + (seg.t0 == 0 ? 1 : 0)) * 2 + t) * L::kRecordFloats;
#pragma unroll 1
        for (int c = 0; c < kHd; c += 16) {
          uint32_t r[16];
          if (my_tiles > 0) {
            tmem_ld_32x16(o_addr + c, r);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = 0u;
          }
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<uint4 *>(record + (((c + i) >> 2) * kTileM + row_in_tile) * 4) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
        *reinterpret_cast<float2 *>(record + kTileM * kHd + 2 * row_in_tile) = make_float2(m_ref, l_run);
      }
      // The accumulator has been read before this warp lets the next segment's first product over it, by its next arrival.
      tc_fence_before();
      give_back();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_word != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(10000);
    if (threadIdx.x == 0) raise_status(p.a.status, *abort_word);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Folds the records of the item that starts in share blockIdx.x: blockIdx.y is eight columns, a thread a row of either Q tile, or,
// of a halved item, a row and every second group of four records. Four records' elements are on their way together: a long cache
// of few rows leaves many records (an item of 9000 keys about 40), of which two at a time, by a thread per row, took 20 us. Eight
// columns to a thread leave room for three blocks on an SM, sixteen for two: 100 tokens over 20000 keys of one KV head 30.6 / 33.0 us.
constexpr int kColumns = 8;
template <bool kBf16, int kHd>
__global__ void __launch_bounds__(2 * kTileM, 3) attention_paged_chunk_fold_kernel(const __grid_constant__ ChunkParams p) {
  using L = Shape<kHd>;
  constexpr int kAtOnce = 4;
  __shared__ float joined[2 + kColumns][kTileM];               // of the second thread of a halved item's row
  pdl_wait();
  pdl_launch_dependents();
  const ChunkSplit split = p.splits[blockIdx.x];
  if (split.records == 0) return;
  const int row = threadIdx.x % kTileM, second = threadIdx.x / kTileM;
  const int t = split.halved ? 0 : second, groups = split.halved ? 2 : 1, group = split.halved ? second : 0;
  const int at = token_of(p, row), token = (2 * split.pair + t) * p.tile_tokens + at;
  const bool used = at < p.tile_tokens && token < split.count;
  // A halved item's halves are records of their own.
  const int records = used ? split.records * (split.halved ? 2 : 1) : 0;
  auto record = [&](int i) {
    const int share = split.halved ? i >> 1 : i;
    return p.records + ((static_cast<int64_t>(blockIdx.x + share) * 2 + (share == 0 ? 1 : 0)) * 2 + (split.halved ? i & 1 : t)) * L::kRecordFloats;
  };
  float top = -INFINITY, l = 0.f, acc[kColumns];
#pragma unroll
  for (int e = 0; e < kColumns; ++e) acc[e] = 0.f;
  auto add = [&](const float (&m)[kAtOnce], const float (&sum)[kAtOnce], const float (&v)[kAtOnce][kColumns]) {
    float next = top;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) next = fmaxf(next, sum[u] > 0.f ? m[u] : -INFINITY);
    const float m_exp = next == -INFINITY ? 0.f : next, alpha = ex2_approx(top - m_exp);
    top = next;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < kColumns; ++e) acc[e] *= alpha;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float w = sum[u] == 0.f ? 0.f : ex2_approx(m[u] - m_exp);
      l = fmaf(sum[u], w, l);
      if (sum[u] == 0.f) continue;                   // a part that saw no key
#pragma unroll
      for (int e = 0; e < kColumns; ++e) acc[e] = fmaf(v[u][e], w, acc[e]);
    }
  };
#pragma unroll 1
  for (int i = group * kAtOnce; i < records; i += groups * kAtOnce) {
    float m[kAtOnce], sum[kAtOnce], v[kAtOnce][kColumns];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      m[u] = sum[u] = 0.f;
      if (i + u < records) {
        const float *r = record(i + u);
        const float2 ml = *reinterpret_cast<const float2 *>(r + kTileM * kHd + 2 * row);
        m[u] = ml.x;
        sum[u] = ml.y;
#pragma unroll
        for (int e = 0; e < kColumns / 4; ++e) *reinterpret_cast<float4 *>(&v[u][4 * e]) = *reinterpret_cast<const float4 *>(r + ((blockIdx.y * (kColumns / 4) + e) * kTileM + row) * 4);
      }
    }
    add(m, sum, v);
  }
  if (split.halved) {
    if (group > 0) {
      joined[0][row] = top;
      joined[1][row] = l;
#pragma unroll
      for (int e = 0; e < kColumns; ++e) joined[2 + e][row] = acc[e];
    }
    __syncthreads();
    if (group > 0) return;
    if (used) {
      float m[kAtOnce] = {joined[0][row]}, sum[kAtOnce] = {joined[1][row]}, v[kAtOnce][kColumns];
#pragma unroll
      for (int e = 0; e < kColumns; ++e) v[0][e] = joined[2 + e][row];
      add(m, sum, v);
    }
  }
  if (!used) return;
  const bool empty = l == 0.f;
  const float coefficient = empty ? 0.f : 1.0f / l;
  const uint32_t filled = p.a.zero_fully_masked ? 0u : (kBf16 ? 0x7fc07fc0u : 0x7e007e00u);
  const int head = split.kv_head * p.group + row - at * p.group;
  uint16_t *dst = static_cast<uint16_t *>(p.a.out) + static_cast<int64_t>(split.begin + token) * p.a.out_token + head * p.a.out_head + blockIdx.y * kColumns;
#pragma unroll
  for (int e = 0; e < kColumns / 8; ++e) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = pack2<kBf16>(acc[8 * e + 2 * k] * coefficient, acc[8 * e + 2 * k + 1] * coefficient);
      if (empty) w[k] = filled;
    }
    *reinterpret_cast<uint4 *>(dst + 8 * e) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (p.a.lse && blockIdx.y == 0)
    p.a.lse[static_cast<int64_t>(split.begin + token) * p.a.q_heads + head] = empty ? -INFINITY : top * 0.69314718055994530942f + logf(l);
}

// What both launches fill in alike.
size_t chunk_record_bytes(int sm_count) { return static_cast<size_t>(sm_count) * 4 * Shape<128>::kRecordFloats * sizeof(float); }

void fill_chunk_params(ChunkParams *p, const AttentionPagedArgs &a, int sm_count) {
  p->a = a;
  p->group = a.q_heads / a.cache.kv_heads;
  p->tile_tokens = kTileM / p->group;
  p->by_group = (1ull << 32) / p->group + 1;
  p->by_grid = ~0ull / static_cast<unsigned>(sm_count) + 1;
  p->scale_log2 = a.scale * 1.4426950408889634f;
  p->records = static_cast<float *>(a.workspace);
  p->splits = reinterpret_cast<ChunkSplit *>(static_cast<uint8_t *>(a.workspace) + chunk_record_bytes(sm_count));
}
// The tensor map of Q: a tile's tokens and the heads of its group, 64 columns. Strides of extents of one are free, but the map wants
// them to span what lies inside.
bool tokens_outside_heads(const AttentionPagedArgs &a) {
  return (a.q_heads == 1 || a.q_head >= a.cache.head_dim) &&
         (a.batch.tokens == 1 || a.q_token >= (a.q_heads == 1 ? a.cache.head_dim : a.q_heads * a.q_head));
}
wb200_status encode_queries(CUtensorMap *map, const AttentionPagedArgs &a, const ChunkParams &p) {
  const uint64_t d = static_cast<uint64_t>(a.cache.head_dim);
  const uint64_t q_head = a.q_heads == 1 ? d * 2 : static_cast<uint64_t>(a.q_head) * 2;
  const uint64_t q_token = a.batch.tokens == 1 ? q_head * a.q_heads : static_cast<uint64_t>(a.q_token) * 2;
  return encode_tmap_strided(map, a.q, a.cache.format, 3, {d, static_cast<uint64_t>(a.q_heads), static_cast<uint64_t>(a.batch.tokens), 1},
                             {q_head, q_token, 0}, {64, static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.tile_tokens), 1});
}

}  // namespace
}  // namespace wb200
