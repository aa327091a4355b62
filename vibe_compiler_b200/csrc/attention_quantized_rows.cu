// Attention of few new tokens over a paged KV cache held in four bits: decoding and drafted tokens (head_dim 64 and 128).
//
// How the work is dealt to the CTAs and folded is the 16-bit kernel's (attention_paged_walk.cuh). What differs is the arithmetic of a
// tile of 32 keys. At 4.5 bits an element, an SM's share of HBM brings 16 keys of K and V (2304 bytes at head_dim 128) every 99
// clocks, 396 issue slots of a scheduler for one warp's tile, so nothing may be widened element by element:
//   codes    are the matrix operands as they are. Bits 0 to 7 of two f16, w & 0x00ff00ff, are (even code + 16 odd code) 2^-24 of two
//            pairs of elements, w & 0x00f000f0 the odd codes' part (subnormal numbers, which the tensor cores multiply exactly): four
//            instructions for the eight elements of a word. The powers of two go into Q, and into the result.
//   K        S^T = C Q^T, keys on the 16-wide side, with the odd codes' share of the even elements' sums taken off by a product with
//            -Q, a sum for each group of 64 elements: s = sum_g step_g (c.q)_g + low_g (sum q)_g. The products are exact: Q is scaled
//            to f16 by a power of two of its own a row (elements 2^24 times smaller than the row's largest lose digits, off by 2^-35 of it).
//   V        O^T = C P^T, sums with the odd codes in them and sums of those alone as rows of one product, subtracted at the end.
//            step_g is folded into the probabilities, p'_g = p step_g 2^e_g, rounded to f16 (11 bits, whatever the type), and
//            sum_j p_j (low + 8 step)_g,j runs beside it in f32: a product with a constant takes 8 off every code, so that both sums
//            are as small as the values are. (A tensor core's f32 sums are cut off, not rounded. Of codes as they are, whose sums only
//            grow, the values' mean is what is left of two numbers 300 times as large: 17 thousand keys in f16 came out 1.3e-2 off
//            in the 2-norm, of 2e-4 with codes less 8.) e_g follows the largest step of the group so far, so p' stays below f16's
//            largest; p' up to 2^-25, of steps 2^-30 of that one with p = 1, vanish from this sum (one e for both groups took all digits
//            of the smaller one from 2^24 on).
//            P, as S^T leaves it, becomes the other operand by movmatrix; rows of K or V are never transposed: two keys' words
//            interleaved by halves (prmt) are the pairs that the instruction wants.
//   four rows  of a sequence or fewer, head_dim 128: Q stands in the columns twice, and P^T in the second four carries the second
//            group's steps, so a lane weighs its probabilities for one group.
//   maximum  The exponent's reference moves only when a score is beyond 2^8 times it: one vote a tile instead of shuffles.
// A CTA is four warps; each streams every fourth 32-key tile of the share through a ring of its own (cp.async, rows XOR-swizzled).
// Bound: 64 sequences of 2000 to 32000 keys, 32/8 heads, f16: 242 us, 4.4 TB/s (the floor is 163). The warps' instructions for 16 keys (306,
// of which 12 + 16 are products) would fit the 396 issue slots that HBM takes, but are issued at 0.55 a clock: with three warps to a
// scheduler, as many as the registers allow, results and busy pipes are waited for.
// Taken back: e4m3 products for K (three instructions a word; 359 us against 221 then);
// the scores of a tile among the products with V of the one before (168 registers do not hold both: 234); tiles of 16 keys with four
// CTAs to an SM (271 against 228).
#include "attention_paged_walk.cuh"
#include "quantized_rows.cuh"

namespace wb200 {
namespace {

constexpr int kWarps = 4;
constexpr int kBlocks = 2;                      // of 16 keys, a side of the matrix instruction, in a warp's tile
constexpr int kTileKeys = 16 * kBlocks;
constexpr int kStepKeys = kWarps * kTileKeys;
// What a unit costs by itself, in steps of 128 keys: 100 sequences of 100 to 4000 keys, 8 KV heads, with 1 / 2 / 3 / 5 / 8 76 / 69 / 67 /
// 70 / 73 us, 100 of 20 to 1000 34 / 30 / 29 / 30 / 31.
constexpr int kUnitSteps = 3;
constexpr int kLeastSteps = 2;
constexpr float kMovesBeyond = 8.f;             // log2
constexpr int kStepExponent = 5;                // of step 2^e when e is chosen; steps of twice that do not move it, so p' < 2^8 2^7
constexpr int kLeastExponent = -120, kMostExponent = 126;        // 2^e and 2^-e are normal numbers of f32
constexpr uint32_t kBoth = 0x00ff00ffu, kOdd = 0x00f000f0u;
constexpr uint32_t kMinusBoth = 0x80888088u, kMinusOdd = 0x80808080u;     // -(8 + 16 * 8) 2^-24, -16 * 8 * 2^-24, twice

template <int kD>
struct QuantShape {
  static constexpr int kGroups = kD / kQuantGroup;
  static constexpr int kRowBytes = kD / 2;
  static constexpr int kCodeBytes = kTileKeys * kRowBytes;
  static constexpr int kStepBytes = kTileKeys * kGroups * 4;
  static constexpr int kStageBytes = 2 * (kCodeBytes + kStepBytes);     // K codes, V codes, K steps, V steps
  static constexpr int kStages = kD == 128 ? 3 : 6;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kRecord = kRowRecord<kD>;
  static constexpr int kRecordsOff = kWarps * kRingBytes;
  static constexpr int kQueryOff = kRecordsOff + kWarps * 8 * kRecord * 4;
  static constexpr int smem_bytes(int rows) { return kQueryOff + (rows > 8 ? 2 : 1) * kGroups * 8 * 128; }   // operands of Q
  static_assert(kStageBytes % 128 == 0, "tiles begin on 128 bytes");
};
// CTAs to an SM: as many as the registers of a thread allow.
constexpr int ctas_per_sm(int rows) { return rows <= 8 ? 3 : 2; }
static_assert(3 * (QuantShape<128>::smem_bytes(8) + 256 + 1024) <= 228 * 1024, "three CTAs to an SM");

// Strides small enough for one 32-bit product: codes in 16 bytes, steps in a row's steps.
struct ShortStrides {
  uint32_t page, row;
};
struct QuantRowsParams : RowsFold {
  QuantizedRowsArgs rows;
  ShortStrides k_codes, v_codes, k_steps, v_steps;
  int step_slots, step_rows;        // a step of keys in pages and rows of the next one
  float scale_log2;
  unsigned long long by_grid;       // as RowsWalk takes it
};

// Byte offset of 16-byte chunk c of row r in a tile of codes: lines of 128 bytes, the chunks of a line swizzled so that the words of
// rows 2t, t = 0 .. 3, which a warp reads at once, lie in different banks.
template <int kRowBytes>
__device__ __forceinline__ uint32_t code_offset(int r, int c) {
  if constexpr (kRowBytes == 64) return static_cast<uint32_t>((r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4));
  else return static_cast<uint32_t>((r >> 2) * 128 + (((((r & 3) << 1) | c) ^ (((r >> 2) & 1) << 1)) << 4));
}
template <int kBytes>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes), "r"(src_bytes) : "memory");
}
// The steps of a row's groups.
template <int kGroups>
__device__ __forceinline__ void load_steps(const uint8_t *src, uint32_t (&v)[kGroups]) {
  if constexpr (kGroups == 2) {
    const uint2 w = *reinterpret_cast<const uint2 *>(src);
    v[0] = w.x;
    v[1] = w.y;
  } else {
    v[0] = *reinterpret_cast<const uint32_t *>(src);
  }
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes 1 and 3 as bytes 0 and 2.
__device__ __forceinline__ uint32_t upper_bytes(uint32_t v) { return __byte_perm(v, 0u, 0x4341); }
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
// 2^(exponent - that of x's leading bit) for x > 0 and finite, within the normal numbers.
__device__ __forceinline__ float power_against(float x, int exponent) {
  const int field = 254 + exponent - static_cast<int>(__float_as_uint(x) >> 23);
  return __uint_as_float(static_cast<uint32_t>(min(max(field, 1), 254)) << 23);
}

// Tiles of kRows rows: 4, 8 or 16.
template <bool kBf16, int kD, int kRows, bool kAligned, bool kClustered>
__global__ void __launch_bounds__(kWarps * 32, ctas_per_sm(kRows)) attention_quantized_rows_kernel(const __grid_constant__ QuantRowsParams p) {
  using S = QuantShape<kD>;
  constexpr int kFormat = kBf16 ? WB200_BF16 : WB200_F16;
  constexpr uint32_t kInfinity = kBf16 ? 0x7f80u : 0x7c00u;
  constexpr int kGroups = S::kGroups, kTiles = kRows == 16 ? 2 : 1;          // eight columns of the products each
  constexpr bool kTwice = kRows == 4;                  // columns 4 to 7 are the same rows, for the second group of V
  constexpr int kWeighed = kTwice ? 1 : kGroups;       // groups that a lane weighs its probabilities for
  static_assert(!kTwice || kGroups == 2, "two groups share the columns");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long warp_totals[kWarps], start_prefix;
  __shared__ int start_sequence;
  const AttentionPagedArgs &a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();

  RowsWalk<kRows, kStepKeys, kUnitSteps, kLeastSteps, kWarps, kClustered> walk(a, p.group, p.by_grid);
  walk.find_share(warp_totals, &start_sequence, &start_prefix);
  uint64_t policy = 0;
  RowsSplit split = {};

  uint8_t *const ring = smem + warp * S::kRingBytes;
  const uint32_t ring_addr = smem_u32(ring);
  float *records = reinterpret_cast<float *>(smem + S::kRecordsOff);   // [warp][8][kRecord]
  uint32_t *operands = reinterpret_cast<uint32_t *>(smem + S::kQueryOff);

  // Of the walk's part this warp takes every fourth tile.
  struct Part : RowsPart {
    int first_key, key_end, tiles;
  } part = {};
  const int *pages = nullptr;
  // Where this lane's chunk of a tile's first row lies in a page, of K and of V, and the steps of its key (a lane has one key of a
  // tile): a row per kChunks lanes, or the row of the lane's own key where tiles span pages.
  constexpr int kChunks = S::kRowBytes / 16, kRowsAtOnce = 32 / kChunks;
  const int chunk_row = lane / kChunks, chunk = lane % kChunks;
  const uint8_t *k_base = nullptr, *v_base = nullptr;
  const uint8_t *k_step_base = nullptr, *v_step_base = nullptr;
  const uint32_t code_dst = code_offset<S::kRowBytes>(chunk_row, chunk);
  const uint32_t step_dst = 2 * S::kCodeBytes + lane * (4 * kGroups);
  // The next tile to be issued: its first key, and the place of that key (kAligned: pages are whole tiles) or of the lane's key of it.
  int issue_key = 0, issue_slot = 0, issue_row = 0, page = -1, page_row = 0;
  auto next_part = [&]() {
    if (!walk.next()) return false;
    static_cast<RowsPart &>(part) = walk.part;
    part.key_end = min(part.keys, part.step1 * kStepKeys);
    part.first_key = part.step0 * kStepKeys + warp * kTileKeys;
    part.tiles = part.key_end > part.first_key ? (part.key_end - part.first_key + kStepKeys - 1) / kStepKeys : 0;
    policy = l2_policy(static_cast<long long>(part.sequence.count) * p.group > kRows);
    pages = a.batch.page_table + part.s * a.batch.table_stride;
    const int row = kAligned ? chunk_row : 0, step_row = kAligned ? lane : 0;
    k_base = p.rows.k.codes + part.kv_head * p.rows.k.codes_head + row * p.rows.k.codes_row + chunk * 16;
    v_base = p.rows.v.codes + part.kv_head * p.rows.v.codes_head + row * p.rows.v.codes_row + chunk * 16;
    k_step_base = reinterpret_cast<const uint8_t *>(p.rows.k.steps + part.kv_head * p.rows.k.steps_head + step_row * p.rows.k.steps_row);
    v_step_base = reinterpret_cast<const uint8_t *>(p.rows.v.steps + part.kv_head * p.rows.v.steps_head + step_row * p.rows.v.steps_row);
    issue_key = part.first_key;
    const int key = issue_key + (kAligned ? 0 : lane);
    issue_slot = key / a.cache.page_size;
    issue_row = key - issue_slot * a.cache.page_size;
    return true;
  };
  // The page of the next tile, looked up one tile ahead of its copies.
  auto look_up = [&]() {
    page_row = issue_row;
    page = issue_key + (kAligned ? 0 : lane) < part.key_end ? pages[issue_slot] : -1;
    issue_slot += p.step_slots;
    issue_row += p.step_rows;
    if (issue_row >= a.cache.page_size) { issue_row -= a.cache.page_size; ++issue_slot; }
  };
  auto issue_tile = [&](uint32_t stage) {
    if (issue_key < part.key_end) {
      const uint32_t code_to = stage + code_dst;
      const int own_key = issue_key + lane;
      const bool inside = page >= 0 && page < a.cache.pages;
      const uint32_t place = inside ? page : 0;
      const uint64_t k_at = static_cast<uint64_t>(place) * p.k_codes.page + static_cast<uint64_t>(static_cast<uint32_t>(page_row)) * p.k_codes.row;
      const uint64_t v_at = static_cast<uint64_t>(place) * p.v_codes.page + static_cast<uint64_t>(static_cast<uint32_t>(page_row)) * p.v_codes.row;
      const uint64_t k_step_at = static_cast<uint64_t>(place) * p.k_steps.page + static_cast<uint64_t>(static_cast<uint32_t>(page_row)) * p.k_steps.row;
      const uint64_t v_step_at = static_cast<uint64_t>(place) * p.v_steps.page + static_cast<uint64_t>(static_cast<uint32_t>(page_row)) * p.v_steps.row;
      if (kAligned && inside && issue_key + kTileKeys <= part.key_end) {
        const uint8_t *const k_from = k_base + k_at * 16, *const v_from = v_base + v_at * 16;
#pragma unroll
        for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
          cp_async16_hint(policy, code_to + i * (kRowsAtOnce * S::kRowBytes), k_from + i * kRowsAtOnce * p.rows.k.codes_row, 16u);
          cp_async16_hint(policy, code_to + S::kCodeBytes + i * (kRowsAtOnce * S::kRowBytes), v_from + i * kRowsAtOnce * p.rows.v.codes_row, 16u);
        }
        cp_async_small<4 * kGroups>(stage + step_dst, k_step_base + k_step_at * (4 * kGroups), 4u * kGroups);
        cp_async_small<4 * kGroups>(stage + step_dst + S::kStepBytes, v_step_base + v_step_at * (4 * kGroups), 4u * kGroups);
      } else {
        if (!inside && own_key < part.key_end) raise_status(a.refused, kRefusedPage);
        const bool mine = inside && own_key < part.key_end;      // other rows are zeros
        const unsigned int seen = __ballot_sync(0xffffffffu, mine);
#pragma unroll
        for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
          const int r = i * kRowsAtOnce + chunk_row;
          const bool reads = (seen >> r) & 1u;
          int64_t k_from, v_from;
          if constexpr (kAligned) {
            k_from = k_at * 16 + i * kRowsAtOnce * p.rows.k.codes_row;
            v_from = v_at * 16 + i * kRowsAtOnce * p.rows.v.codes_row;
          } else {
            k_from = __shfl_sync(0xffffffffu, k_at, r) * 16;
            v_from = __shfl_sync(0xffffffffu, v_at, r) * 16;
          }
          cp_async16_hint(policy, code_to + i * (kRowsAtOnce * S::kRowBytes), reads ? k_base + k_from : p.rows.k.codes, reads ? 16u : 0u);
          cp_async16_hint(policy, code_to + S::kCodeBytes + i * (kRowsAtOnce * S::kRowBytes), reads ? v_base + v_from : p.rows.v.codes, reads ? 16u : 0u);
        }
        const uint8_t *const some = reinterpret_cast<const uint8_t *>(p.rows.k.steps);
        cp_async_small<4 * kGroups>(stage + step_dst, mine ? k_step_base + k_step_at * (4 * kGroups) : some, mine ? 4u * kGroups : 0u);
        cp_async_small<4 * kGroups>(stage + step_dst + S::kStepBytes, mine ? v_step_base + v_step_at * (4 * kGroups) : some, mine ? 4u * kGroups : 0u);
      }
    }
    cp_async_commit();
    issue_key += kStepKeys;
  };
  auto fill_ring = [&]() {
#pragma unroll 1
    for (int i = 0; i < S::kStages; ++i) {
      look_up();
      issue_tile(ring_addr + i * S::kStageBytes);
    }
    look_up();
  };

  bool more = next_part();
  if (more) fill_ring();
  while (more) {
    // A lane's columns are 2t and 2t + 1 of each eight, its elements 8g .. 8g + 7 of each group: acc[.][.][i] holds the sums over both
    // codes of elements 2i and 2i + 1 (two columns), and over the odd ones (two columns). A column's row: column_row().
    auto middle = [](uint32_t pair) { return fmaf(8.f, quant_step(pair, kFormat), quant_low(pair, kFormat)); };
    auto column_row = [](int column) { return kTwice ? column & 3 : column; };
    const int own_group = kTwice ? t >> 1 : 0;         // the first that this lane weighs for
    float minus_reference[kTiles][2], bound[kTiles][2];          // of the exponent; relative scores beyond the bound move it
    float l_run[kTiles][2], low_sum[kTiles][kWeighed][2], acc[kTiles][kGroups][4][4];
    float row_scale[kTiles][2], q_sum[kTiles][kGroups][2];       // of a row's scores; of the lows, in the units of the sums over codes
    uint32_t q_frag[kTiles][kGroups][2][2][2], q_fix[kTiles][kGroups][2][2];
    int last_key[kTiles][2];                           // that the row sees
    bool beyond = false;
    int exponent[kWeighed];                            // e
    uint32_t step_limit[kWeighed];                     // bits of a step; greater ones move e
#pragma unroll
    for (int gr = 0; gr < kWeighed; ++gr) {
      exponent[gr] = 0;
      step_limit[gr] = 0;
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      // The row's elements 64 gr + 16 t + .. of this lane's column g.
      const int packed = part.row0 + 8 * n + column_row(g), token = packed / p.group;
      uint4 bits[kGroups][2];
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        bits[gr][0] = bits[gr][1] = make_uint4(0u, 0u, 0u, 0u);
        if (8 * n + column_row(g) < part.rows) {
          const uint4 *row = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + static_cast<int64_t>(part.sequence.begin + token) * a.q_token +
                                                             (part.kv_head * p.group + packed - token * p.group) * a.q_head + gr * kQuantGroup + 16 * t);
          bits[gr][0] = row[0];
          bits[gr][1] = row[1];
        }
      }
      auto element = [&](int gr, int e) {
        const uint4 w = bits[gr][e >> 3];
        const uint32_t pair = (e & 4) ? ((e & 2) ? w.w : w.z) : ((e & 2) ? w.y : w.x);
        return widen_bits(e & 1 ? pair >> 16 : pair & 0xffffu, kFormat);
      };
      float largest = 0.f, sums[kGroups];
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
        for (int e = 0; e < 16; ++e) largest = fmaxf(largest, fabsf(element(gr, e)));
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, off));
      // Scaled by a power of two that brings the row's largest to 2^14, and those that meet odd codes, 16 times as large, to a sixteenth.
      // The operands are the same for all warps, who make a part of them each.
      const float power = largest > 0.f && largest < INFINITY ? power_against(largest, 14) : 1.f;
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        sums[gr] = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[gr] = fmaf(element(gr, e), power, sums[gr]);
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) sums[gr] += __shfl_xor_sync(0xffffffffu, sums[gr], off);
      }
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (((n * kGroups + gr) * 2 + w) % kWarps != warp) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int e = 8 * w + 2 * h;
            const __half2 even = __floats2half2_rn(element(gr, e) * power, element(gr, e + 4) * power);
            const __half2 odd = __floats2half2_rn(element(gr, e + 1) * (power * 0.0625f), element(gr, e + 5) * (power * 0.0625f));
            operands[((((n * kGroups + gr) * 2 + w) * 2 + h) * 2 + 0) * 32 + lane] = *reinterpret_cast<const uint32_t *>(&even);
            operands[((((n * kGroups + gr) * 2 + w) * 2 + h) * 2 + 1) * 32 + lane] = *reinterpret_cast<const uint32_t *>(&odd);
          }
        }
      const float reach = 1.f / power;
      beyond = beyond || !(p.scale_log2 * 0x1p24f * reach < INFINITY);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row_scale[n][i] = __shfl_sync(0xffffffffu, reach, 4 * (2 * t + i));
        bound[n][i] = -INFINITY;
        minus_reference[n][i] = 0.f;
        l_run[n][i] = 0.f;
        last_key[n][i] = paged_visible(part.sequence, (part.row0 + 8 * n + column_row(2 * t + i)) / p.group, a.causal) - 1;
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) q_sum[n][gr][i] = __shfl_sync(0xffffffffu, sums[gr], 4 * (2 * t + i));
#pragma unroll
        for (int gr = 0; gr < kWeighed; ++gr) low_sum[n][gr][i] = 0.f;
      }
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][gr][j][0] = acc[n][gr][j][1] = acc[n][gr][j][2] = acc[n][gr][j][3] = 0.f;
    }
    // The sums' unit, 2^-24, goes into the rows' scale. Where that would leave f32 (queries from about 2^118 / scale on, whose scores may
    // well be finite) it goes into the sums, beside the mask. A scale is not zero, so that what is masked stays at -infinity.
    beyond = __any_sync(0xffffffffu, beyond);
    const float sums_scale = beyond ? 0x1p24f : 1.f;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row_scale[n][i] = fmaxf((beyond ? p.scale_log2 : p.scale_log2 * 0x1p24f) * row_scale[n][i], 0x1p-149f);
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) q_sum[n][gr][i] *= 0x1p-24f;
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) q_frag[n][gr][w][h][odd] = operands[((((n * kGroups + gr) * 2 + w) * 2 + h) * 2 + odd) * 32 + lane];
            q_fix[n][gr][w][h] = q_frag[n][gr][w][h][0] ^ 0x80008000u;
          }
    // Hidden from some row from here on, or all tiles whose sums are scaled.
    const int masked_from = beyond ? 0 : min(part.key_end, paged_visible(part.sequence, part.row0 / p.group, a.causal));

    int stage = 0;                                     // byte offset in the ring
    int key0 = part.first_key;
#pragma unroll 1
    for (int tile = part.tiles; tile > 0; --tile, key0 += kStepKeys) {
      cp_async_wait<S::kStages - 1>();
      __syncwarp();
      const uint8_t *const k_src = ring + stage, *const v_src = k_src + S::kCodeBytes, *const step_src = v_src + S::kCodeBytes;
      // S^T: keys g and g + 8 of each block, in the rows' units
      float score[kTiles][2 * kBlocks][2];             // [tile][key][column]
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        float dot[kTiles][kGroups][4];
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
          const uint2 w0 = *reinterpret_cast<const uint2 *>(k_src + code_offset<S::kRowBytes>(16 * b + g, 2 * gr + (t >> 1)) + 8 * (t & 1));
          const uint2 w1 = *reinterpret_cast<const uint2 *>(k_src + code_offset<S::kRowBytes>(16 * b + g + 8, 2 * gr + (t >> 1)) + 8 * (t & 1));
#pragma unroll
          for (int n = 0; n < kTiles; ++n) dot[n][gr][0] = dot[n][gr][1] = dot[n][gr][2] = dot[n][gr][3] = 0.f;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t x = w ? w0.y : w0.x, y = w ? w1.y : w1.x;
            const uint32_t x0 = x & kBoth, x1 = upper_bytes(x), y0 = y & kBoth, y1 = upper_bytes(y);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
              mma_f16(dot[n][gr], x0, y0, x0 & kOdd, y0 & kOdd, q_frag[n][gr][w][0][0], q_frag[n][gr][w][0][1]);
              mma_f16(dot[n][gr], x1, y1, x1 & kOdd, y1 & kOdd, q_frag[n][gr][w][1][0], q_frag[n][gr][w][1][1]);
              mma_f16(dot[n][gr], x0 & kOdd, y0 & kOdd, x1 & kOdd, y1 & kOdd, q_fix[n][gr][w][0], q_fix[n][gr][w][1]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pairs[kGroups];
          load_steps<kGroups>(step_src + (16 * b + g + 8 * h) * (4 * kGroups), pairs);
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float x = quant_low(pairs[0], kFormat) * q_sum[n][0][i];
#pragma unroll
              for (int gr = 1; gr < kGroups; ++gr) x = fmaf(quant_low(pairs[gr], kFormat), q_sum[n][gr][i], x);
#pragma unroll
              for (int gr = 0; gr < kGroups; ++gr) x = fmaf(quant_step(pairs[gr], kFormat), dot[n][gr][2 * h + i], x);
              score[n][2 * b + h][i] = x;
            }
        }
      }
      if (key0 + kTileKeys > masked_from) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int k = 0; k < 2 * kBlocks; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              score[n][k][i] = key0 + g + 8 * k >= part.key_end || key0 + g + 8 * k > last_key[n][i] ? -INFINITY : score[n][k][i] * sums_scale;
      }
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int k = 0; k < 2 * kBlocks; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) score[n][k][i] = fmaf(score[n][k][i], row_scale[n][i], minus_reference[n][i]);
      uint32_t v_steps[2 * kBlocks][kWeighed], largest_step[kWeighed] = {};
#pragma unroll
      for (int k = 0; k < 2 * kBlocks; ++k) {
        load_steps<kWeighed>(step_src + S::kStepBytes + (g + 8 * k) * (4 * kGroups) + 4 * own_group, v_steps[k]);
#pragma unroll
        for (int gr = 0; gr < kWeighed; ++gr) largest_step[gr] = __vmaxu2(largest_step[gr], v_steps[k][gr]);     // steps are not negative: their bits are in order
      }
      bool moves = false;
#pragma unroll
      for (int gr = 0; gr < kWeighed; ++gr) moves = moves || (largest_step[gr] & 0xffffu) > step_limit[gr];
      float row_top[kTiles][2];
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          row_top[n][i] = score[n][0][i];
#pragma unroll
          for (int k = 1; k < 2 * kBlocks; ++k) row_top[n][i] = fmaxf(row_top[n][i], score[n][k][i]);
          moves = moves || row_top[n][i] > bound[n][i];
        }
      if (__any_sync(0xffffffffu, moves)) {
        // e of the groups that have a step beyond the limit, and references, to the rows' largest scores where those are beyond the bound.
        float change[kWeighed];                          // of 2^e
#pragma unroll
        for (int gr = 0; gr < kWeighed; ++gr) {
          uint32_t most = 0;                             // of the finite ones: others make their group NaN, and no more
#pragma unroll
          for (int k = 0; k < 2 * kBlocks; ++k)
            if ((v_steps[k][gr] & 0xffffu) < kInfinity) most = max(most, v_steps[k][gr] & 0xffffu);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));     // lanes of the same groups
          const int before = exponent[gr];
          if (most > step_limit[gr]) {
            const uint32_t field = __float_as_uint(quant_step(most, kFormat)) >> 23;
            exponent[gr] = min(max(kStepExponent + 127 - static_cast<int>(field), kLeastExponent), kMostExponent);
            step_limit[gr] = narrow_bits(__uint_as_float(min(field + 2, 255u) << 23), kFormat) - 1;
          }
          change[gr] = exp2_fast(static_cast<float>(exponent[gr] - before));     // the first e meets sums of nothing
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = row_top[n][i];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            float shift = 0.f, alpha = 1.f;
            if (top > bound[n][i]) {
              shift = top;
              alpha = bound[n][i] == -INFINITY ? 0.f : exp2_fast(-shift);
              bound[n][i] = kMovesBeyond;
            }
            minus_reference[n][i] -= shift;
#pragma unroll
            for (int k = 0; k < 2 * kBlocks; ++k) score[n][k][i] -= shift;
            l_run[n][i] *= alpha;
#pragma unroll
            for (int gr = 0; gr < kWeighed; ++gr) low_sum[n][gr][i] *= alpha;
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                acc[n][gr][j][i] *= alpha * change[kTwice ? 0 : gr];
                acc[n][gr][j][2 + i] *= alpha * change[kTwice ? 0 : gr];
              }
          }
      }
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        uint32_t p_frag[kTiles][kWeighed][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float pr[2][2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            pr[0][i] = exp2_fast(score[n][2 * b][i]);
            pr[1][i] = exp2_fast(score[n][2 * b + 1][i]);
            l_run[n][i] += pr[0][i] + pr[1][i];
#pragma unroll
            for (int gr = 0; gr < kWeighed; ++gr)
              low_sum[n][gr][i] = fmaf(pr[0][i], middle(v_steps[2 * b][gr]), fmaf(pr[1][i], middle(v_steps[2 * b + 1][gr]), low_sum[n][gr][i]));
          }
          // p' is rounded to f16, as the product's operands are; p itself, in the sum and beside the lows, is not.
#pragma unroll
          for (int gr = 0; gr < kWeighed; ++gr)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float step = quant_step(v_steps[2 * b + h][gr], kFormat) * __uint_as_float(static_cast<uint32_t>(exponent[gr] + 127) << 23);
              const __half2 both = __floats2half2_rn(pr[h][0] * step, pr[h][1] * step);
              p_frag[n][gr][h] = transposed(*reinterpret_cast<const uint32_t *>(&both));
            }
        }
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
          uint32_t x[2][2];                            // keys 2t and 2t + 1 (+ 8): elements 8g .. + 3, .. + 7
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = 16 * b + 2 * t + 8 * h;
            const uint32_t w0 = *reinterpret_cast<const uint32_t *>(v_src + code_offset<S::kRowBytes>(row, 2 * gr + (g >> 2)) + 4 * (g & 3));
            const uint32_t w1 = *reinterpret_cast<const uint32_t *>(v_src + code_offset<S::kRowBytes>(row + 1, 2 * gr + (g >> 2)) + 4 * (g & 3));
            x[h][0] = __byte_perm(w0, w1, 0x5410);
            x[h][1] = __byte_perm(w0, w1, 0x7632);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t u = (j & 1) ? upper_bytes(x[0][j >> 1]) : x[0][j >> 1] & kBoth, w = (j & 1) ? upper_bytes(x[1][j >> 1]) : x[1][j >> 1] & kBoth;
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
              const uint32_t (&weights)[2] = p_frag[n][kTwice ? 0 : gr];
              mma_f16(acc[n][gr][j], kMinusBoth, kMinusOdd, kMinusBoth, kMinusOdd, weights[0], weights[1]);
              mma_f16(acc[n][gr][j], u, u & kOdd, w, w & kOdd, weights[0], weights[1]);
            }
          }
        }
      }
      __syncwarp();   // every lane has read the slot
      issue_tile(ring_addr + stage);
      look_up();
      stage += S::kStageBytes;
      if (stage == S::kRingBytes) stage = 0;
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          l_run[n][i] += __shfl_xor_sync(0xffffffffu, l_run[n][i], off);
#pragma unroll
          for (int gr = 0; gr < kWeighed; ++gr) low_sum[n][gr][i] += __shfl_xor_sync(0xffffffffu, low_sum[n][gr][i], off);
        }
        if (bound[n][i] == -INFINITY) minus_reference[n][i] = INFINITY;
      }
    float unscale[kWeighed];                           // the sums are put together without e
#pragma unroll
    for (int gr = 0; gr < kWeighed; ++gr) unscale[gr] = __uint_as_float(static_cast<uint32_t>(127 - exponent[gr]) << 23);
    // The next part's first tiles are on their way while this one's state is put together. (The ring's groups of copies have all
    // been waited for but the empty ones behind the last tile.)
    const Part done = part;
    more = next_part();
    if (more) fill_ring();
    const bool whole = done.whole();
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {                 // eight rows at a time
      __syncthreads();                                 // the records of the rows before have been read
      float *mine_records = records + warp * (8 * S::kRecord);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = column_row(2 * t + i);
#pragma unroll
        for (int gr = 0; gr < kWeighed; ++gr) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float both = kTwice && own_group ? acc[n][kGroups - 1][j][i] : acc[n][gr][j][i];
            const float odd = kTwice && own_group ? acc[n][kGroups - 1][j][2 + i] : acc[n][gr][j][2 + i];
            v[2 * j] = fmaf((both - odd) * 0x1p24f, unscale[gr], low_sum[n][gr][i]);
            v[2 * j + 1] = fmaf(odd * 0x1p20f, unscale[gr], low_sum[n][gr][i]);
          }
          float4 *to = reinterpret_cast<float4 *>(mine_records + row * S::kRecord + (gr + own_group) * kQuantGroup + 8 * g);
          to[0] = make_float4(v[0], v[1], v[2], v[3]);
          to[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
        if (g == 0 && own_group == 0) *reinterpret_cast<float2 *>(mine_records + row * S::kRecord + kD) = make_float2(-minus_reference[n][i], l_run[n][i]);
      }
      __syncthreads();
      for (int r = warp; r < 8 && r + 8 * n < done.rows; r += kWarps) {      // a warp per row
        float top, l;
        Slice<kD> sum;
        fold_warps<kD, kWarps>(records, r, lane, top, l, sum);
        const int row = r + 8 * n;
        if constexpr (kClustered) {                    // over the first warp's record, which this warp has read
          __syncwarp();
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
          for (int r = warp; r < 8 && r + 8 * n < done.rows; r += kWarps) {
            float top, l;
            Slice<kD> sum;
            fold_cluster<kD>(records + r * S::kRecord, lane, top, l, sum);
            const int packed = done.row0 + r + 8 * n, token = packed / p.group;
            write_row<kBf16, kD>(a, done.sequence.begin + token, done.kv_head * p.group + packed - token * p.group, lane, top, l, sum);
          }
        }
        cluster_sync_all();                            // and are kept until they have been read
      }
    }
    if (!kClustered && done.step0 == 0 && !whole) split = walk.split_of(done);
  }
  cp_async_wait<0>();
  if (!kClustered && threadIdx.x == 0) p.splits[blockIdx.x] = split;
}

using QuantRowsKernel = void (*)(const QuantRowsParams);
// Tiles of 4, 8 or 16 rows (index 0, 1, 2), the narrowest that a sequence's rows fit, as far as the caller says. Four rows share their
// columns with a second group, which head_dim 64 has not.
constexpr int kSizes = 3;
constexpr int size_rows(int size, int head_dim) { return size == 0 ? (head_dim == 128 ? 4 : 8) : 8 * size; }
template <bool kBf16, int kD, int kSize, bool kAligned, bool kClustered>
constexpr QuantRowsKernel rows_kernel() { return attention_quantized_rows_kernel<kBf16, kD, size_rows(kSize, kD), kAligned, kClustered>; }
#define WB200_QUANT_ROWS_KERNELS(D, SIZE, CLUSTERED)                                                     \
  {{rows_kernel<false, D, SIZE, false, CLUSTERED>(), rows_kernel<false, D, SIZE, true, CLUSTERED>()},    \
   {rows_kernel<true, D, SIZE, false, CLUSTERED>(), rows_kernel<true, D, SIZE, true, CLUSTERED>()}}
#define WB200_QUANT_ROWS_SIZES(D, CLUSTERED) \
  {WB200_QUANT_ROWS_KERNELS(D, 0, CLUSTERED), WB200_QUANT_ROWS_KERNELS(D, 1, CLUSTERED), WB200_QUANT_ROWS_KERNELS(D, 2, CLUSTERED)}
const QuantRowsKernel kKernels[2][2][kSizes][2][2] = {      // [clustered][head_dim 128][size][bf16][aligned]
    {WB200_QUANT_ROWS_SIZES(64, false), WB200_QUANT_ROWS_SIZES(128, false)}, {WB200_QUANT_ROWS_SIZES(64, true), WB200_QUANT_ROWS_SIZES(128, true)}};
#define WB200_QUANT_FOLDS(D, SIZE) {attention_paged_fold_kernel<false, D, size_rows(SIZE, D)>, attention_paged_fold_kernel<true, D, size_rows(SIZE, D)>}
void (*const kFoldKernels[2][kSizes][2])(const RowsFold) = {      // [head_dim 128][size][bf16]
    {WB200_QUANT_FOLDS(64, 0), WB200_QUANT_FOLDS(64, 1), WB200_QUANT_FOLDS(64, 2)},
    {WB200_QUANT_FOLDS(128, 0), WB200_QUANT_FOLDS(128, 1), WB200_QUANT_FOLDS(128, 2)}};

constexpr int kMostCtas = ctas_per_sm(8);
size_t rows_record_bytes(int sm_count) { return static_cast<size_t>(sm_count) * kMostCtas * 2 * 16 * kRowRecord<128> * sizeof(float); }
int size_of(const AttentionPagedArgs &a) {
  const int64_t rows = static_cast<int64_t>(a.q_heads / a.cache.kv_heads) * (a.batch.max_query > 0 ? a.batch.max_query : 1);
  return rows <= 4 ? 0 : rows <= 8 ? 1 : 2;
}

}  // namespace

bool attention_quantized_rows_supports(const AttentionPagedArgs &a, const QuantizedRowsArgs &rows) {
  if (a.cache.head_dim != 64 && a.cache.head_dim != 128) return false;
  const uint64_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) |
                        static_cast<uint64_t>((a.q_token | a.q_head | a.out_token | a.out_head) * 2) | reinterpret_cast<uintptr_t>(rows.k.codes) |
                        reinterpret_cast<uintptr_t>(rows.v.codes) |
                        static_cast<uint64_t>(rows.k.codes_page | rows.k.codes_row | rows.k.codes_head | rows.v.codes_page | rows.v.codes_row | rows.v.codes_head);
  const uint64_t steps = reinterpret_cast<uintptr_t>(rows.k.steps) | reinterpret_cast<uintptr_t>(rows.v.steps) |
                         static_cast<uint64_t>((rows.k.steps_page | rows.k.steps_row | rows.k.steps_head | rows.v.steps_page | rows.v.steps_row | rows.v.steps_head) * 4);
  const uint64_t step_bytes = a.cache.head_dim / kQuantGroup * 4;
  // Strides of pages and rows fit 32 bits in units of what they are aligned to.
  const QuantizedRows *both[2] = {&rows.k, &rows.v};
  for (const QuantizedRows *r : both)
    for (const int64_t stride : {r->codes_page / 16, r->codes_row / 16, r->steps_page, r->steps_row})
      if (stride < 0 || stride > 0x7fffffffll) return false;
  return (bits & 15u) == 0 && (steps & (step_bytes - 1)) == 0;     // rows begin on 16 bytes, a row's steps on their size
}

// Clusters where all units' are resident at once and, at the longest the page table can hold, an eighth of a unit's keys go through one
// CTA (16 bytes / ns) in 8 us: the second launch costs about 3, and beyond, equal shares for the whole GPU are the shorter. One launch
// and two, head_dim 128, 16-row pages, per call in a graph: 1 x 8 KV heads, 500 / 2000 / 4000 / 16000 keys 6.6 / 8.0 / 9.9 / 23.4 and
// 9.6 / 10.6 / 11.7 / 17.0 us; 3 x 4 7.3 / 8.5 / 10.7 / 24.2 and 11.9 / 12.7 / 13.5 / 20.2; 4 x 8 8.2 / 10.0 / 13.1 / 33.3 and
// 10.6 / 12.9 / 14.7 / 29.4.
bool attention_quantized_rows_clustered(const AttentionPagedArgs &a, int sm_count) {
  const int64_t units = static_cast<int64_t>(a.batch.sequences) * a.cache.kv_heads;
  if (units * kRowsCluster > sm_count * 2 * 7 / 8) return false;
  const double unit_bytes = (a.cache.head_dim + 8.0 * (a.cache.head_dim / kQuantGroup)) * a.cache.page_size * a.batch.table_width;
  return unit_bytes / kRowsCluster / 16.0 <= 8000.0;
}

size_t attention_quantized_rows_workspace(int sm_count) { return rows_record_bytes(sm_count) + static_cast<size_t>(sm_count) * kMostCtas * sizeof(RowsSplit); }

wb200_status launch_attention_quantized_rows(const AttentionPagedArgs &a, const QuantizedRowsArgs &rows, int sm_count, cudaStream_t stream) {
  const int size = size_of(a), size_row_count = size_rows(size, a.cache.head_dim);
  const unsigned grid = static_cast<unsigned>(sm_count * ctas_per_sm(size_row_count));
  QuantRowsParams p{};
  p.a = a;
  p.rows = rows;
  p.group = a.q_heads / a.cache.kv_heads;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.by_grid = ~0ull / grid + 1;
  const int64_t groups = a.cache.head_dim / kQuantGroup;
  auto shorten = [](int64_t page, int64_t row, int64_t unit) { return ShortStrides{static_cast<uint32_t>(page / unit), static_cast<uint32_t>(row / unit)}; };
  p.k_codes = shorten(rows.k.codes_page, rows.k.codes_row, 16);
  p.v_codes = shorten(rows.v.codes_page, rows.v.codes_row, 16);
  p.k_steps = shorten(rows.k.steps_page, rows.k.steps_row, groups);
  p.v_steps = shorten(rows.v.steps_page, rows.v.steps_row, groups);
  p.step_slots = kStepKeys / a.cache.page_size;
  p.step_rows = kStepKeys % a.cache.page_size;
  p.records = static_cast<float *>(a.workspace);
  p.splits = reinterpret_cast<RowsSplit *>(static_cast<uint8_t *>(a.workspace) + rows_record_bytes(sm_count));
  const int wide = a.cache.head_dim == 128 ? 1 : 0, bf16 = a.cache.format == WB200_BF16 ? 1 : 0;
  static PerDeviceOnce attributes;
  const wb200_status st = attributes.run([]() -> wb200_status {
    for (int d = 0; d < 2; ++d)
      for (int n = 0; n < kSizes; ++n)
        for (int b = 0; b < 2; ++b)
          for (int al = 0; al < 2; ++al)
            for (int c = 0; c < 2; ++c)
              WB200_CUDA_CHECK(cudaFuncSetAttribute(kKernels[c][d][n][b][al], cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                    d ? QuantShape<128>::smem_bytes(size_rows(n, 128)) : QuantShape<64>::smem_bytes(size_rows(n, 64))));
    return WB200_OK;
  });
  if (st != WB200_OK) return st;
  const size_t smem = wide ? QuantShape<128>::smem_bytes(size_row_count) : QuantShape<64>::smem_bytes(size_row_count);
  const bool aligned = a.cache.page_size % kTileKeys == 0;
  if (attention_quantized_rows_clustered(a, sm_count)) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(kRowsCluster, static_cast<unsigned>(a.batch.sequences) * a.cache.kv_heads);
    config.blockDim = dim3(kWarps * 32);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes_of[2];
    attributes_of[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes_of[0].val.programmaticStreamSerializationAllowed = 1;
    attributes_of[1].id = cudaLaunchAttributeClusterDimension;
    attributes_of[1].val.clusterDim.x = kRowsCluster; attributes_of[1].val.clusterDim.y = 1; attributes_of[1].val.clusterDim.z = 1;
    config.attrs = attributes_of;
    config.numAttrs = 2;
    WB200_CUDA_CHECK(cudaLaunchKernelEx(&config, kKernels[1][wide][size][bf16][aligned], p));
    return WB200_OK;
  }
  WB200_CUDA_CHECK(launch_dependent(kKernels[0][wide][size][bf16][aligned], grid, kWarps * 32, smem, stream, p));
  WB200_CUDA_CHECK(launch_dependent(kFoldKernels[wide][size][bf16], dim3(grid, size_row_count), a.cache.head_dim, 0, stream, static_cast<const RowsFold &>(p)));
  return WB200_OK;
}

}  // namespace wb200
