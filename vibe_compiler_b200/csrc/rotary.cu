// Rotary positions: every pair of a head's elements is turned by the token's position times the pair's frequency, on rows
// anywhere in memory (wb200_rope), or on the rows of a fused projection with the new K and V rows stored to the pages of a
// KV cache on the way (wb200_rope_append).
//
// The angle. A frequency is given in 2^-64 turns per position, so position * frequency in 64-bit integers IS the angle
// modulo whole turns, for positions of either sign and any size; a product in f32 has lost the angle's fourth digit at
// position 1000 and all of them at 10^6. Of the 64 bits the two highest (rounded) are the quadrant and the rest, within an
// eighth of a turn, is rounded to 24 significant bits of its own for sincospif, so that the small sines of slow pairs are as
// right as any. The sines and cosines of a token serve all its heads: a block computes them once, into shared memory.
//
// Both kernels are HBM-bound: every element is read once and written once, in 16-byte accesses; measured at launch() below.
#include "attention_paged.cuh"

namespace wb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokensPerBlock = 16;
constexpr int kMaxAnglesPerBlock = 2048;   // (sin, cos) pairs in shared memory
static_assert(kMaxRotaryPairs <= kMaxAnglesPerBlock, "one token's angles must fit");

struct RotaryParams {
  RopeArgs a;
  int tokens_per_block;
  int items;             // per head: an item is 2 * kVec elements, kVec pairs in front of the first copied element
  // with a cache
  PagedCacheArgs cache;
  PagedBatchArgs batch;
  int q_heads;
  int *refused;
};

__device__ __forceinline__ float2 sin_cos_of_turns(unsigned long long phase) {
  const unsigned int quadrant = static_cast<unsigned int>((phase + (1ull << 61)) >> 62) & 3u;
  const long long rest = static_cast<long long>(phase - (static_cast<unsigned long long>(quadrant) << 62));   // +- 2^61
  float s, c;
  sincospif(static_cast<float>(rest) * 0x1p-63f, &s, &c);   // half turns
  const float sine = (quadrant & 1u) ? c : s, cosine = (quadrant & 1u) ? s : c;
  return make_float2((quadrant & 2u) ? -sine : sine, (quadrant == 1u || quadrant == 2u) ? -cosine : cosine);
}

// kVec elements of storage type kFormat, as they are stored: elements that are only copied keep their bits.
template <int kFormat, int kVec>
struct Elements {
  static constexpr int kWords = kFormat == WB200_F32 ? kVec : (kVec + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void *p) {
    if constexpr (kVec > 1) *reinterpret_cast<uint4 *>(w) = *static_cast<const uint4 *>(p);
    else if constexpr (kFormat == WB200_F32) w[0] = *static_cast<const uint32_t *>(p);
    else w[0] = *static_cast<const uint16_t *>(p);
  }
  __device__ __forceinline__ void store(void *p) const {
    if constexpr (kVec > 1) *static_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(w);
    else if constexpr (kFormat == WB200_F32) *static_cast<uint32_t *>(p) = w[0];
    else *static_cast<uint16_t *>(p) = static_cast<uint16_t>(w[0]);
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (kFormat == WB200_F32) return __uint_as_float(w[i]);
    else return widen_bits(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu, kFormat);
  }
  // Elements i (even) and i + 1; the last of an odd count by itself.
  __device__ __forceinline__ void set(int i, float lo, float hi) {
    if constexpr (kFormat == WB200_F32) {
      w[i] = __float_as_uint(lo);
      if constexpr (kVec > 1) w[i + 1] = __float_as_uint(hi);
    } else if constexpr (kFormat == WB200_BF16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
      w[i >> 1] = *reinterpret_cast<const uint32_t *>(&v);
    } else {
      const __half2 v = __floats2half2_rn(lo, hi);
      w[i >> 1] = *reinterpret_cast<const uint32_t *>(&v);
    }
  }
};
// Turns the pairs of two vectors by (sin, cos) of turns[i]: (v0[i], v1[i]) in the half layout, neighbours when interleaved.
template <int kFormat, int kVec>
__device__ __forceinline__ void turn(Elements<kFormat, kVec> &v0, Elements<kFormat, kVec> &v1, const float2 *turns, int interleaved) {
  if constexpr (kVec == 1) {
    const float x = v0.get(0), y = v1.get(0);
    const float2 u = turns[0];
    v0.set(0, fmaf(x, u.y, -(y * u.x)), 0.f);
    v1.set(0, fmaf(y, u.y, x * u.x), 0.f);
  } else if (interleaved) {
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
      const float2 u = turns[i / 2], w = turns[kVec / 2 + i / 2];
      const float x = v0.get(i), y = v0.get(i + 1), z = v1.get(i), q = v1.get(i + 1);
      v0.set(i, fmaf(x, u.y, -(y * u.x)), fmaf(y, u.y, x * u.x));
      v1.set(i, fmaf(z, w.y, -(q * w.x)), fmaf(q, w.y, z * w.x));
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
      const float2 u = turns[i], w = turns[i + 1];
      const float x = v0.get(i), y = v1.get(i), z = v0.get(i + 1), q = v1.get(i + 1);
      v0.set(i, fmaf(x, u.y, -(y * u.x)), fmaf(z, w.y, -(q * w.x)));
      v1.set(i, fmaf(y, u.y, x * u.x), fmaf(q, w.y, z * w.x));
    }
  }
}

// A block takes `tokens_per_block` tokens; an item is 2 * kVec elements of one head: kVec pairs, or elements that are copied.
template <int kFormat, int kVec, bool kAppend>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(const __grid_constant__ RotaryParams p, const __grid_constant__ RotaryConstants c) {
  constexpr int kElementBytes = kFormat == WB200_F32 ? 4 : 2;
  __shared__ float2 angles[kMaxAnglesPerBlock];
  __shared__ int64_t k_row[kMaxTokensPerBlock], v_row[kMaxTokensPerBlock];   // element offsets of the tokens' cache rows
  __shared__ long long position_of[kMaxTokensPerBlock];
  __shared__ int sequence_of[kMaxTokensPerBlock], state_of[kMaxTokensPerBlock];
  const RopeArgs &a = p.a;
  const int first = blockIdx.x * p.tokens_per_block;
  const int count = min(p.tokens_per_block, a.tokens - first);
  pdl_wait();
  pdl_launch_dependents();
  if constexpr (kAppend) {
    // The tokens' sequences: every thread compares some sequences' token ranges with the block's tokens. A range that is not one of
    // the rows' is reported whether or not a token of the block lies in it.
    if (threadIdx.x < count) sequence_of[threadIdx.x] = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < p.batch.sequences; s += kThreads) {
      const int begin = p.batch.query_starts[s], end = p.batch.query_starts[s + 1];
      if (begin < end && (begin < 0 || end > a.tokens)) {
        raise_status(p.refused, kRefusedLength);
        continue;
      }
      for (int t = max(begin, first); t < min(end, first + count); ++t) sequence_of[t - first] = s;
    }
    __syncthreads();
    if (threadIdx.x < count) {
      const int s = sequence_of[threadIdx.x], token = first + static_cast<int>(threadIdx.x);
      int state = 0;
      // What attention would leave out as a whole is not written here in part: its positions mean nothing.
      const PagedSequence sequence = s >= 0 ? paged_sequence(p.batch, p.cache, s, p.refused, true) : PagedSequence{0, 0, 0};
      if (sequence.count > 0) {
        const int position = sequence.keys - sequence.count + (token - sequence.begin);      // less than keys, which the table holds
        if (position < 0) {
          raise_status(p.refused, kRefusedLength);
        } else {
          const int slot = position / p.cache.page_size, row = position - slot * p.cache.page_size;
          const int page = p.batch.page_table[s * p.batch.table_stride + slot];
          if (page < 0 || page >= p.cache.pages) {
            raise_status(p.refused, kRefusedPage);
          } else {
            state = 1;
            k_row[threadIdx.x] = page * p.cache.k_page + row * p.cache.k_row;
            v_row[threadIdx.x] = page * p.cache.v_page + row * p.cache.v_row;
            position_of[threadIdx.x] = position;
          }
        }
      }
      state_of[threadIdx.x] = state;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < count * c.pairs; i += kThreads) {
    const int t = i / c.pairs, pair = i - t * c.pairs;
    long long position;
    if (kAppend && !a.positions) position = state_of[t] ? position_of[t] : 0;
    else position = a.position_bytes == 8 ? static_cast<const long long *>(a.positions)[first + t] : static_cast<const int *>(a.positions)[first + t];
    float2 sc = sin_cos_of_turns(static_cast<unsigned long long>(position) * c.turns[pair]);
    if (a.backward) sc.x = -sc.x;
    angles[i] = make_float2(sc.x * c.magnitude, sc.y * c.magnitude);
  }
  __syncthreads();
  // A thread keeps to one item of the head (or every lanes-th) and takes every groups-th head of the block's tokens; nothing is
  // divided in the loop.
  const int lanes = min(p.items, kThreads), groups = kThreads / lanes, group = static_cast<int>(threadIdx.x) / lanes;
  if (group >= groups) return;
  for (int item = static_cast<int>(threadIdx.x) - group * lanes; item < p.items; item += lanes) {
    int t = 0, head = group;
    while (true) {
      while (head >= a.heads) { head -= a.heads; ++t; }
      if (t >= count) break;
      int64_t dst = (first + t) * a.out_token + head * a.out_head;
      uint8_t *base = static_cast<uint8_t *>(a.out);
      bool rotates = item * kVec < c.pairs, live = true;
      if constexpr (kAppend) {
        live = state_of[t] != 0;
        if (head >= p.q_heads + p.cache.kv_heads) {
          base = static_cast<uint8_t *>(p.cache.v);
          dst = v_row[t] + (head - p.q_heads - p.cache.kv_heads) * p.cache.v_head;
          rotates = false;
        } else if (head >= p.q_heads) {
          base = static_cast<uint8_t *>(p.cache.k);
          dst = k_row[t] + (head - p.q_heads) * p.cache.k_head;
        }
      }
      if (live) {
        // The item's two vectors: of the pairs, or the 2 kVec elements in their place where they are copied.
        const int d0 = (rotates && !a.interleaved ? 1 : 2) * item * kVec, d1 = d0 + (rotates && !a.interleaved ? c.pairs : kVec);
        const bool has1 = d1 + kVec <= a.head_dim;
        const uint8_t *x = static_cast<const uint8_t *>(a.x) + ((first + t) * a.x_token + head * a.x_head) * kElementBytes;
        Elements<kFormat, kVec> v0, v1;
        v0.load(x + static_cast<int64_t>(d0) * kElementBytes);
        if (has1) v1.load(x + static_cast<int64_t>(d1) * kElementBytes);
        if (rotates) turn(v0, v1, angles + t * c.pairs + item * kVec, a.interleaved);
        v0.store(base + (dst + d0) * kElementBytes);
        if (has1) v1.store(base + (dst + d1) * kElementBytes);
      }
      head += groups;
    }
  }
}

template <bool kAppend>
wb200_status launch(RotaryParams p, const RotaryConstants &c, bool aligned, cudaStream_t stream) {
  const RopeArgs &a = p.a;
  const int vec = a.format == WB200_F32 ? 4 : 8;
  // 16-byte accesses where every row begins on 16 bytes and the pairs and the copied elements come in whole vectors.
  const bool wide = aligned && c.pairs % vec == 0 && a.head_dim % vec == 0;
  const int step = 2 * (wide ? vec : 1);
  p.items = (a.head_dim + step - 1) / step;   // rotated pairs fill whole items
  // A block's threads pass over its tokens' heads about twice, so that the eight blocks of an SM overlap one another's positions,
  // angles, loads and stores; few tokens get a block each. Gradient of 16384 x 40 x 128 bf16 (336 MB, 51 us at the copy rate) and
  // prompts of 13 thousand tokens x 48 heads: 60 / 73 us; four passes 61 / 74, eight 61 / 76, sixteen 72 / 88; two heads of a thread
  // in flight 65 / 84 (58 registers, four blocks to an SM); blocks of 128 threads 67 / 84, of 512 70 / 78.
  const int groups = p.items < kThreads ? kThreads / p.items : 1;
  int per_block = (2 * groups + a.heads - 1) / a.heads;
  if (per_block > kMaxTokensPerBlock) per_block = kMaxTokensPerBlock;
  if (c.pairs > 0 && per_block > kMaxAnglesPerBlock / c.pairs) per_block = kMaxAnglesPerBlock / c.pairs;
  while (per_block > 1 && a.tokens / per_block < 148 * 8) --per_block;
  p.tokens_per_block = per_block;
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(a.tokens) + per_block - 1) / per_block);
  void (*kernel)(const RotaryParams, const RotaryConstants);
  if (a.format == WB200_F32) kernel = wide ? rotary_kernel<WB200_F32, 4, kAppend> : rotary_kernel<WB200_F32, 1, kAppend>;
  else if (a.format == WB200_BF16) kernel = wide ? rotary_kernel<WB200_BF16, 8, kAppend> : rotary_kernel<WB200_BF16, 1, kAppend>;
  else kernel = wide ? rotary_kernel<WB200_F16, 8, kAppend> : rotary_kernel<WB200_F16, 1, kAppend>;
  WB200_CUDA_CHECK(launch_dependent(kernel, blocks, kThreads, 0, stream, p, c));
  return WB200_OK;
}

bool rows_aligned(const void *base, int64_t stride0, int64_t stride1, int element_bytes, int64_t stride2 = 0) {
  return ((reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(stride0 * element_bytes) | static_cast<uint64_t>(stride1 * element_bytes) |
           static_cast<uint64_t>(stride2 * element_bytes)) & 15u) == 0;
}

}  // namespace

wb200_status launch_rope(const RopeArgs &a, const RotaryConstants &c, cudaStream_t stream) {
  RotaryParams p{};
  p.a = a;
  const int bytes = a.format == WB200_F32 ? 4 : 2;
  return launch<false>(p, c, rows_aligned(a.x, a.x_token, a.x_head, bytes) && rows_aligned(a.out, a.out_token, a.out_head, bytes), stream);
}

wb200_status launch_rope_append(const RopeArgs &a, const RotaryConstants &c, const PagedCacheArgs &cache, const PagedBatchArgs &batch, int *refused,
                                cudaStream_t stream) {
  RotaryParams p{};
  p.a = a;
  p.cache = cache;
  p.batch = batch;
  p.q_heads = a.heads - 2 * cache.kv_heads;
  p.refused = refused;
  const bool aligned = rows_aligned(a.x, a.x_token, a.x_head, 2) && rows_aligned(a.out, a.out_token, a.out_head, 2) &&
                       rows_aligned(cache.k, cache.k_page, cache.k_row, 2, cache.k_head) && rows_aligned(cache.v, cache.v_page, cache.v_row, 2, cache.v_head);
  return launch<true>(p, c, aligned, stream);
}

}  // namespace wb200
