// Rotary positions: every pair of a head's elements is turned by the token's position times the pair's frequency, on rows
// anywhere in memory (wb200_rope), or on the rows of a fused projection with the new K and V rows stored to the pages of a
// KV cache on the way (wb200_rope_append).
//
// The angle. A frequency is given in 2^-64 turns per position, so position * frequency in 64-bit integers IS the angle
// modulo whole turns, for positions of either sign and any size; a product in f32 has lost the angle's fourth digit at
// position 1000 and all of them at 10^6. Of the 64 bits the two highest (rounded) are the quadrant and the rest, within an
// eighth of a turn, keeps 24 significant bits for sincospif. The sines and cosines of a token serve all its heads: a block
// computes them once, into shared memory.
//
// Both kernels are HBM-bound: every element is read once and written once, in 16-byte accesses.
#include "kernels.h"
#include "ptx_sm100.cuh"

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
  sincospif(static_cast<float>(static_cast<int>(rest >> 30)) * 0x1p-33f, &s, &c);   // half turns
  const float sine = (quadrant & 1u) ? c : s, cosine = (quadrant & 1u) ? s : c;
  return make_float2((quadrant & 2u) ? -sine : sine, (quadrant == 1u || quadrant == 2u) ? -cosine : cosine);
}

// kVec elements of storage type kFormat.
template <int kFormat, int kVec>
struct Elements {
  static constexpr int kBytes = (kFormat == WB200_F32 ? 4 : 2) * kVec;
  float v[kVec];
  __device__ __forceinline__ void load(const void *base, int64_t element) {
    if constexpr (kFormat == WB200_F32) {
      const float *p = static_cast<const float *>(base) + element;
      if constexpr (kVec == 4) {
        const float4 w = *reinterpret_cast<const float4 *>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
      } else {
        v[0] = *p;
      }
    } else {
      const uint16_t *p = static_cast<const uint16_t *>(base) + element;
      if constexpr (kVec == 8) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = widen_bits(bits[i] & 0xffffu, kFormat); v[2 * i + 1] = widen_bits(bits[i] >> 16, kFormat); }
      } else {
        v[0] = widen_bits(*p, kFormat);
      }
    }
  }
  __device__ __forceinline__ void store(void *base, int64_t element) const {
    if constexpr (kFormat == WB200_F32) {
      float *p = static_cast<float *>(base) + element;
      if constexpr (kVec == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
      else *p = v[0];
    } else {
      uint16_t *p = static_cast<uint16_t *>(base) + element;
      if constexpr (kVec == 8) {
        uint32_t bits[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) bits[i] = narrow(v[2 * i]) | (narrow(v[2 * i + 1]) << 16);
        *reinterpret_cast<uint4 *>(p) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
      } else {
        *p = static_cast<uint16_t>(narrow(v[0]));
      }
    }
  }
  static __device__ __forceinline__ uint32_t narrow(float x) {
    if constexpr (kFormat == WB200_BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
    else return __half_as_ushort(__float2half_rn(x));
  }
};
// Elements that are only copied keep their bits.
template <int kBytes>
__device__ __forceinline__ void copy_bits(const void *from, void *to) {
  if constexpr (kBytes == 16) *static_cast<uint4 *>(to) = *static_cast<const uint4 *>(from);
  else if constexpr (kBytes == 4) *static_cast<uint32_t *>(to) = *static_cast<const uint32_t *>(from);
  else *static_cast<uint16_t *>(to) = *static_cast<const uint16_t *>(from);
}

// A block takes `tokens_per_block` tokens; an item is 2 * kVec elements of one head: kVec pairs, or elements that are copied.
template <int kFormat, int kVec, bool kAppend>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p, const __grid_constant__ RotaryConstants c) {
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
    // The tokens' sequences: every thread compares some sequences' token ranges with the block's tokens.
    if (threadIdx.x < count) sequence_of[threadIdx.x] = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < p.batch.sequences; s += kThreads) {
      const int begin = max(p.batch.query_starts[s], first), end = min(p.batch.query_starts[s + 1], first + count);
      for (int t = begin; t < end; ++t) sequence_of[t - first] = s;
    }
    __syncthreads();
    if (threadIdx.x < count) {
      const int s = sequence_of[threadIdx.x], token = first + static_cast<int>(threadIdx.x);
      int state = 0;
      if (s >= 0) {
        const int begin = p.batch.query_starts[s], end = p.batch.query_starts[s + 1];
        const long long position = static_cast<long long>(p.batch.key_lengths[s]) - (static_cast<long long>(end) - token);
        if (position < 0 || position >= static_cast<long long>(p.batch.table_width) * p.cache.page_size || begin < 0) {
          raise_status(p.refused, kRefusedLength);
        } else {
          const int slot = static_cast<int>(position / p.cache.page_size), row = static_cast<int>(position - static_cast<long long>(slot) * p.cache.page_size);
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
  const int items_per_token = a.heads * p.items;
  for (int i = threadIdx.x; i < count * items_per_token; i += kThreads) {
    const int t = i / items_per_token, in_token = i - t * items_per_token;
    const int head = in_token / p.items, item = in_token - head * p.items;
    const int64_t src = (first + t) * a.x_token + head * a.x_head;
    void *base = a.out;
    int64_t dst;
    bool rotates = item * kVec < c.pairs;
    int first_copied = 2 * c.pairs;       // where this head's copied elements begin
    int copy_item = item - c.pairs / kVec;
    if constexpr (kAppend) {
      if (!state_of[t]) continue;
      if (head < p.q_heads) {
        dst = (first + t) * a.out_token + head * a.out_head;
      } else if (head < p.q_heads + p.cache.kv_heads) {
        base = p.cache.k;
        dst = k_row[t] + (head - p.q_heads) * p.cache.k_head;
      } else {
        base = p.cache.v;
        dst = v_row[t] + (head - p.q_heads - p.cache.kv_heads) * p.cache.v_head;
        rotates = false;
        first_copied = 0;
        copy_item = item;
      }
    } else {
      dst = (first + t) * a.out_token + head * a.out_head;
    }
    if (rotates) {
      const int pair = item * kVec;
      const float2 *turn = angles + t * c.pairs + pair;
      Elements<kFormat, kVec> lo, hi;
      if (a.interleaved) {
        lo.load(a.x, src + 2 * pair);
        hi.load(a.x, src + 2 * pair + kVec);
        if constexpr (kVec == 1) {
          const float x = lo.v[0], y = hi.v[0];
          lo.v[0] = fmaf(x, turn[0].y, -(y * turn[0].x));
          hi.v[0] = fmaf(y, turn[0].y, x * turn[0].x);
        } else {
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) {
            const float2 u = turn[e], w = turn[kVec / 2 + e];
            const float x = lo.v[2 * e], y = lo.v[2 * e + 1], z = hi.v[2 * e], q = hi.v[2 * e + 1];
            lo.v[2 * e] = fmaf(x, u.y, -(y * u.x));
            lo.v[2 * e + 1] = fmaf(y, u.y, x * u.x);
            hi.v[2 * e] = fmaf(z, w.y, -(q * w.x));
            hi.v[2 * e + 1] = fmaf(q, w.y, z * w.x);
          }
        }
        lo.store(base, dst + 2 * pair);
        hi.store(base, dst + 2 * pair + kVec);
      } else {
        lo.load(a.x, src + pair);
        hi.load(a.x, src + c.pairs + pair);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float x = lo.v[e], y = hi.v[e];
          lo.v[e] = fmaf(x, turn[e].y, -(y * turn[e].x));
          hi.v[e] = fmaf(y, turn[e].y, x * turn[e].x);
        }
        lo.store(base, dst + pair);
        hi.store(base, dst + c.pairs + pair);
      }
    } else {
      const int d = first_copied + 2 * kVec * copy_item;
      const uint8_t *from = static_cast<const uint8_t *>(a.x) + (src + d) * kElementBytes;
      uint8_t *to = static_cast<uint8_t *>(base) + (dst + d) * kElementBytes;
      if (d + kVec <= a.head_dim) copy_bits<kElementBytes * kVec>(from, to);
      if (d + 2 * kVec <= a.head_dim) copy_bits<kElementBytes * kVec>(from + kElementBytes * kVec, to + kElementBytes * kVec);
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
  // Tokens of few heads share a block, once there are blocks for every SM: 512 items keep its threads busy.
  const int items_per_token = a.heads * p.items;
  int per_block = (512 + items_per_token - 1) / items_per_token;
  if (per_block > kMaxTokensPerBlock) per_block = kMaxTokensPerBlock;
  if (c.pairs > 0 && per_block > kMaxAnglesPerBlock / c.pairs) per_block = kMaxAnglesPerBlock / c.pairs;
  while (per_block > 1 && a.tokens / per_block < 592) --per_block;
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
