// Rotary positions: every pair of a head's elements is turned by the token's position times the pair's frequency, on rows
// anywhere in memory (wb200_rope), or on the rows of a fused projection with the new K and V rows stored to the pages of a
// KV cache on the way (wb200_rope_append), or quantised on the way (wb200_rope_append_quantized).
//
// The angle. A frequency is given in 2^-64 turns per position, so position * frequency in 64-bit integers IS the angle
// modulo whole turns, for positions of either sign and any size; a product in f32 has lost the angle's fourth digit at
// position 1000 and all of them at 10^6. Of the 64 bits the two highest (rounded) are the quadrant and the rest, within an
// eighth of a turn, is rounded to 24 significant bits of its own for sincospif, so that the small sines of slow pairs are as
// right as any. The sines and cosines of a token serve all its heads: a block computes them once, into shared memory.
//
// The first two are HBM-bound: every element is read once and written once, in 16-byte accesses; measured at launch() below. The one that
// quantises waits for memory, shared memory and barriers: at launch_rope_append_quantized().
#include "attention_paged.cuh"
#include "quantized_rows.cuh"

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
    if (threadIdx.x < count) state_of[threadIdx.x] = 0;
    place_tokens(p.batch, p.cache, first, count, p.refused, sequence_of, [&](int t, int page, int row, int position) {
      state_of[t] = 1;
      k_row[t] = page * p.cache.k_page + row * p.cache.k_row;
      v_row[t] = page * p.cache.v_page + row * p.cache.v_row;
      position_of[t] = position;
    });
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

// Sine and cosine as sums of two f32: (sine, its rest, cosine, its rest).
__device__ __forceinline__ float4 fine_sin_cos_of_turns(unsigned long long phase, float magnitude) {
  double s, c;
  sincospi(static_cast<double>(static_cast<long long>(phase)) * 0x1p-63, &s, &c);
  s *= magnitude;
  c *= magnitude;
  const float sine = static_cast<float>(s), cosine = static_cast<float>(c);
  return make_float4(sine, static_cast<float>(s - sine), cosine, static_cast<float>(c - cosine));
}
// a * (x + xr) + b * (y + yr), rounded once to f32: the products and their sum with what they leave (an FMA gives a product's rounding
// error, Knuth's two-sum a sum's), good to about 2^-46 of the larger product.
__device__ __forceinline__ float fine_sum(float a, float x, float xr, float b, float y, float yr) {
  const float p = __fmul_rn(a, x), q = __fmul_rn(b, y), sum = __fadd_rn(p, q), q_part = __fsub_rn(sum, p);
  const float left = __fadd_rn(__fsub_rn(p, __fsub_rn(sum, q_part)), __fsub_rn(q, q_part));
  const float products = __fadd_rn(__fmaf_rn(a, x, -p), __fmaf_rn(b, y, -q));
  return __fadd_rn(sum, __fadd_rn(left, __fmaf_rn(a, xr, __fmaf_rn(b, yr, products))));
}

// Rows of the fused projection with K and V quantised on the way to their pages. Q as above. Of a K or V row a lane takes sixteen
// elements, a quad of lanes a group of 64, whose least and largest element it finds by two shuffles.
// K is turned as if in more than f32 and rounded once to f32 and to the type: a code is a decision next to a border, and so is a step's
// rounding, so the f32 rotation's last bit would give codes that differ between this kernel and the definition (and any other that
// follows it) in one group of 30 thousand, by a whole step in an element of ten there. It takes fifteen f32 operations an element.
constexpr int kMaxQuantizeAngles = 1024;
template <int kFormat, bool kWide>
__global__ void __launch_bounds__(kThreads) rotary_quantize_kernel(const __grid_constant__ RotaryParams p, const __grid_constant__ QuantizedRowsArgs rows,
                                                                   const __grid_constant__ RotaryConstants c) {
  constexpr int kVec = kWide ? 8 : 1;
  __shared__ float2 angles[kMaxQuantizeAngles];
  __shared__ float4 fine_angles[kMaxQuantizeAngles];
  __shared__ int64_t codes_at[2][kMaxTokensPerBlock], steps_at[2][kMaxTokensPerBlock];    // of the token's row, of K and of V
  __shared__ int state_of[kMaxTokensPerBlock], position_of[kMaxTokensPerBlock];
  __shared__ int sequence_of[kMaxTokensPerBlock];
  const RopeArgs &a = p.a;
  const int first = blockIdx.x * p.tokens_per_block;
  const int count = min(p.tokens_per_block, a.tokens - first);
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < count) state_of[threadIdx.x] = 0;
  place_tokens(p.batch, p.cache, first, count, p.refused, sequence_of, [&](int t, int page, int row, int position) {
    state_of[t] = 1;
    position_of[t] = position;
    codes_at[0][t] = page * rows.k.codes_page + row * rows.k.codes_row;
    codes_at[1][t] = page * rows.v.codes_page + row * rows.v.codes_row;
    steps_at[0][t] = page * rows.k.steps_page + row * rows.k.steps_row;
    steps_at[1][t] = page * rows.v.steps_page + row * rows.v.steps_row;
  });
  for (int i = threadIdx.x; i < count * c.pairs; i += kThreads) {
    const int t = i / c.pairs, pair = i - t * c.pairs;
    long long position;
    if (!a.positions) position = state_of[t] ? position_of[t] : 0;
    else position = a.position_bytes == 8 ? static_cast<const long long *>(a.positions)[first + t] : static_cast<const int *>(a.positions)[first + t];
    const unsigned long long phase = static_cast<unsigned long long>(position) * c.turns[pair];
    const float2 sc = sin_cos_of_turns(phase);
    angles[i] = make_float2(sc.x * c.magnitude, sc.y * c.magnitude);
    fine_angles[i] = fine_sin_cos_of_turns(phase, c.magnitude);
  }
  __syncthreads();
  const uint16_t *const x_rows = static_cast<const uint16_t *>(a.x);
  // Q: a thread keeps to one item of the head and takes every groups-th head of the block's tokens.
  const int lanes = min(p.items, kThreads), groups = kThreads / lanes, group = static_cast<int>(threadIdx.x) / lanes;
  if (group < groups && p.q_heads > 0) {
    for (int item = static_cast<int>(threadIdx.x) - group * lanes; item < p.items; item += lanes) {
      int t = 0, head = group;
      while (true) {
        while (head >= p.q_heads) { head -= p.q_heads; ++t; }
        if (t >= count) break;
        if (state_of[t]) {
          const bool rotates = item * kVec < c.pairs;
          const int d0 = (rotates && !a.interleaved ? 1 : 2) * item * kVec, d1 = d0 + (rotates && !a.interleaved ? c.pairs : kVec);
          const bool has1 = d1 + kVec <= a.head_dim;
          const uint16_t *x = x_rows + (first + t) * a.x_token + head * a.x_head;
          uint16_t *out = static_cast<uint16_t *>(a.out) + (first + t) * a.out_token + head * a.out_head;
          Elements<kFormat, kVec> v0, v1;
          v0.load(x + d0);
          if (has1) v1.load(x + d1);
          if (rotates) turn(v0, v1, angles + t * c.pairs + item * kVec, a.interleaved);
          v0.store(out + d0);
          if (has1) v1.store(out + d1);
        }
        head += groups;
      }
    }
  }
  // K and V: rows of 4, 8 or 16 lanes, sixteen elements a lane.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = a.head_dim <= 64 ? 2 : a.head_dim <= 128 ? 3 : 4;
  const int at_once = 32 >> shift, heads = 2 * p.cache.kv_heads, all = count * heads;
  const int slot = lane & ((1 << shift) - 1), e0 = 16 * slot, octets = max(0, min(2, (a.head_dim - e0) >> 3));
  int t = (warp * at_once + (lane >> shift)) / heads, row_head = warp * at_once + (lane >> shift) - t * heads;
#pragma unroll 1
  for (int base = warp * at_once; base < all; base += (kThreads / 32) * at_once, row_head += (kThreads / 32) * at_once) {
    while (row_head >= heads) { row_head -= heads; ++t; }
    const bool is_v = row_head >= p.cache.kv_heads;
    const int head = row_head - (is_v ? p.cache.kv_heads : 0);
    const int live = t < count && state_of[t] ? octets : 0;
    uint32_t v[8] = {};                                // as it is quantised: two elements to a word
    const uint16_t *const x = x_rows + static_cast<int64_t>(first + t) * a.x_token + (p.q_heads + row_head) * a.x_head;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      if (o >= live) continue;
      const int e1 = e0 + 8 * o;
      Elements<kFormat, kVec> own[8 / kVec];
#pragma unroll
      for (int i = 0; i < 8 / kVec; ++i) own[i].load(x + e1 + i * kVec);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * o + i] = kWide ? own[0].w[i & (Elements<kFormat, kVec>::kWords - 1)] : own[2 * i / kVec].w[0] | (own[(2 * i + 1) / kVec].w[0] << 16);
      if (is_v || e1 >= 2 * c.pairs) continue;
      const float4 *turns = fine_angles + t * c.pairs;
      auto element = [&](int i) { return own[i / kVec].get(i % kVec); };
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          if (!kWide && e1 + i >= 2 * c.pairs) break;
          const float4 u = turns[(e1 + i) >> 1];
          const float b = element(i), w = element(i + 1);
          v[4 * o + (i >> 1)] = narrow_pair<kFormat>(fine_sum(b, u.z, u.w, -w, u.x, u.y), fine_sum(w, u.z, u.w, b, u.x, u.y));
        }
      } else {
        Elements<kFormat, kVec> other[8 / kVec];
#pragma unroll
        for (int i = 0; i < 8 / kVec; ++i) {
          const int e = e1 + i * kVec;
          if (e < 2 * c.pairs) other[i].load(x + (e < c.pairs ? e + c.pairs : e - c.pairs));
        }
        // Only rows with narrow accesses have elements that are copied beside others that are turned.
        auto turned = [&](int i) {
          const int e = e1 + i;
          if (!kWide && e >= 2 * c.pairs) return element(i);
          const float4 u = turns[e < c.pairs ? e : e - c.pairs];
          const float partner = other[i / kVec].get(i % kVec);
          return fine_sum(element(i), u.z, u.w, e < c.pairs ? -partner : partner, u.x, u.y);
        };
#pragma unroll
        for (int i = 0; i < 8; i += 2) v[4 * o + (i >> 1)] = narrow_pair<kFormat>(turned(i), turned(i + 1));
      }
    }
    uint32_t pair;
    const uint2 words = quantize16<kFormat>(v, live, &pair);
    if (live > 0) {
      const QuantizedRows &to = is_v ? rows.v : rows.k;
      uint32_t *codes = reinterpret_cast<uint32_t *>(to.codes + codes_at[is_v][t] + head * to.codes_head) + 2 * slot;
      codes[0] = words.x;
      if (live > 1) codes[1] = words.y;
      if ((slot & 3) == 0) to.steps[steps_at[is_v][t] + head * to.steps_head + (slot >> 2)] = pair;
    }
  }
}

// A block's threads pass over its tokens' heads about `passes` times, so that the blocks of an SM overlap one another's positions,
// angles, loads and stores; few tokens get a block each.
int tokens_per_block(const RopeArgs &a, const RotaryConstants &c, int items, int passes, int most_angles) {
  const int groups = items < kThreads ? kThreads / items : 1;
  int per_block = (passes * groups + a.heads - 1) / a.heads;
  if (per_block > kMaxTokensPerBlock) per_block = kMaxTokensPerBlock;
  if (c.pairs > 0 && per_block > most_angles / c.pairs) per_block = most_angles / c.pairs;
  while (per_block > 1 && a.tokens / per_block < 148 * 8) --per_block;
  return per_block;
}

template <bool kAppend>
wb200_status launch(RotaryParams p, const RotaryConstants &c, bool aligned, cudaStream_t stream) {
  const RopeArgs &a = p.a;
  const int vec = a.format == WB200_F32 ? 4 : 8;
  // 16-byte accesses where every row begins on 16 bytes and the pairs and the copied elements come in whole vectors.
  const bool wide = aligned && c.pairs % vec == 0 && a.head_dim % vec == 0;
  const int step = 2 * (wide ? vec : 1);
  p.items = (a.head_dim + step - 1) / step;   // rotated pairs fill whole items
  // Gradient of 16384 x 40 x 128 bf16 (336 MB, 51 us at the copy rate) and prompts of 13 thousand tokens x 48 heads: 60 / 73 us; four
  // passes of a block 61 / 74, eight 61 / 76, sixteen 72 / 88; two heads of a thread in flight 65 / 84 (58 registers, four blocks to
  // an SM); blocks of 128 threads 67 / 84, of 512 70 / 78.
  const int per_block = tokens_per_block(a, c, p.items, 2, kMaxAnglesPerBlock);
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

wb200_status launch_rope_append_quantized(const RopeArgs &a, const RotaryConstants &c, const PagedCacheArgs &cache, const QuantizedRowsArgs &rows,
                                          const PagedBatchArgs &batch, int *refused, cudaStream_t stream) {
  RotaryParams p{};
  p.a = a;
  p.cache = cache;
  p.batch = batch;
  p.q_heads = a.heads - 2 * cache.kv_heads;
  p.refused = refused;
  // head_dim is a multiple of 8
  const bool wide = rows_aligned(a.x, a.x_token, a.x_head, 2) && rows_aligned(a.out, a.out_token, a.out_head, 2) && c.pairs % 8 == 0;
  const int step = wide ? 16 : 2;
  p.items = (a.head_dim + step - 1) / step;
  // Prompts of 12174 tokens, 32/8 heads, bf16, with two / four / eight passes (eight elements a lane then): 116 / 108 / 114 us; now 89,
  // of 40 for its 263 MB at the copy rate.
  p.tokens_per_block = tokens_per_block(a, c, p.items, 4, kMaxQuantizeAngles);
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(a.tokens) + p.tokens_per_block - 1) / p.tokens_per_block);
  const bool bf16 = a.format == WB200_BF16;
  const auto kernel = wide ? (bf16 ? rotary_quantize_kernel<WB200_BF16, true> : rotary_quantize_kernel<WB200_F16, true>)
                           : (bf16 ? rotary_quantize_kernel<WB200_BF16, false> : rotary_quantize_kernel<WB200_F16, false>);
  WB200_CUDA_CHECK(launch_dependent(kernel, blocks, kThreads, 0, stream, p, rows, c));
  return WB200_OK;
}

}  // namespace wb200
