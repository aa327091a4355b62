// Attention over a paged KV cache, the general kernel: any head dimension that is a multiple of 8, up to 256, any page size and
// any strides. A warp takes one row (token, query head) and walks its keys 32 at a time: a lane scores one key, the warp
// carries the running maximum and sum in f32, and every lane accumulates eight elements of the row.
#include "attention_paged.cuh"

namespace wb200 {
namespace {

constexpr int kRows = 4;            // rows (warps) per block
constexpr int kMaxHeadDim = 256;

template <int kFormat, bool kWide>
__device__ __forceinline__ void load8(const uint16_t *p, float (&v)[8]) {
  uint32_t w[4];
  if constexpr (kWide) {
    *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = widen_bits(w[i] & 0xffffu, kFormat); v[2 * i + 1] = widen_bits(w[i] >> 16, kFormat); }
}

template <int kFormat, bool kWide>
__global__ void __launch_bounds__(kRows * 32) attention_paged_general_kernel(const __grid_constant__ AttentionPagedArgs a) {
  __shared__ float q_rows[kRows][kMaxHeadDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + warp;
  pdl_wait();
  pdl_launch_dependents();
  const int token = static_cast<int>(row / a.q_heads), head = static_cast<int>(row - static_cast<int64_t>(token) * a.q_heads);
  if (token >= a.batch.tokens) return;
  int s = -1;
  for (int base = 0; base < a.batch.sequences && s < 0; base += 32) {
    const int i = base + lane;
    const bool mine = i < a.batch.sequences && a.batch.query_starts[i] <= token && token < a.batch.query_starts[i + 1];
    const unsigned int found = __ballot_sync(0xffffffffu, mine);
    if (found) s = base + __ffs(found) - 1;
  }
  if (s < 0) return;                // a token of no sequence
  const PagedSequence sequence = paged_sequence(a.batch, a.cache, s, a.refused, lane == 0);
  if (sequence.count == 0) return;
  const int visible = paged_visible(sequence, token - sequence.begin, a.causal);
  const int kv_head = head / (a.q_heads / a.cache.kv_heads), d = a.cache.head_dim;
  const uint16_t *q = static_cast<const uint16_t *>(a.q) + token * a.q_token + head * a.q_head;
  for (int i = lane; i < d; i += 32) q_rows[warp][i] = widen_bits(q[i], kFormat);
  __syncwarp();
  const float scale_log2 = a.scale * 1.4426950408889634f;
  const int *pages = a.batch.page_table + s * a.batch.table_stride;
  const uint16_t *k = static_cast<const uint16_t *>(a.cache.k) + kv_head * a.cache.k_head;
  const uint16_t *v = static_cast<const uint16_t *>(a.cache.v) + kv_head * a.cache.v_head;
  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  for (int base = 0; base < visible; base += 32) {
    const int key = base + lane;
    float score = -INFINITY;
    long long v_at = -1;
    if (key < visible) {
      const int slot = key / a.cache.page_size, in_page = key - slot * a.cache.page_size, page = pages[slot];
      if (page < 0 || page >= a.cache.pages) {
        raise_status(a.refused, kRefusedPage);
      } else {
        const uint16_t *k_row = k + page * a.cache.k_page + in_page * a.cache.k_row;
        v_at = page * a.cache.v_page + in_page * a.cache.v_row;
        float sum = 0.f;
        for (int c = 0; c < d; c += 8) {
          float x[8];
          load8<kFormat, kWide>(k_row + c, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(x[e], q_rows[warp][c + e], sum);
        }
        score = sum * scale_log2;
      }
    }
    float top = score;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float m_new = fmaxf(m, top), m_exp = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - m_exp), p = exp2f(score - m_exp);
    float sum = p;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    l = l * alpha + sum;
    m = m_new;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= alpha;
    const int count = min(32, visible - base);
    for (int j = 0; j < count; ++j) {
      const long long at = __shfl_sync(0xffffffffu, v_at, j);
      const float weight = __shfl_sync(0xffffffffu, p, j);
      if (at < 0 || 8 * lane >= d) continue;
      float x[8];
      load8<kFormat, kWide>(v + at + 8 * lane, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(weight, x[e], acc[e]);
    }
  }
  const float coefficient = l == 0.f && a.zero_fully_masked ? 0.f : 1.0f / l;
  uint16_t *out = static_cast<uint16_t *>(a.out) + token * a.out_token + head * a.out_head;
  if (8 * lane < d) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[8 * lane + e] = static_cast<uint16_t>(narrow_bits(acc[e] * coefficient, kFormat));
  }
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : m * 0.69314718055994530942f + logf(l);
}

}  // namespace

wb200_status launch_attention_paged_general(const AttentionPagedArgs &a, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.batch.tokens) * a.q_heads;
  const int64_t blocks = (rows + kRows - 1) / kRows;
  if (blocks > 0x7fffffff) return fail(WB200_ERR_LIMIT, "more than 2^33 rows in one paged attention launch");
  const uint64_t bits = reinterpret_cast<uintptr_t>(a.cache.k) | reinterpret_cast<uintptr_t>(a.cache.v) |
                        static_cast<uint64_t>((a.cache.k_page | a.cache.k_row | a.cache.k_head | a.cache.v_page | a.cache.v_row | a.cache.v_head) * 2);
  const bool wide = (bits & 15u) == 0, bf16 = a.cache.format == WB200_BF16;
  const auto kernel = wide ? (bf16 ? attention_paged_general_kernel<WB200_BF16, true> : attention_paged_general_kernel<WB200_F16, true>)
                           : (bf16 ? attention_paged_general_kernel<WB200_BF16, false> : attention_paged_general_kernel<WB200_F16, false>);
  WB200_CUDA_CHECK(launch_dependent(kernel, static_cast<unsigned>(blocks), kRows * 32, 0, stream, a));
  return WB200_OK;
}

}  // namespace wb200
