// K and V rows of a batch's tokens out of the pages of a cache, as they stand there (wb200_cache_read*): the inverse of the append.
// A row held in four bits is widened and rounded once to the cache's type.
//
// A thread keeps to its elements of the token's K and V heads, sixteen where they are codes, eight of 16 bits, and walks the block's
// tokens, four loads on their way together.
// Bound: HBM, the rows read and the rows written: 359545 keys of 8 heads, f16, 313 us for 1.9 GB, 6.0 TB/s.
#include "attention_paged.cuh"
#include "quantized_rows.cuh"

namespace wb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;
constexpr int kAtOnce = 4;

struct ReadParams {
  CacheReadArgs a;
  PagedCacheArgs cache;
  QuantizedRowsArgs rows;
  PagedBatchArgs batch;
  int tokens_per_block;
  int *refused;
};

// kWide: 16-byte accesses to every 16-bit row.
template <int kFormat, bool kQuantized, bool kWide>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ ReadParams p) {
  __shared__ int state_of[kMaxTokens], sequence_of[kMaxTokens];
  __shared__ int64_t rows_at[2][kMaxTokens], steps_at[2][kMaxTokens];        // of the token's row, of K and of V
  const int first = blockIdx.x * p.tokens_per_block, count = min(p.tokens_per_block, p.batch.tokens - first);
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < kMaxTokens) state_of[threadIdx.x] = 0;
  place_tokens(p.batch, p.cache, first, count, p.refused, sequence_of, [&](int t, int page, int row, int) {
    state_of[t] = 1;
    if constexpr (kQuantized) {
      rows_at[0][t] = page * p.rows.k.codes_page + row * p.rows.k.codes_row;
      rows_at[1][t] = page * p.rows.v.codes_page + row * p.rows.v.codes_row;
      steps_at[0][t] = page * p.rows.k.steps_page + row * p.rows.k.steps_row;
      steps_at[1][t] = page * p.rows.v.steps_page + row * p.rows.v.steps_row;
    } else {
      rows_at[0][t] = page * p.cache.k_page + row * p.cache.k_row;
      rows_at[1][t] = page * p.cache.v_page + row * p.cache.v_row;
    }
  });
  // Octets of elements to an item: of codes one of each half of the row, so that both are stored by lanes side by side.
  constexpr int kOctets = kQuantized ? 2 : 1;
  const int octets = (p.cache.head_dim + 7) / 8, chunks = (octets + kOctets - 1) / kOctets, items = 2 * p.cache.kv_heads * chunks;
#pragma unroll 1
  for (int item = threadIdx.x; item < items; item += kThreads) {
    const int row_head = item / chunks, chunk = item - row_head * chunks, e0 = 8 * chunk;
    const bool is_v = row_head >= p.cache.kv_heads;
    const int head = row_head - (is_v ? p.cache.kv_heads : 0);
    const int64_t to_token = is_v ? p.a.v_token : p.a.k_token;
    uint16_t *to = static_cast<uint16_t *>(is_v ? p.a.v : p.a.k) + head * (is_v ? p.a.v_head : p.a.k_head) + e0 + first * to_token;
    const int width = min(8, p.cache.head_dim - e0);
    const bool both = kOctets == 2 && chunk + chunks < octets;
    const QuantizedRows &r = is_v ? p.rows.v : p.rows.k;
    const uint8_t *const codes = kQuantized ? r.codes + head * r.codes_head + e0 / 2 : nullptr;
    const uint32_t *const steps = kQuantized ? r.steps + head * r.steps_head + chunk / (kQuantGroup / 8) : nullptr;
    const int next_step = (chunk + chunks) / (kQuantGroup / 8) - chunk / (kQuantGroup / 8);
    const uint16_t *const plain = static_cast<const uint16_t *>(is_v ? p.cache.v : p.cache.k) + head * (is_v ? p.cache.v_head : p.cache.k_head) + e0;
#pragma unroll 1
    for (int t0 = 0; t0 < count; t0 += kAtOnce) {
      uint32_t w[kAtOnce][4];                          // of codes two words and two pairs of steps
      bool live[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int t = t0 + u;
        live[u] = t < count && state_of[t];
        if (!live[u]) continue;
        if constexpr (kQuantized) {
          const uint32_t *const from = reinterpret_cast<const uint32_t *>(codes + rows_at[is_v][t]);
          w[u][0] = from[0];
          w[u][1] = steps[steps_at[is_v][t]];
          if (both) {
            w[u][2] = from[chunks];
            w[u][3] = steps[steps_at[is_v][t] + next_step];
          }
        } else {
          const uint16_t *const from = plain + rows_at[is_v][t];
          if constexpr (kWide) {
            *reinterpret_cast<uint4 *>(w[u]) = *reinterpret_cast<const uint4 *>(from);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[u][i] = (2 * i < width ? from[2 * i] : 0u) | ((2 * i + 1 < width ? static_cast<uint32_t>(from[2 * i + 1]) : 0u) << 16);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u, to += to_token) {
        if (!live[u]) continue;
#pragma unroll
        for (int o = 0; o < kOctets; ++o) {
          if (o > 0 && !both) continue;
          uint32_t out[4];
          if constexpr (kQuantized) {
            decode_word<kFormat == WB200_BF16>(w[u][2 * o], __byte_perm(w[u][2 * o + 1], 0u, 0x1010), __byte_perm(w[u][2 * o + 1], 0u, 0x3232), out);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = w[u][i];
          }
          uint16_t *const dst = to + 8 * chunks * o;
          if constexpr (kWide) {
            *reinterpret_cast<uint4 *>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (o > 0 || i < width) dst[i] = static_cast<uint16_t>(out[i >> 1] >> (16 * (i & 1)));
          }
        }
      }
    }
  }
}

}  // namespace

wb200_status launch_cache_read(const CacheReadArgs &a, const PagedCacheArgs &cache, const QuantizedRowsArgs *rows, const PagedBatchArgs &batch,
                               int *refused, cudaStream_t stream) {
  ReadParams p{};
  p.a = a;
  p.cache = cache;
  if (rows) p.rows = *rows;
  p.batch = batch;
  p.refused = refused;
  // Few tokens get a block each.
  p.tokens_per_block = kMaxTokens;
  while (p.tokens_per_block > 1 && batch.tokens / p.tokens_per_block < 148 * 8) p.tokens_per_block >>= 1;
  uint64_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | static_cast<uint64_t>((a.k_token | a.k_head | a.v_token | a.v_head) * 2) |
                  static_cast<uint64_t>(cache.head_dim * 2);
  if (!rows)
    bits |= reinterpret_cast<uintptr_t>(cache.k) | reinterpret_cast<uintptr_t>(cache.v) |
            static_cast<uint64_t>((cache.k_page | cache.k_row | cache.k_head | cache.v_page | cache.v_row | cache.v_head) * 2);
  const bool wide = (bits & 15u) == 0, bf16 = cache.format == WB200_BF16;
  void (*kernel)(const ReadParams);
  if (!rows) kernel = wide ? cache_read_kernel<WB200_BF16, false, true> : cache_read_kernel<WB200_BF16, false, false>;     // copies bits of either type
  else if (bf16) kernel = wide ? cache_read_kernel<WB200_BF16, true, true> : cache_read_kernel<WB200_BF16, true, false>;
  else kernel = wide ? cache_read_kernel<WB200_F16, true, true> : cache_read_kernel<WB200_F16, true, false>;
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(batch.tokens) + p.tokens_per_block - 1) / p.tokens_per_block);
  WB200_CUDA_CHECK(launch_dependent(kernel, blocks, kThreads, 0, stream, p));
  return WB200_OK;
}

}  // namespace wb200
