// Attention of chunks of new tokens over a paged KV cache of bf16 or f16 (head_dim 64 and 128): the kernel of attention_paged_chunk.cuh
// with K and V tiles brought in by TMA, and its launch.
#include "attention_paged_chunk.cuh"

namespace wb200 {
namespace {

// The largest power of two that divides the page size, at most a tile.
int box_rows_of(int page_size) {
  int rows = 1;
  while (rows < kTileN && page_size % (2 * rows) == 0) rows *= 2;
  return rows;
}

// Extents and strides (in bytes) of the cache's tensor maps, innermost first: rows inside heads or heads inside rows, pages
// outside both, K and V alike; false for other orders. Strides of extents of one are free, but the map wants them to span
// what lies inside.
struct CacheMap {
  int rows_inside;
  uint64_t extents[4], strides[2][3];
};
bool make_cache_map(const PagedCacheArgs &c, CacheMap *m) {
  const int64_t strides[2][3] = {{c.k_row, c.k_head, c.k_page}, {c.v_row, c.v_head, c.v_page}};
  m->rows_inside = c.kv_heads > 1 && (c.page_size == 1 || c.k_row < c.k_head) ? 1 : 0;
  const int order[3] = {m->rows_inside ? 0 : 1, m->rows_inside ? 1 : 0, 2};
  const uint64_t extents[3] = {static_cast<uint64_t>(c.page_size), static_cast<uint64_t>(c.kv_heads), static_cast<uint64_t>(c.pages)};
  m->extents[0] = static_cast<uint64_t>(c.head_dim);
  for (int i = 0; i < 3; ++i) m->extents[i + 1] = extents[order[i]];
  for (int kind = 0; kind < 2; ++kind) {
    uint64_t span = m->extents[0] * 2;
    for (int i = 0; i < 3; ++i) {
      uint64_t stride = static_cast<uint64_t>(strides[kind][order[i]]) * 2;
      if (m->extents[i + 1] == 1) stride = span;
      if (stride < span) return false;
      m->strides[kind][i] = stride;
      span = stride * m->extents[i + 1];
    }
  }
  return true;
}

}  // namespace

bool attention_paged_chunk_supports(const AttentionPagedArgs &a) {
  const int group = a.q_heads / a.cache.kv_heads;
  if (!attention_paged_rows_supports(a) || group > kTileM || a.batch.sequences > kMaxSequences) return false;
  if (box_rows_of(a.cache.page_size) < 8) return false;      // a box covers whole 8-row groups of the swizzle
  CacheMap map;
  return make_cache_map(a.cache, &map) && tokens_outside_heads(a);
}

size_t attention_paged_chunk_workspace(int sm_count) { return chunk_record_bytes(sm_count) + static_cast<size_t>(sm_count) * sizeof(ChunkSplit); }

wb200_status launch_attention_paged_chunk(const AttentionPagedArgs &a, int sm_count, cudaStream_t stream) {
  ChunkParams p{};
  fill_chunk_params(&p, a, sm_count);
  p.box_rows = box_rows_of(a.cache.page_size);
  CUtensorMap tq, tk, tv;
  wb200_status st = encode_queries(&tq, a, p);
  if (st != WB200_OK) return st;
  CacheMap map;
  if (!make_cache_map(a.cache, &map)) return fail(WB200_ERR_UNSUPPORTED, "paged cache outside the chunk kernel's domain");
  p.rows_inside = map.rows_inside;
  const uint32_t box = static_cast<uint32_t>(p.box_rows);
  for (int kind = 0; kind < 2; ++kind) {
    st = encode_tmap_strided(kind ? &tv : &tk, kind ? a.cache.v : a.cache.k, a.cache.format, 4, map.extents, map.strides[kind],
                             {64, map.rows_inside ? box : 1u, map.rows_inside ? 1u : box, 1});
    if (st != WB200_OK) return st;
  }
  const bool bf16 = a.cache.format == WB200_BF16, wide = a.cache.head_dim == 128;
  const auto kernel = wide ? (bf16 ? attention_paged_chunk_kernel<true, 128, false> : attention_paged_chunk_kernel<false, 128, false>)
                           : (bf16 ? attention_paged_chunk_kernel<true, 64, false> : attention_paged_chunk_kernel<false, 64, false>);
  const auto fold = wide ? (bf16 ? attention_paged_chunk_fold_kernel<true, 128> : attention_paged_chunk_fold_kernel<false, 128>)
                         : (bf16 ? attention_paged_chunk_fold_kernel<true, 64> : attention_paged_chunk_fold_kernel<false, 64>);
  static PerDeviceOnce attributes;
  st = attributes.run([]() -> wb200_status {
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<true, 128, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<128>::kBytes)));
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<false, 128, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<128>::kBytes)));
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<true, 64, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<64>::kBytes)));
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<false, 64, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<64>::kBytes)));
    return WB200_OK;
  });
  if (st != WB200_OK) return st;
  WB200_CUDA_CHECK(launch_dependent(kernel, sm_count, kChunkThreads<false>, wide ? Shape<128>::kBytes : Shape<64>::kBytes, stream, tq, tk, tv, p));
  WB200_CUDA_CHECK(launch_dependent(fold, dim3(sm_count, a.cache.head_dim / kColumns), 2 * kTileM, 0, stream, p));
  return WB200_OK;
}

}  // namespace wb200
