// Attention of chunks of new tokens over a paged KV cache held in four bits (head_dim 64 and 128): the kernel of
// attention_paged_chunk.cuh with K and V tiles decoded on the way into shared memory, and its launch. 4096 tokens behind 32768 cached
// ones, 32/8 heads, bf16: 2.36 ms, 0.99 PFLOP/s (the 16-bit cache 1.85); 8 chunks of 100 to 512 tokens 198 us.
#include "attention_paged_chunk.cuh"

namespace wb200 {

bool attention_quantized_chunk_supports(const AttentionPagedArgs &a, const QuantizedRowsArgs &rows) {
  return attention_quantized_rows_supports(a, rows) && a.q_heads / a.cache.kv_heads <= kTileM && a.batch.sequences <= kMaxSequences && tokens_outside_heads(a);
}

size_t attention_quantized_chunk_workspace(int sm_count) { return chunk_record_bytes(sm_count) + static_cast<size_t>(sm_count) * sizeof(ChunkSplit); }

wb200_status launch_attention_quantized_chunk(const AttentionPagedArgs &a, const QuantizedRowsArgs &rows, int sm_count, cudaStream_t stream) {
  QuantizedChunkParams p{};
  fill_chunk_params(&p, a, sm_count);
  p.rows = rows;
  CUtensorMap tq;
  wb200_status st = encode_queries(&tq, a, p);
  if (st != WB200_OK) return st;
  const bool bf16 = a.cache.format == WB200_BF16, wide = a.cache.head_dim == 128;
  const auto kernel = wide ? (bf16 ? attention_paged_chunk_kernel<true, 128, true> : attention_paged_chunk_kernel<false, 128, true>)
                           : (bf16 ? attention_paged_chunk_kernel<true, 64, true> : attention_paged_chunk_kernel<false, 64, true>);
  const auto fold = wide ? (bf16 ? attention_paged_chunk_fold_kernel<true, 128> : attention_paged_chunk_fold_kernel<false, 128>)
                         : (bf16 ? attention_paged_chunk_fold_kernel<true, 64> : attention_paged_chunk_fold_kernel<false, 64>);
  static PerDeviceOnce attributes;
  st = attributes.run([]() -> wb200_status {
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<true, 128, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<128>::kBytes)));
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<false, 128, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<128>::kBytes)));
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<true, 64, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<64>::kBytes)));
    WB200_CUDA_CHECK(cudaFuncSetAttribute(attention_paged_chunk_kernel<false, 64, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<64>::kBytes)));
    return WB200_OK;
  });
  if (st != WB200_OK) return st;
  WB200_CUDA_CHECK(launch_dependent(kernel, sm_count, kChunkThreads<true>, wide ? Shape<128>::kBytes : Shape<64>::kBytes, stream, tq, tq, tq, p));
  WB200_CUDA_CHECK(launch_dependent(fold, dim3(sm_count, a.cache.head_dim / kColumns), 2 * kTileM, 0, stream, static_cast<const ChunkParams &>(p)));
  return WB200_OK;
}

}  // namespace wb200
