// Entry points of serving from a paged KV cache: rotary positions, cache writes, attention over the pages, and the pages
// themselves. Device buffers only; arguments are checked here, device data by the kernels.
#include "backend.h"

using namespace wb200;

namespace wb200 {
const char *refused_data_message(int code) {
  switch (code) {
    case kRefusedPage: return "a paged-cache kernel left out a page number outside the cache";
    case kRefusedLength: return "a paged-cache kernel left out a length, token range or position outside the page table or the buffers";
    case kRefusedSequence: return "a paged-cache kernel left out a sequence index outside the page table";
    case kRefusedReference: return "a page was freed more often than it is held";
    default: return "a paged-cache kernel found device data outside its buffers";
  }
}
}  // namespace wb200

namespace {

// Addresses of elements of `bytes` bytes; null counts. The kernels load and store whole elements.
template <typename... Pointers>
bool on_elements(uint32_t bytes, const Pointers *...pointers) {
  return ((reinterpret_cast<uintptr_t>(pointers) | ... | 0u) & (bytes - 1)) == 0;
}
wb200_status off_elements() { return fail(WB200_ERR_INVALID_ARGUMENT, "device arrays must be aligned to their elements"); }

wb200_status make_rotary_constants(const wb200_rope_table &t, uint32_t head_dim, RotaryConstants *c) {
  if (t.rotary_dim % 2 != 0 || t.rotary_dim > head_dim || t.rotary_dim > 2 * kMaxRotaryPairs)
    return fail(WB200_ERR_INVALID_ARGUMENT, "rotary_dim must be even and at most head_dim and 512");
  if (t.rotary_dim != 0 && !t.turns) return fail(WB200_ERR_INVALID_ARGUMENT, "the rotary table's turns must not be null");
  c->pairs = static_cast<int>(t.rotary_dim / 2);
  c->magnitude = t.magnitude;
  for (int i = 0; i < kMaxRotaryPairs; ++i) c->turns[i] = i < c->pairs ? t.turns[i] : 0;
  return WB200_OK;
}

// Rows (page, row, head) of head_dim elements that do not overlap: strides sorted, each spans what lies inside it.
bool rows_apart(int64_t head_dim, const int64_t (&stride)[3], const int64_t (&extent)[3]) {
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (stride[order[j]] > stride[order[j + 1]]) { const int t = order[j]; order[j] = order[j + 1]; order[j + 1] = t; }
  int64_t span = head_dim;
  for (int i : order) {
    if (extent[i] == 1) continue;
    if (stride[i] < span) return false;
    span += (extent[i] - 1) * stride[i];
  }
  return true;
}

wb200_status make_cache(const wb200_paged_cache *c, bool f32_too, PagedCacheArgs *a) {
  if (c->format != WB200_BF16 && c->format != WB200_F16 && !(f32_too && c->format == WB200_F32))
    return fail(WB200_ERR_UNSUPPORTED, "a paged cache holds bf16 or f16");
  if (c->pages == 0 || c->page_size == 0 || c->kv_heads == 0 || c->head_dim == 0)
    return fail(WB200_ERR_INVALID_ARGUMENT, "paged cache extents must be positive");
  if (c->pages > 0x7fffffffu || c->page_size > 0x7fffffffu || c->kv_heads > 0xffffu || c->head_dim > 0xffffu)
    return fail(WB200_ERR_LIMIT, "paged cache extents too large");
  if (!c->k || !c->v) return fail(WB200_ERR_INVALID_ARGUMENT, "k and v of the paged cache must not be null");
  if (!on_elements(c->format == WB200_F32 ? 4 : 2, c->k, c->v)) return off_elements();
  const int64_t extent[3] = {c->pages, c->page_size, c->kv_heads};
  if (!rows_apart(c->head_dim, {c->k_page_stride, c->k_row_stride, c->k_head_stride}, extent) ||
      !rows_apart(c->head_dim, {c->v_page_stride, c->v_row_stride, c->v_head_stride}, extent))
    return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the paged cache overlap");
  a->pages = static_cast<int>(c->pages); a->page_size = static_cast<int>(c->page_size);
  a->kv_heads = static_cast<int>(c->kv_heads); a->head_dim = static_cast<int>(c->head_dim); a->format = static_cast<int>(c->format);
  a->k = c->k; a->v = c->v;
  a->k_page = c->k_page_stride; a->k_row = c->k_row_stride; a->k_head = c->k_head_stride;
  a->v_page = c->v_page_stride; a->v_row = c->v_row_stride; a->v_head = c->v_head_stride;
  return WB200_OK;
}

// A cache held in four bits: its extents and where its rows lie.
wb200_status make_quantized(const wb200_quantized_cache *c, PagedCacheArgs *a, QuantizedRowsArgs *rows) {
  if (c->format != WB200_BF16 && c->format != WB200_F16) return fail(WB200_ERR_UNSUPPORTED, "a quantized cache stands for bf16 or f16");
  if (c->bits != 4) return fail(WB200_ERR_UNSUPPORTED, "a quantized cache holds codes of 4 bits");
  if (c->pages == 0 || c->page_size == 0 || c->kv_heads == 0 || c->head_dim == 0)
    return fail(WB200_ERR_INVALID_ARGUMENT, "paged cache extents must be positive");
  if (c->head_dim % 8 != 0 || c->head_dim > static_cast<uint32_t>(kQuantMaxHeadDim))
    return fail(WB200_ERR_UNSUPPORTED, "a quantized cache takes head dimensions that are multiples of 8, up to 256");
  if (c->pages > 0x7fffffffu || c->page_size > 0x7fffffffu || c->kv_heads > 0xffffu) return fail(WB200_ERR_LIMIT, "paged cache extents too large");
  *a = PagedCacheArgs{};
  a->pages = static_cast<int>(c->pages); a->page_size = static_cast<int>(c->page_size);
  a->kv_heads = static_cast<int>(c->kv_heads); a->head_dim = static_cast<int>(c->head_dim); a->format = static_cast<int>(c->format);
  const int64_t extent[3] = {c->pages, c->page_size, c->kv_heads};
  const int64_t groups = (c->head_dim + kQuantGroup - 1) / kQuantGroup;
  const wb200_quantized_rows *from[2] = {&c->k, &c->v};
  QuantizedRows *to[2] = {&rows->k, &rows->v};
  for (int i = 0; i < 2; ++i) {
    const wb200_quantized_rows &r = *from[i];
    if (!r.codes || !r.steps) return fail(WB200_ERR_INVALID_ARGUMENT, "codes and steps of the quantized cache must not be null");
    if (!on_elements(4, r.codes, r.steps) || ((r.codes_page_stride | r.codes_row_stride | r.codes_head_stride) & 3) != 0)
      return fail(WB200_ERR_INVALID_ARGUMENT, "rows of codes and pairs of steps must begin on 4 bytes");
    if (!rows_apart(c->head_dim / 2, {r.codes_page_stride, r.codes_row_stride, r.codes_head_stride}, extent) ||
        !rows_apart(groups, {r.steps_page_stride, r.steps_row_stride, r.steps_head_stride}, extent))
      return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the quantized cache overlap");
    *to[i] = {static_cast<uint8_t *>(r.codes), static_cast<uint32_t *>(r.steps), r.codes_page_stride, r.codes_row_stride, r.codes_head_stride,
              r.steps_page_stride, r.steps_row_stride, r.steps_head_stride};
  }
  return WB200_OK;
}

wb200_status make_batch(const wb200_paged_batch *b, const PagedCacheArgs &c, PagedBatchArgs *a) {
  if (b->sequences > 0x7ffffffeu || b->tokens > 0x7fffffffu || b->table_width > 0x7fffffffu || b->max_query > 0x7fffffffu)
    return fail(WB200_ERR_LIMIT, "paged batch extents too large");
  if (static_cast<uint64_t>(b->table_width) * static_cast<uint64_t>(c.page_size) > (1ull << 30))
    return fail(WB200_ERR_LIMIT, "a row of the page table covers more than 2^30 tokens");
  if (b->sequences != 0 && b->tokens != 0) {
    if (!b->key_lengths || !b->query_starts || (b->table_width != 0 && !b->page_table))
      return fail(WB200_ERR_INVALID_ARGUMENT, "page_table, key_lengths and query_starts must not be null");
    if (b->sequences > 1 && b->table_stride < static_cast<int64_t>(b->table_width))
      return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the page table overlap");
    if (!on_elements(4, b->page_table, b->key_lengths, b->query_starts)) return off_elements();
  }
  a->sequences = static_cast<int>(b->sequences); a->table_width = static_cast<int>(b->table_width);
  a->tokens = static_cast<int>(b->tokens); a->max_query = static_cast<int>(b->max_query);
  a->page_table = b->page_table; a->key_lengths = b->key_lengths; a->query_starts = b->query_starts; a->table_stride = b->table_stride;
  a->least_count = 0; a->most_count = 0x7fffffff;
  return WB200_OK;
}

// Rows (token, head) that do not overlap, in an array that is written.
bool output_rows_apart(int64_t head_dim, int64_t token_stride, int64_t head_stride, int64_t tokens, int64_t heads) {
  return rows_apart(head_dim, {token_stride, head_stride, 1}, {tokens, heads, 1});
}

// `a->cache` is made already.
wb200_status make_attention(wb200_backend *backend, const wb200_paged_batch *batch, const wb200_attention_paged_params *p, AttentionPagedArgs *a) {
  wb200_status st = make_batch(batch, a->cache, &a->batch);
  if (st != WB200_OK) return st;
  if (p->q_heads == 0 || p->q_heads > 0xffffu || p->q_heads % static_cast<uint32_t>(a->cache.kv_heads) != 0)
    return fail(WB200_ERR_INVALID_ARGUMENT, "q_heads must be a positive multiple of kv_heads");
  if (a->cache.head_dim % 8 != 0 || a->cache.head_dim > 256) return fail(WB200_ERR_UNSUPPORTED, "paged attention takes head dimensions that are multiples of 8, up to 256");
  if (static_cast<uint64_t>(batch->tokens) * p->q_heads > 0x7fffffffull) return fail(WB200_ERR_LIMIT, "more than 2^31 - 1 rows in one paged attention");
  if (!(p->scale > 0.f) || !(p->scale <= 1e38f)) return fail(WB200_ERR_INVALID_ARGUMENT, "scale must be positive and at most 1e38");
  a->q_heads = static_cast<int>(p->q_heads);
  a->causal = p->causal ? 1 : 0;
  a->zero_fully_masked = p->zero_fully_masked ? 1 : 0;
  a->scale = p->scale;
  a->q = p->q; a->out = p->out; a->lse = p->lse;
  a->q_token = p->q_token_stride; a->q_head = p->q_head_stride; a->out_token = p->out_token_stride; a->out_head = p->out_head_stride;
  a->workspace = p->workspace;
  a->refused = backend ? backend->d_status + 2 : nullptr;
  a->status = backend ? backend->d_status : nullptr;
  return WB200_OK;
}

wb200_status make_attention_paged(wb200_backend *backend, const wb200_paged_cache *cache, const wb200_paged_batch *batch,
                                  const wb200_attention_paged_params *p, AttentionPagedArgs *a) {
  const wb200_status st = make_cache(cache, false, &a->cache);
  return st != WB200_OK ? st : make_attention(backend, batch, p, a);
}
wb200_status make_attention_quantized(wb200_backend *backend, const wb200_quantized_cache *cache, const wb200_paged_batch *batch,
                                      const wb200_attention_paged_params *p, AttentionPagedArgs *a, QuantizedRowsArgs *rows) {
  const wb200_status st = make_quantized(cache, &a->cache, rows);
  return st != WB200_OK ? st : make_attention(backend, batch, p, a);
}

// Which kernel a call takes, from what the host knows: sizes, alignment and the caller's word on the longest chunk. Any choice
// is right for any lengths. Where a sequence has at most kRowsAtMost packed rows (one tile of its MMA) the rows kernel streams
// the keys, which HBM bounds; a row tile of the chunk kernel takes as long for one row as for 128.
constexpr int kRowsAtMost = 16;
enum class PagedKernel { general, rows, chunk, dealt };
// The most packed rows of one sequence.
int64_t most_rows(const AttentionPagedArgs &a) {
  int64_t longest = a.batch.max_query > 0 ? a.batch.max_query : (a.batch.tokens <= a.batch.sequences ? 1 : a.batch.tokens);
  if (longest > a.batch.tokens) longest = a.batch.tokens;
  return longest * (a.q_heads / a.cache.kv_heads);
}
PagedKernel choose_attention_paged(const AttentionPagedArgs &a) {
  if (!attention_paged_rows_supports(a)) return PagedKernel::general;
  return most_rows(a) > kRowsAtMost && attention_paged_chunk_supports(a) ? PagedKernel::chunk : PagedKernel::rows;
}
uint64_t aligned256(uint64_t bytes) { return (bytes + 255) & ~255ull; }
PagedKernel choose_attention_quantized(const AttentionPagedArgs &a, const QuantizedRowsArgs &rows) {
  if (!attention_quantized_rows_supports(a, rows)) return PagedKernel::general;
  // Two tiles of 16 rows a sequence, which read its keys twice, still are the shorter at head_dim 64: 17 sequences of 5000 keys, 4 KV
  // heads, 32 rows 32 us and 36 us, 48 rows 41 and 36; at head_dim 128, 8 KV heads, 20 rows 81 and 81.
  const int64_t at_most = a.cache.head_dim == 64 ? 2 * kRowsAtMost : kRowsAtMost;
  if (most_rows(a) <= at_most || !attention_quantized_chunk_supports(a, rows)) return PagedKernel::rows;
  // Sequences of one token among chunks, of which there are many where the tokens are few for the longest chunk, go to the rows kernel:
  // a row tile of the chunk kernel takes 1.7 us for 128 keys whether it holds one token or 32, three times as long as the keys' bytes.
  const bool mixed = a.batch.max_query > 1 && 2ll * a.batch.tokens <= static_cast<int64_t>(a.batch.sequences) * a.batch.max_query;
  return mixed && a.q_heads / a.cache.kv_heads <= kRowsAtMost ? PagedKernel::dealt : PagedKernel::chunk;
}
uint64_t attention_quantized_workspace(PagedKernel kernel, int sm_count) {
  if (kernel == PagedKernel::general) return 0;
  const uint64_t rows = aligned256(attention_quantized_rows_workspace(sm_count)), chunk = attention_quantized_chunk_workspace(sm_count);
  return kernel == PagedKernel::rows ? rows : kernel == PagedKernel::chunk ? chunk : rows + chunk;
}
// The single tokens' part of the workspace in front of the chunks'.
wb200_status launch_attention_quantized_dealt(AttentionPagedArgs a, const QuantizedRowsArgs &rows, int sm_count, cudaStream_t stream) {
  AttentionPagedArgs single = a;
  single.batch.max_query = single.batch.most_count = 1;
  a.batch.least_count = 2;
  a.workspace = static_cast<uint8_t *>(a.workspace) + aligned256(attention_quantized_rows_workspace(sm_count));
  const wb200_status st = launch_attention_quantized_rows(single, rows, sm_count, stream);
  return st != WB200_OK ? st : launch_attention_quantized_chunk(a, rows, sm_count, stream);
}
uint64_t attention_paged_workspace(PagedKernel kernel, int sm_count) {
  if (kernel == PagedKernel::general) return 0;
  return kernel == PagedKernel::rows ? attention_paged_rows_workspace(sm_count) : attention_paged_chunk_workspace(sm_count);
}

wb200_status make_page_tables(wb200_backend *backend, const wb200_page_tables *t, bool lengths_out, PageTablesArgs *a) {
  if (!backend || !t) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  if (t->sequences == 0 || t->table_width == 0 || t->pages == 0 || t->page_size == 0)
    return fail(WB200_ERR_INVALID_ARGUMENT, "page table extents must be positive");
  if (t->sequences > static_cast<uint32_t>(kMaxPagedSequences)) return fail(WB200_ERR_LIMIT, "more than 16384 sequences in one page table");
  if (t->pages > 0x7fffffffu || t->page_size > 0x7fffffffu || static_cast<uint64_t>(t->sequences) * t->table_width > (1ull << 30) ||
      static_cast<uint64_t>(t->table_width) * t->page_size > (1ull << 30))
    return fail(WB200_ERR_LIMIT, "page table extents too large");
  if (!t->table || !t->lengths || !t->refs || !t->table_out || !t->refs_out || (lengths_out && !t->lengths_out))
    return fail(WB200_ERR_INVALID_ARGUMENT, "page table, lengths and refs must not be null");
  if (!on_elements(4, t->table, t->lengths, t->refs, t->table_out, t->lengths_out, t->refs_out)) return off_elements();
  if (t->sequences > 1 && (t->table_stride < static_cast<int64_t>(t->table_width) || t->table_out_stride < static_cast<int64_t>(t->table_width)))
    return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the page table overlap");
  if (t->table == t->table_out && t->sequences > 1 && t->table_stride != t->table_out_stride)
    return fail(WB200_ERR_INVALID_ARGUMENT, "a page table written in place keeps its stride");
  a->sequences = static_cast<int>(t->sequences); a->table_width = static_cast<int>(t->table_width);
  a->pages = static_cast<int>(t->pages); a->page_size = static_cast<int>(t->page_size);
  a->table = t->table; a->lengths = t->lengths; a->refs = t->refs;
  a->table_out = t->table_out; a->lengths_out = t->lengths_out; a->refs_out = t->refs_out;
  a->table_stride = t->table_stride; a->table_out_stride = t->table_out_stride;
  a->refused = backend->d_status + 2;
  return WB200_OK;
}

// The append onto either kind of cache, whose extents are in `c`; `rows` null: the 16-bit one.
wb200_status rope_append(wb200_backend *backend, const PagedCacheArgs &c, const QuantizedRowsArgs *rows, const wb200_paged_batch *batch,
                         const wb200_rope_append_params *p) {
  PagedBatchArgs b;
  RotaryConstants constants;
  wb200_status st = make_batch(batch, c, &b);
  if (st != WB200_OK) return st;
  const uint32_t kv_heads = static_cast<uint32_t>(c.kv_heads), head_dim = static_cast<uint32_t>(c.head_dim);
  if ((st = make_rotary_constants(p->table, head_dim, &constants)) != WB200_OK) return st;
  if (p->q_heads > 0xffffu || (static_cast<uint64_t>(p->q_heads) + 2ull * kv_heads) * head_dim > (1u << 24))
    return fail(WB200_ERR_LIMIT, "rope extents too large");
  if (p->positions && p->position_bytes != 4 && p->position_bytes != 8) return fail(WB200_ERR_INVALID_ARGUMENT, "positions are int32 or int64");
  if (b.tokens == 0 || b.sequences == 0) return WB200_OK;
  if (!p->qkv || (p->q_heads != 0 && !p->q)) return fail(WB200_ERR_INVALID_ARGUMENT, "qkv and q must not be null");
  if (!on_elements(2, p->qkv, p->q) || (p->positions && !on_elements(p->position_bytes, p->positions))) return off_elements();
  if (p->q_heads != 0 && !output_rows_apart(head_dim, p->q_token_stride, p->q_head_stride, b.tokens, p->q_heads))
    return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the output overlap");
  RopeArgs a{};
  a.tokens = b.tokens; a.heads = static_cast<int>(p->q_heads) + 2 * c.kv_heads; a.head_dim = c.head_dim; a.format = c.format;
  a.interleaved = p->interleaved ? 1 : 0; a.position_bytes = p->position_bytes;
  a.positions = p->positions; a.x = p->qkv; a.out = p->q;
  a.x_token = p->qkv_token_stride; a.x_head = c.head_dim; a.out_token = p->q_token_stride; a.out_head = p->q_head_stride;
  DeviceGuard guard(backend->device);
  const cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  st = rows ? launch_rope_append_quantized(a, constants, c, *rows, b, backend->d_status + 2, stream)
            : launch_rope_append(a, constants, c, b, backend->d_status + 2, stream);
  if (st == WB200_OK) backend->launches += 1;
  return st;
}

wb200_status cache_read(wb200_backend *backend, const PagedCacheArgs &c, const QuantizedRowsArgs *rows, const wb200_paged_batch *batch,
                        const wb200_cache_read_params *p) {
  PagedBatchArgs b;
  wb200_status st = make_batch(batch, c, &b);
  if (st != WB200_OK) return st;
  if (static_cast<uint64_t>(c.kv_heads) * static_cast<uint64_t>(c.head_dim) > (1u << 23)) return fail(WB200_ERR_LIMIT, "rows of one token too large");
  if (b.tokens == 0 || b.sequences == 0) return WB200_OK;
  if (!p->k || !p->v) return fail(WB200_ERR_INVALID_ARGUMENT, "k and v must not be null");
  if (!on_elements(2, p->k, p->v)) return off_elements();
  if (!output_rows_apart(c.head_dim, p->k_token_stride, p->k_head_stride, b.tokens, c.kv_heads) ||
      !output_rows_apart(c.head_dim, p->v_token_stride, p->v_head_stride, b.tokens, c.kv_heads))
    return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the output overlap");
  DeviceGuard guard(backend->device);
  st = launch_cache_read({p->k, p->v, p->k_token_stride, p->k_head_stride, p->v_token_stride, p->v_head_stride}, c, rows, b, backend->d_status + 2,
                         static_cast<cudaStream_t>(p->stream));
  if (st == WB200_OK) backend->launches += 1;
  return st;
}

// What attention needs beside its sizes, checked before any kernel is chosen; `done`: there is nothing to do.
wb200_status check_attention_buffers(const AttentionPagedArgs &a, bool *done) {
  *done = a.batch.tokens == 0 || a.batch.sequences == 0;
  if (*done) return WB200_OK;
  if (!a.q || !a.out) return fail(WB200_ERR_INVALID_ARGUMENT, "q and out must not be null");
  if (!on_elements(2, a.q, a.out) || !on_elements(4, a.lse)) return off_elements();
  if (!output_rows_apart(a.cache.head_dim, a.out_token, a.out_head, a.batch.tokens, a.q_heads))
    return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the output overlap");
  return WB200_OK;
}
wb200_status check_workspace(const wb200_attention_paged_params *p, uint64_t needed, const char *query) {
  if (needed > 0 && (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) || p->workspace_bytes < needed))
    return fail(WB200_ERR_INVALID_ARGUMENT, std::string("the workspace must be 256-byte aligned and hold ") + query + "() bytes");
  return WB200_OK;
}

}  // namespace

extern "C" {

wb200_status wb200_rope(wb200_backend *backend, const wb200_rope_params *p) {
  if (!backend || !p) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  if (!is_float_format(p->format)) return fail(WB200_ERR_UNSUPPORTED, "rope takes bf16, f16 or f32 storage");
  if (p->heads == 0 || p->head_dim == 0) return fail(WB200_ERR_INVALID_ARGUMENT, "heads and head_dim must be positive");
  if (p->tokens > 0x7fffffffu || p->heads > 0xffffu || p->head_dim > 0xffffu || static_cast<uint64_t>(p->heads) * p->head_dim > (1u << 24))
    return fail(WB200_ERR_LIMIT, "rope extents too large");
  if (p->position_bytes != 4 && p->position_bytes != 8) return fail(WB200_ERR_INVALID_ARGUMENT, "positions are int32 or int64");
  RotaryConstants c;
  wb200_status st = make_rotary_constants(p->table, p->head_dim, &c);
  if (st != WB200_OK) return st;
  if (p->tokens == 0) return WB200_OK;
  if (!p->x || !p->out || !p->positions) return fail(WB200_ERR_INVALID_ARGUMENT, "x, out and positions must not be null");
  if (!on_elements(p->format == WB200_F32 ? 4 : 2, p->x, p->out) || !on_elements(p->position_bytes, p->positions)) return off_elements();
  if (!output_rows_apart(p->head_dim, p->out_token_stride, p->out_head_stride, p->tokens, p->heads))
    return fail(WB200_ERR_INVALID_ARGUMENT, "rows of the output overlap");
  if (p->x == p->out && ((p->tokens > 1 && p->x_token_stride != p->out_token_stride) || (p->heads > 1 && p->x_head_stride != p->out_head_stride)))
    return fail(WB200_ERR_INVALID_ARGUMENT, "rope in place keeps the strides");
  RopeArgs a{};
  a.tokens = static_cast<int>(p->tokens); a.heads = static_cast<int>(p->heads); a.head_dim = static_cast<int>(p->head_dim); a.format = p->format;
  a.interleaved = p->interleaved ? 1 : 0; a.backward = p->backward ? 1 : 0; a.position_bytes = p->position_bytes;
  a.positions = p->positions; a.x = p->x; a.out = p->out;
  a.x_token = p->x_token_stride; a.x_head = p->x_head_stride; a.out_token = p->out_token_stride; a.out_head = p->out_head_stride;
  DeviceGuard guard(backend->device);
  st = launch_rope(a, c, static_cast<cudaStream_t>(p->stream));
  if (st == WB200_OK) backend->launches += 1;
  return st;
}

wb200_status wb200_rope_append(wb200_backend *backend, const wb200_paged_cache *cache, const wb200_paged_batch *batch,
                               const wb200_rope_append_params *p) {
  if (!backend || !cache || !batch || !p) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  PagedCacheArgs c;
  const wb200_status st = make_cache(cache, false, &c);
  return st != WB200_OK ? st : rope_append(backend, c, nullptr, batch, p);
}

wb200_status wb200_rope_append_quantized(wb200_backend *backend, const wb200_quantized_cache *cache, const wb200_paged_batch *batch,
                                         const wb200_rope_append_params *p) {
  if (!backend || !cache || !batch || !p) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  PagedCacheArgs c;
  QuantizedRowsArgs rows;
  const wb200_status st = make_quantized(cache, &c, &rows);
  return st != WB200_OK ? st : rope_append(backend, c, &rows, batch, p);
}

wb200_status wb200_cache_read(wb200_backend *backend, const wb200_paged_cache *cache, const wb200_paged_batch *batch, const wb200_cache_read_params *p) {
  if (!backend || !cache || !batch || !p) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  PagedCacheArgs c;
  const wb200_status st = make_cache(cache, false, &c);
  return st != WB200_OK ? st : cache_read(backend, c, nullptr, batch, p);
}

wb200_status wb200_cache_read_quantized(wb200_backend *backend, const wb200_quantized_cache *cache, const wb200_paged_batch *batch,
                                        const wb200_cache_read_params *p) {
  if (!backend || !cache || !batch || !p) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  PagedCacheArgs c;
  QuantizedRowsArgs rows;
  const wb200_status st = make_quantized(cache, &c, &rows);
  return st != WB200_OK ? st : cache_read(backend, c, &rows, batch, p);
}

uint64_t wb200_attention_paged_workspace_bytes(const wb200_backend *backend, const wb200_paged_cache *cache, const wb200_paged_batch *batch,
                                               const wb200_attention_paged_params *p) {
  if (!backend) { fail(WB200_ERR_INVALID_ARGUMENT, "null argument"); return 0; }
  if (!cache && !batch && !p) {
    const uint64_t rows = attention_paged_rows_workspace(backend->sm_count), chunk = attention_paged_chunk_workspace(backend->sm_count);
    return rows > chunk ? rows : chunk;
  }
  if (!cache || !batch || !p) { fail(WB200_ERR_INVALID_ARGUMENT, "null argument"); return 0; }
  AttentionPagedArgs a{};
  if (make_attention_paged(nullptr, cache, batch, p, &a) != WB200_OK) return 0;
  return attention_paged_workspace(choose_attention_paged(a), backend->sm_count);
}

wb200_status wb200_attention_paged(wb200_backend *backend, const wb200_paged_cache *cache, const wb200_paged_batch *batch,
                                   const wb200_attention_paged_params *p) {
  if (!backend || !cache || !batch || !p) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  AttentionPagedArgs a{};
  wb200_status st = make_attention_paged(backend, cache, batch, p, &a);
  if (st != WB200_OK) return st;
  bool done;
  if ((st = check_attention_buffers(a, &done)) != WB200_OK || done) return st;
  const PagedKernel kernel = choose_attention_paged(a);
  if ((st = check_workspace(p, attention_paged_workspace(kernel, backend->sm_count), "wb200_attention_paged_workspace_bytes")) != WB200_OK) return st;
  DeviceGuard guard(backend->device);
  const cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  if (kernel == PagedKernel::general) st = launch_attention_paged_general(a, stream);
  else if (kernel == PagedKernel::rows) st = launch_attention_paged_rows(a, backend->sm_count, stream);
  else st = launch_attention_paged_chunk(a, backend->sm_count, stream);
  const bool one = kernel == PagedKernel::general || (kernel == PagedKernel::rows && attention_paged_rows_clustered(a, backend->sm_count));
  if (st == WB200_OK) backend->launches += one ? 1 : 2;
  return st;
}

uint64_t wb200_attention_quantized_workspace_bytes(const wb200_backend *backend, const wb200_quantized_cache *cache, const wb200_paged_batch *batch,
                                                   const wb200_attention_paged_params *p) {
  if (!backend) { fail(WB200_ERR_INVALID_ARGUMENT, "null argument"); return 0; }
  if (!cache && !batch && !p) return attention_quantized_workspace(PagedKernel::dealt, backend->sm_count);
  if (!cache || !batch || !p) { fail(WB200_ERR_INVALID_ARGUMENT, "null argument"); return 0; }
  AttentionPagedArgs a{};
  QuantizedRowsArgs rows;
  if (make_attention_quantized(nullptr, cache, batch, p, &a, &rows) != WB200_OK) return 0;
  return attention_quantized_workspace(choose_attention_quantized(a, rows), backend->sm_count);
}

wb200_status wb200_attention_quantized(wb200_backend *backend, const wb200_quantized_cache *cache, const wb200_paged_batch *batch,
                                       const wb200_attention_paged_params *p) {
  if (!backend || !cache || !batch || !p) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  AttentionPagedArgs a{};
  QuantizedRowsArgs rows;
  wb200_status st = make_attention_quantized(backend, cache, batch, p, &a, &rows);
  if (st != WB200_OK) return st;
  bool done;
  if ((st = check_attention_buffers(a, &done)) != WB200_OK || done) return st;
  const PagedKernel kernel = choose_attention_quantized(a, rows);
  if ((st = check_workspace(p, attention_quantized_workspace(kernel, backend->sm_count), "wb200_attention_quantized_workspace_bytes")) != WB200_OK) return st;
  DeviceGuard guard(backend->device);
  const cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  if (kernel == PagedKernel::general) st = launch_attention_quantized_general(a, rows, stream);
  else if (kernel == PagedKernel::rows) st = launch_attention_quantized_rows(a, rows, backend->sm_count, stream);
  else if (kernel == PagedKernel::chunk) st = launch_attention_quantized_chunk(a, rows, backend->sm_count, stream);
  else st = launch_attention_quantized_dealt(a, rows, backend->sm_count, stream);
  if (st != WB200_OK) return st;
  if (kernel == PagedKernel::rows || kernel == PagedKernel::dealt) backend->launches += attention_quantized_rows_clustered(a, backend->sm_count) ? 1 : 2;
  if (kernel == PagedKernel::chunk || kernel == PagedKernel::dealt) backend->launches += 2;
  if (kernel == PagedKernel::general) backend->launches += 1;
  return st;
}

wb200_status wb200_pages_reserve(wb200_backend *backend, const wb200_page_tables *tables, const int32_t *wanted, int32_t *result) {
  PageTablesArgs a;
  wb200_status st = make_page_tables(backend, tables, true, &a);
  if (st != WB200_OK) return st;
  if (!wanted || !result) return fail(WB200_ERR_INVALID_ARGUMENT, "wanted and result must not be null");
  if (!on_elements(4, wanted, result)) return off_elements();
  DeviceGuard guard(backend->device);
  if ((st = launch_pages_reserve(a, wanted, result, static_cast<cudaStream_t>(tables->stream))) == WB200_OK) backend->launches += 1;
  return st;
}

wb200_status wb200_pages_fork(wb200_backend *backend, const wb200_page_tables *tables, uint32_t count, const int32_t *parents,
                              const int32_t *children, int32_t *sources, int32_t *destinations, int32_t *result) {
  PageTablesArgs a;
  wb200_status st = make_page_tables(backend, tables, true, &a);
  if (st != WB200_OK) return st;
  if (count > tables->sequences) return fail(WB200_ERR_INVALID_ARGUMENT, "more forks than sequences");
  if (!result || (count != 0 && (!parents || !children || !sources || !destinations)))
    return fail(WB200_ERR_INVALID_ARGUMENT, "parents, children, sources, destinations and result must not be null");
  if (!on_elements(4, parents, children, sources, destinations, result)) return off_elements();
  DeviceGuard guard(backend->device);
  st = launch_pages_fork(a, static_cast<int>(count), parents, children, sources, destinations, result, static_cast<cudaStream_t>(tables->stream));
  if (st == WB200_OK) backend->launches += 1;
  return st;
}

wb200_status wb200_pages_free(wb200_backend *backend, const wb200_page_tables *tables, uint32_t count, const int32_t *sequences) {
  PageTablesArgs a;
  wb200_status st = make_page_tables(backend, tables, true, &a);
  if (st != WB200_OK) return st;
  if (count > (1u << 30)) return fail(WB200_ERR_LIMIT, "more than 2^30 sequences to free");
  if (count != 0 && !sequences) return fail(WB200_ERR_INVALID_ARGUMENT, "sequences must not be null");
  if (!on_elements(4, sequences)) return off_elements();
  DeviceGuard guard(backend->device);
  if ((st = launch_pages_free(a, static_cast<int>(count), sequences, static_cast<cudaStream_t>(tables->stream))) == WB200_OK) backend->launches += 1;
  return st;
}

wb200_status wb200_pages_compact(wb200_backend *backend, const wb200_page_tables *tables, int32_t *sources, int32_t *destinations) {
  PageTablesArgs a;
  wb200_status st = make_page_tables(backend, tables, false, &a);
  if (st != WB200_OK) return st;
  if (tables->pages >= 2 && (!sources || !destinations)) return fail(WB200_ERR_INVALID_ARGUMENT, "sources and destinations must not be null");
  if (!on_elements(4, sources, destinations)) return off_elements();
  DeviceGuard guard(backend->device);
  if ((st = launch_pages_compact(a, sources, destinations, static_cast<cudaStream_t>(tables->stream))) == WB200_OK) backend->launches += 1;
  return st;
}

// A quantized cache moves as two caches of words, its codes and its steps.
wb200_status wb200_pages_copy_quantized(wb200_backend *backend, const wb200_quantized_cache *caches, uint32_t cache_count, uint32_t count,
                                        const int32_t *sources, const int32_t *destinations, void *stream) {
  if (!backend || (cache_count != 0 && !caches)) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  if (count > 0x7fffffffu) return fail(WB200_ERR_LIMIT, "more than 2^31 - 1 pages to copy");
  for (uint32_t i = 0; i < cache_count; ++i) {
    PagedCacheArgs one;
    QuantizedRowsArgs rows;
    const wb200_status st = make_quantized(caches + i, &one, &rows);
    if (st != WB200_OK) return st;
    wb200_quantized_cache like = caches[i];
    like.k.codes = caches[0].k.codes; like.k.steps = caches[0].k.steps;
    like.v.codes = caches[0].v.codes; like.v.steps = caches[0].v.steps;
    if (memcmp(&like, &caches[0], sizeof(like)) != 0)
      return fail(WB200_ERR_INVALID_ARGUMENT, "the caches of one copy must have the same extents, strides and format");
  }
  if (cache_count == 0 || count == 0) return WB200_OK;
  if (!sources || !destinations) return fail(WB200_ERR_INVALID_ARGUMENT, "sources and destinations must not be null");
  if (!on_elements(4, sources, destinations)) return off_elements();
  DeviceGuard guard(backend->device);
  for (int steps = 0; steps < 2; ++steps) {
    for (uint32_t first = 0; first < cache_count; first += kMaxCachesPerCopy) {
      PagedCacheArgs part[kMaxCachesPerCopy];
      const uint32_t n = cache_count - first < kMaxCachesPerCopy ? cache_count - first : kMaxCachesPerCopy;
      for (uint32_t i = 0; i < n; ++i) {
        QuantizedRowsArgs rows;
        make_quantized(caches + first + i, part + i, &rows);
        PagedCacheArgs &c = part[i];
        c.format = WB200_F32;                                // words
        c.head_dim = steps ? (c.head_dim + kQuantGroup - 1) / kQuantGroup : c.head_dim / 8;
        c.k = steps ? static_cast<void *>(rows.k.steps) : rows.k.codes;
        c.v = steps ? static_cast<void *>(rows.v.steps) : rows.v.codes;
        const int64_t k[3] = {rows.k.codes_page, rows.k.codes_row, rows.k.codes_head}, v[3] = {rows.v.codes_page, rows.v.codes_row, rows.v.codes_head};
        const int64_t ks[3] = {rows.k.steps_page, rows.k.steps_row, rows.k.steps_head}, vs[3] = {rows.v.steps_page, rows.v.steps_row, rows.v.steps_head};
        c.k_page = steps ? ks[0] : k[0] / 4; c.k_row = steps ? ks[1] : k[1] / 4; c.k_head = steps ? ks[2] : k[2] / 4;
        c.v_page = steps ? vs[0] : v[0] / 4; c.v_row = steps ? vs[1] : v[1] / 4; c.v_head = steps ? vs[2] : v[2] / 4;
      }
      const wb200_status st = launch_pages_copy(part, static_cast<int>(n), static_cast<int>(count), sources, destinations, backend->d_status + 2,
                                                static_cast<cudaStream_t>(stream));
      if (st != WB200_OK) return st;
      backend->launches += 1;
    }
  }
  return WB200_OK;
}

wb200_status wb200_pages_copy(wb200_backend *backend, const wb200_paged_cache *caches, uint32_t cache_count, uint32_t count,
                              const int32_t *sources, const int32_t *destinations, void *stream) {
  if (!backend || (cache_count != 0 && !caches)) return fail(WB200_ERR_INVALID_ARGUMENT, "null argument");
  if (count > 0x7fffffffu) return fail(WB200_ERR_LIMIT, "more than 2^31 - 1 pages to copy");
  for (uint32_t i = 0; i < cache_count; ++i) {
    PagedCacheArgs one;
    wb200_status st = make_cache(caches + i, true, &one);
    if (st != WB200_OK) return st;
    wb200_paged_cache like = caches[i];
    like.k = caches[0].k; like.v = caches[0].v; like.reserved = caches[0].reserved;
    if (memcmp(&like, &caches[0], sizeof(like)) != 0)
      return fail(WB200_ERR_INVALID_ARGUMENT, "the caches of one copy must have the same extents, strides and format");
  }
  if (cache_count == 0 || count == 0) return WB200_OK;
  if (!sources || !destinations) return fail(WB200_ERR_INVALID_ARGUMENT, "sources and destinations must not be null");
  if (!on_elements(4, sources, destinations)) return off_elements();
  DeviceGuard guard(backend->device);
  for (uint32_t first = 0; first < cache_count; first += kMaxCachesPerCopy) {
    PagedCacheArgs part[kMaxCachesPerCopy];
    const uint32_t n = cache_count - first < kMaxCachesPerCopy ? cache_count - first : kMaxCachesPerCopy;
    for (uint32_t i = 0; i < n; ++i) make_cache(caches + first + i, true, part + i);
    const wb200_status st = launch_pages_copy(part, static_cast<int>(n), static_cast<int>(count), sources, destinations, backend->d_status + 2,
                                              static_cast<cudaStream_t>(stream));
    if (st != WB200_OK) return st;
    backend->launches += 1;
  }
  return WB200_OK;
}

}  // extern "C"
