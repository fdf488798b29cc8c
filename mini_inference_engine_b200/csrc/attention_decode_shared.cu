// The second half of attention over shared prefixes: every row's own keys (those behind its group's prefix), by the kernel of attention_decode.cu, whose
// merge takes in what attention_prefix.cu left for the prefix.  A row of no group, or of one without a prefix, is ordinary decode attention.
#include "attention_decode.cuh"

// Parameters as mie_decode_attention (attention_decode.cu), without a window, modifiers and the rotation inside the kernel; the splits merge through scratch
// memory.  The groups, the layout, the partial results and `pre_chunk` are those of mie_prefix_attention (attention_prefix.cu) on the same stream before.
extern "C" int mie_decode_attention_shared(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, const int* block_tables,
                                           int table_stride, const int* row_q_start, const int* row_q_len, const int* row_ctx_len, int num_rows,
                                           const int* group_start, const int* group_prefix, int groups, const int* layout, const float* pre_o,
                                           const float* pre_lse, const int* pre_chunk, long long most_slots, void* out, int num_heads, int num_kv_heads, int head_dim,
                                           int page_size, float scale, int splits, float* part_o, float* part_lse, int* counters, int stages,
                                           int64_t num_pages, int64_t check_pages, int min_part_tiles, int out_f32, cudaStream_t stream) {
    const int64_t covered = (int64_t)table_stride * page_size;
    const PrefixGroups g{group_start, group_prefix, groups, num_rows, (int)(covered < 0x7fffff00ll ? covered : 0x7fffff00ll), num_kv_heads * layout[1], layout[2], layout[3]};
    return decode_attention_launch<false, true>(q, q_stride, k_cache, v_cache, block_tables, table_stride, row_q_start, row_q_len, row_ctx_len, num_rows, out,
                                                num_heads, num_kv_heads, head_dim, page_size, scale, 0, splits, part_o, part_lse, counters, stream, stages,
                                                num_pages, check_pages, g_range_report, min_part_tiles, nullptr, nullptr, 0, out_f32 != 0, nullptr, 0, &g,
                                                pre_o, pre_lse, pre_chunk, most_slots);
}

// Non-zero when a block of any launch so far gave up a bounded wait (TMA copies that did not arrive).
extern "C" int mie_decode_attention_shared_error(void) { return g_error_host ? *g_error_host : 0; }
extern "C" void mie_decode_attention_shared_clear_error(void) { if (g_error_host) *g_error_host = 0; }
