// Attention over shared prefixes where reading them row by row costs less than taking rows together: decode attention in which a row's first keys lie
// where the block table of its group's first row says.  One launch instead of two that depend on one another, and the second row to ask finds a page in L2.
#include "attention_decode.cuh"
#include "prefix_args.cuh"

extern "C" int mie_decode_attention_through(const SharedArgs* a, cudaStream_t stream) {
    const PrefixGroups g = shared_groups_of(*a);
    return decode_attention_launch<false, DEC_THROUGH>(a->q, a->q_stride, a->k_cache, a->v_cache, a->block_tables, a->table_stride, a->row_q_start, a->row_q_len,
                                                       a->row_ctx_len, a->num_rows, a->out, a->num_heads, a->num_kv_heads, a->head_dim, a->page_size, a->scale, 0,
                                                       a->splits, a->part_o, a->part_lse, a->counters, stream, a->stages, a->tma ? a->num_pages : 0, a->num_pages,
                                                       g_range_report, a->min_part_tiles, nullptr, nullptr, 0, a->out_f32 != 0, nullptr, 0, &g);
}

// Non-zero when a block of any launch so far gave up a bounded wait (TMA copies that did not arrive).
extern "C" int mie_decode_attention_through_error(void) { return g_error_host ? *g_error_host : 0; }
extern "C" void mie_decode_attention_through_clear_error(void) { if (g_error_host) *g_error_host = 0; }
