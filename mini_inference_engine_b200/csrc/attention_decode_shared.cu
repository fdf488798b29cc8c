// The second half of attention over shared prefixes where the first is attention_prefix.cu's kernel for any head size: every row's own keys (those behind its
// group's prefix), by the kernel of attention_decode.cu, whose merge takes in what was left for the prefix.  A row of no group, or of one without a prefix, is
// ordinary decode attention.
#include "attention_decode.cuh"
#include "prefix_args.cuh"

// `a`: as for mie_prefix_attention (attention_prefix.cu) before, on the same stream; groups 0: nothing came before.  The splits merge through scratch memory.
extern "C" int mie_decode_attention_shared(const SharedArgs* a, cudaStream_t stream) {
    const PrefixGroups g = shared_groups_of(*a);
    return decode_attention_launch<false, DEC_SHARED>(a->q, a->q_stride, a->k_cache, a->v_cache, a->block_tables, a->table_stride, a->row_q_start, a->row_q_len,
                                                a->row_ctx_len, a->num_rows, a->out, a->num_heads, a->num_kv_heads, a->head_dim, a->page_size, a->scale, 0,
                                                a->splits, a->part_o, a->part_lse, a->counters, stream, a->stages, a->tma ? a->num_pages : 0, a->num_pages,
                                                g_range_report, a->min_part_tiles, nullptr, nullptr, 0, a->out_f32 != 0, nullptr, 0, &g, a->pre_o, a->pre_lse,
                                                a->pre_chunk, a->most_slots);
}

// Non-zero when a block of any launch so far gave up a bounded wait (TMA copies that did not arrive).
extern "C" int mie_decode_attention_shared_error(void) { return g_error_host ? *g_error_host : 0; }
extern "C" void mie_decode_attention_shared_clear_error(void) { if (g_error_host) *g_error_host = 0; }
