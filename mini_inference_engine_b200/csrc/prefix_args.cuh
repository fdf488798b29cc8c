// Arguments of attention over shared prefixes, laid out alike in kernels/ops.py (_SharedArgs).
#pragma once
#include "prefix_plan.cuh"

struct SharedArgs {
    // a call's own: packed by the caller in front of what a plan keeps
    const void* q; const void* k_cache; const void* v_cache;
    const int* block_tables; const int* row_q_start; const int* row_q_len; const int* row_ctx_len;
    const int* group_start; const int* group_prefix;
    void* out;
    long long q_stride;
    int table_stride, out_f32;
    float scale;
    int walk;                                                                     // 2: row by row (attention_decode_through.cu); 1: prefix and own keys in one walk; 0: a kernel for the prefixes, then ...
    int (*own_keys)(const SharedArgs*, cudaStream_t);                             // ... this one for own keys (mie_decode_attention_shared, another library's)
    float* pre_o; float* pre_lse; int* pre_chunk; int* row_info; int* marks;      // scratch: partial results of ranges, how prefixes are cut, a row's results, rows marked
    float* part_o; float* part_lse; int* counters;                                // scratch of the decode kernel (splits > 1); counters and marks are left zero
    long long num_pages, most_slots;
    int num_rows, groups, num_heads, num_kv_heads, head_dim, page_size;
    int splits, stages, tma, min_part_tiles;                                      // the decode kernel's plan for the rows' own keys
    int chunk_heads, chunks, tile_rows, places;                                   // mie_prefix_layout (with walk) ...
    int most_prefix, most_own;                                                    // ... which goes by these bounds on a prefix and on a row's own keys
};

static inline PrefixGroups shared_groups_of(const SharedArgs& a) {
    const long long covered = (long long)a.table_stride * a.page_size;
    return PrefixGroups{a.group_start, a.group_prefix, a.groups, a.num_rows, (int)(covered < 0x7fffff00ll ? covered : 0x7fffff00ll), a.num_kv_heads * a.chunks, a.tile_rows,
                        a.places};
}
