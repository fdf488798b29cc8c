// Attention of decoding rows over keys that they share: every (row, query head) pair of a group against the group's prefix, computed once for
// all rows, in bfloat16 with float32 scores, softmax statistics and sums.  Leaves, for a pair and a range of the prefix,
//     o = sum_j 2^(s_j - m) v_j / l   and   m + log2 l,     l = sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j
// which the kernel for the rows' own keys (attention_decode_shared.cu) joins with its own.  prefix_plan.cuh says how the work is cut.
//
// Any head size in steps of 16: a block takes 64 pairs, 16 a warp (mma.sync m16n8k16), and walks its range of keys in tiles of 64 that arrive by
// cp.async, two in flight; a tile serves all 64 pairs.
#include "mma_common.cuh"
#include "prefix_plan.cuh"
#include "range_check.cuh"

#define MIE_K_ATTENTION_PREFIX 16      // this kernel's number in the range report (csrc/range_check.cuh)
#define PFX_WARPS 4
#define PFX_PAIRS 64
#define PFX_TILE 64

struct PrefixParams {
    const bf16* q; int64_t q_stride;
    const bf16* k_cache; const bf16* v_cache;
    const int* block_tables; int table_stride;
    const int* row_q_start; const int* row_q_len;
    PrefixGroups groups;
    float* part_o; float* part_lse; int64_t most_slots;
    int num_heads, num_kv_heads, page_size, page_shift, chunks, chunk_heads;       // a unit: up to chunk_heads query heads of a key head, `chunks` units each
    float scale_log2e;
    int64_t num_pages; int* report;
};

__device__ __forceinline__ float exp2_fast(float x) {      // two units in the last place; -inf gives 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int D>
__global__ void __launch_bounds__(PFX_WARPS * 32)
prefix_attention_kernel(const PrefixParams p) {
    constexpr int DP = D + 8, KSTEPS = D / 16, NBLK = D / 8, PIECES = D / 8;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    bf16* k_s = reinterpret_cast<bf16*>(smem_raw);         // [2][64][DP]
    bf16* v_s = k_s + 2 * PFX_TILE * DP;
    __shared__ PrefixPart s_part;
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, tq = lane & 3;
    if (warp == 0) {
        const PrefixPart t = prefix_find(p.groups, prefix_chunk(p.groups), (int)blockIdx.x, false);
        if (lane == 0) s_part = t;
    }
    __syncthreads();
    const PrefixPart t = s_part;
    if (t.rows == 0 || t.splits == 0) {
        pdl_wait();                                        // a block without work waits too: see common.cuh
        return;
    }
    int index = (int)blockIdx.x - t.item0;
    const int split = index % t.splits;
    index /= t.splits;
    const int tile = index % t.tiles, unit = index / t.tiles;
    const int G = p.num_heads / p.num_kv_heads, kvh = unit / p.chunks, h0 = (unit - kvh * p.chunks) * p.chunk_heads;
    const int heads = min(p.chunk_heads, G - h0);          // of this unit
    const int row0 = t.first_row + tile * p.groups.tile_rows, rows = min(p.groups.tile_rows, t.first_row + t.rows - row0);
    const int pairs = rows * heads;                        // pair i: row i / heads, head i % heads of the unit
    int step0, steps;
    prefix_range(t.steps, t.splits, split, step0, steps);
    const int key_lo = step0 * PREFIX_STEP, key_hi = min(t.keys, (step0 + steps) * PREFIX_STEP);
    const int ntiles = (key_hi - key_lo + PFX_TILE - 1) / PFX_TILE;
    const int* table = p.block_tables + (int64_t)t.first_row * p.table_stride;     // the prefix lies where the group's first row says

    auto load_tile = [&](int j, int stage) {
        const int k0 = key_lo + j * PFX_TILE;
        bf16* kd = k_s + stage * PFX_TILE * DP;
        bf16* vd = v_s + stage * PFX_TILE * DP;
        for (int idx = threadIdx.x; idx < PFX_TILE * PIECES; idx += PFX_WARPS * 32) {
            const int r = idx / PIECES, c = (idx - r * PIECES) * 8, key = k0 + r;
            if (key < key_hi) {
                const int page = checked_page(table[key >> p.page_shift], p.num_pages, p.report, MIE_K_ATTENTION_PREFIX, key >> p.page_shift);
                const int64_t src = (((int64_t)page * p.num_kv_heads + kvh) * p.page_size + (key & (p.page_size - 1))) * D + c;
                cp_async16(kd + r * DP + c, p.k_cache + src);
                cp_async16(vd + r * DP + c, p.v_cache + src);
            } else {                                       // behind the prefix: zeros, so that 0 * v stays 0
                *reinterpret_cast<uint4*>(kd + r * DP + c) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(vd + r * DP + c) = make_uint4(0, 0, 0, 0);
            }
        }
    };
    load_tile(0, 0);                                       // the prefix is older than the step: before the wait
    cp_async_commit();
    pdl_wait();

    unsigned qf[KSTEPS][4];
    const bf16* q_of[2];                                   // this lane's two pairs: quad and quad + 8 of the warp's sixteen
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = warp * 16 + quad + 8 * h, r = row0 + i / heads;
        const bool on = i < pairs && p.row_q_len[r] == 1;
        q_of[h] = on ? p.q + (int64_t)p.row_q_start[r] * p.q_stride + (int64_t)(kvh * G + h0 + i % heads) * D : nullptr;
    }
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16* src = q_of[i & 1];
            qf[ks][i] = src ? *reinterpret_cast<const unsigned*>(src + ks * 16 + tq * 2 + (i >> 1) * 8) : 0u;
        }

    float o[NBLK][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NBLK; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f; }
    for (int j = 0; j < ntiles; ++j) {
        const int stage = j & 1;
        if (j + 1 < ntiles) load_tile(j + 1, stage ^ 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        if (warp * 16 < pairs) {                           // warp-uniform
            const bf16* kt = k_s + stage * PFX_TILE * DP;
            const bf16* vt = v_s + stage * PFX_TILE * DP;
            const int left = key_hi - (key_lo + j * PFX_TILE);      // keys of the tile that there are
            float s[8][4];
#pragma unroll
            for (int n = 0; n < 8; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f; }
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
                for (int n2 = 0; n2 < 4; ++n2) {
                    unsigned b0, b1, b2, b3;
                    ldmatrix_x4(b0, b1, b2, b3, kt + (n2 * 16 + (lane & 7) + (lane >> 4) * 8) * DP + ks * 16 + ((lane >> 3) & 1) * 8);
                    mma_bf16(s[2 * n2], qf[ks], b0, b1);
                    mma_bf16(s[2 * n2 + 1], qf[ks], b2, b3);
                }
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][i] = n * 8 + tq * 2 + (i & 1) < left ? s[n][i] * p.scale_log2e : -INFINITY;
                    mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
                }
            float alpha[2], ref[2], sum[2] = {0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                const float mn = fmaxf(m[h], mx[h]);
                ref[h] = mn == -INFINITY ? 0.f : mn;        // (scores that are no numbers leave the maximum alone and show in the sum)
                alpha[h] = exp2_fast(m[h] - ref[h]);
                m[h] = mn;
            }
#pragma unroll
            for (int n = 0; n < NBLK; ++n) { o[n][0] *= alpha[0]; o[n][1] *= alpha[0]; o[n][2] *= alpha[1]; o[n][3] *= alpha[1]; }
#pragma unroll
            for (int n2 = 0; n2 < 4; ++n2) {               // sixteen keys: their weights are the left operand of the product with the values
                float pv[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        pv[u][i] = exp2_fast(s[2 * n2 + u][i] - ref[i >> 1]);
                        sum[i >> 1] += pv[u][i];
                    }
                unsigned pf[4] = {pack_bf16(pv[0][0], pv[0][1]), pack_bf16(pv[0][2], pv[0][3]), pack_bf16(pv[1][0], pv[1][1]), pack_bf16(pv[1][2], pv[1][3])};
#pragma unroll
                for (int d2 = 0; d2 < NBLK / 2; ++d2) {
                    unsigned b0, b1, b2, b3;
                    ldmatrix_x4_trans(b0, b1, b2, b3, vt + (n2 * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * DP + d2 * 16 + (lane >> 4) * 8);
                    mma_bf16(o[2 * d2], pf, b0, b1);
                    mma_bf16(o[2 * d2 + 1], pf, b2, b3);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
                l[h] = l[h] * alpha[h] + sum[h];
            }
        }
        __syncthreads();                                   // the stage may be overwritten next round
    }
    cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = warp * 16 + quad + 8 * h;
        if (i >= pairs) continue;
        const int r = i / heads, head = kvh * G + h0 + i - r * heads;
        const int64_t slot = t.slot0 + (int64_t)(row0 - t.first_row + r) * t.splits + split;
        if (slot >= p.most_slots) continue;                // (the host sizes the scratch memory for every plan)
        const float inv = l[h] > 0.f ? __frcp_rn(l[h]) : l[h] == 0.f ? 0.f : NAN;      // a sum that is no number stays none
        float* op = p.part_o + (slot * p.num_heads + head) * D;
#pragma unroll
        for (int n = 0; n < NBLK; ++n) *reinterpret_cast<float2*>(op + n * 8 + tq * 2) = make_float2(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
        if (tq == 0) p.part_lse[slot * p.num_heads + head] = l[h] != 0.f ? m[h] + __log2f(l[h]) : -INFINITY;
    }
}

template <int D>
static int launch_prefix(const PrefixParams& p, long long items, cudaStream_t stream) {
    const size_t smem = (size_t)4 * PFX_TILE * (D + 8) * sizeof(bf16);
    cudaError_t e = cudaFuncSetAttribute(prefix_attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return launch_kernel(prefix_attention_kernel<D>, dim3((unsigned)items), dim3(PFX_WARPS * 32), smem, stream, p);
}

// How a launch on `sms` SMs cuts (row, head) pairs: out[0] query heads a unit, out[1] units a key head, out[2] rows a tile, out[3] items side by side.  Also
// the most slots (rows of num_heads x head_dim float32, and num_heads float32) that it writes, as the return value; -1: a size it does not take.
extern "C" long long mie_prefix_layout(int num_rows, int num_heads, int num_kv_heads, int head_dim, int sms, int* out) {
    if (num_rows < 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads || head_dim < 16 || head_dim > 128 || head_dim % 16 || sms <= 0) return -1;
    const int G = num_heads / num_kv_heads;
    out[1] = (G + PFX_PAIRS - 1) / PFX_PAIRS;
    out[0] = (G + out[1] - 1) / out[1];
    out[2] = PFX_PAIRS / out[0];
    out[3] = 2 * sms;
    return prefix_most_slots(num_rows, num_kv_heads * out[1], out[2], out[3]);
}

extern "C" int mie_prefix_attention(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, const int* block_tables, int table_stride,
                                    const int* row_q_start, const int* row_q_len, int num_rows, const int* group_start, const int* group_prefix, int groups,
                                    int num_heads, int num_kv_heads, int head_dim, int page_size, float scale, const int* layout, float* part_o,
                                    float* part_lse, long long most_slots, long long num_pages, cudaStream_t stream) {
    if (num_rows <= 0 || groups <= 0) return 0;
    if (num_kv_heads <= 0 || num_heads % num_kv_heads) return MIE_ERR_BAD_ARG;
    if (page_size < 1 || (page_size & (page_size - 1))) return MIE_ERR_BAD_ARG;
    PrefixParams p = {};
    p.q = (const bf16*)q; p.q_stride = q_stride; p.k_cache = (const bf16*)k_cache; p.v_cache = (const bf16*)v_cache;
    p.block_tables = block_tables; p.table_stride = table_stride; p.row_q_start = row_q_start; p.row_q_len = row_q_len;
    p.part_o = part_o; p.part_lse = part_lse; p.most_slots = most_slots;
    p.num_heads = num_heads; p.num_kv_heads = num_kv_heads; p.page_size = page_size;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.chunk_heads = layout[0]; p.chunks = layout[1];
    p.scale_log2e = scale * 1.4426950408889634f;
    p.num_pages = num_pages; p.report = g_range_report;
    const int64_t covered = (int64_t)table_stride * page_size;
    p.groups = PrefixGroups{group_start, group_prefix, groups, num_rows, (int)(covered < 0x7fffff00ll ? covered : 0x7fffff00ll), num_kv_heads * layout[1], layout[2], layout[3]};
    const long long items = prefix_most_items(num_rows, groups, p.groups.units, p.groups.tile_rows, p.groups.places);
    if (items > 0x7fffffffll) return MIE_ERR_TOO_LARGE;
    switch (head_dim) {
        case 16: return launch_prefix<16>(p, items, stream);
        case 32: return launch_prefix<32>(p, items, stream);
        case 48: return launch_prefix<48>(p, items, stream);
        case 64: return launch_prefix<64>(p, items, stream);
        case 80: return launch_prefix<80>(p, items, stream);
        case 96: return launch_prefix<96>(p, items, stream);
        case 112: return launch_prefix<112>(p, items, stream);
        case 128: return launch_prefix<128>(p, items, stream);
    }
    return MIE_ERR_BAD_ARG;
}
