// Attention of decoding rows over keys that they share: every (row, query head) pair of a group against the group's prefix, computed once for
// all rows, in bfloat16 with float32 scores, softmax statistics and sums.  Leaves, for a pair and a range of keys,
//     o = sum_j 2^(s_j - m) v_j / l   and   m + log2 l,     l = sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j
// which a kernel behind joins with the pair's other ranges.  prefix_plan.cuh says how the work is cut.  (Where little is shared the rows go one by one:
// attention_decode_through.cu.)
//
// Two ways.  Heads of 64 and 128 on pages of 8 positions or more: tcgen05, prefix and own keys in one walk, below.  Any head size in steps of 16: a
// block takes 64 pairs, 16 a warp (mma.sync m16n8k16), and walks its range of the prefix in tiles of 64 keys that arrive by cp.async, two in flight; a tile
// serves all 64 pairs, and the kernel for the rows' own keys (attention_decode_shared.cu) joins its results with its own.
#include "mma_common.cuh"
#include "tcgen05_common.cuh"
#include "prefix_plan.cuh"

#define PFX_WARPS 4
#define PFX_PAIRS 64
#define PFX_TILE 64

struct PrefixParams {
    const bf16* q; int64_t q_stride;
    const bf16* k_cache; const bf16* v_cache;
    const int* block_tables; int table_stride;
    const int* row_q_start; const int* row_q_len; const int* row_ctx_len;
    PrefixGroups groups;
    float* part_o; float* part_lse; int64_t most_slots; int* chunk;       // chunk: how the prefixes are cut, for the kernel behind
    int num_heads, num_kv_heads, page_size, page_shift, chunks, chunk_heads;       // a unit: up to chunk_heads query heads of a key head, `chunks` units each
    float scale_log2e;
    int64_t num_pages; int* report; int* error;
};

__device__ __forceinline__ float exp2_fast(float x) {      // two units in the last place; -inf gives 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ bool writes_prefix(const PrefixParams& p, int row, int keys) { return writes_prefix(p.row_q_len[row], p.row_ctx_len[row], keys); }

template <int D>
__global__ void __launch_bounds__(PFX_WARPS * 32)
prefix_attention_kernel(const PrefixParams p) {
    constexpr int DP = D + 8, KSTEPS = D / 16, NBLK = D / 8, PIECES = D / 8;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    bf16* k_s = reinterpret_cast<bf16*>(smem_raw);         // [2][64][DP]
    bf16* v_s = k_s + 2 * PFX_TILE * DP;
    __shared__ PrefixPart s_part;
    __shared__ int s_chunk;
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, tq = lane & 3;
    if (blockIdx.x == 0 && warp == 1)
        for (int g = lane; g < p.groups.groups; g += 32) check_group(p.groups, g, p.report);
    if (warp == 0) {
        const int chunk = prefix_chunk(p.groups);
        const PrefixPart t = prefix_find(p.groups, chunk, (int)blockIdx.x, false);
        if (lane == 0) { s_part = t; s_chunk = chunk; }
    }
    __syncthreads();
    const PrefixPart t = s_part;
    if (t.rows == 0 || t.splits == 0) {
        pdl_wait();                                        // a block without work waits too: see common.cuh
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.chunk = s_chunk;
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
    // The prefix is older than the step, so that its first tile is asked for before the wait -- unless a row of the group writes a key of it in this step.
    bool young = false;
    for (int r = t.first_row + threadIdx.x; r < t.first_row + t.rows; r += PFX_WARPS * 32) young |= writes_prefix(p, r, t.keys);
    young = __syncthreads_or(young);
    if (young) pdl_wait();
    load_tile(0, 0);
    cp_async_commit();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.chunk = s_chunk;

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

// The shared memory of a kernel, asked for once a device (`granted`: the kernel's devices).
template <typename K>
static int grant_shared(K kernel, size_t bytes, unsigned long long& granted) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (device <= 63 && (__atomic_load_n(&granted, __ATOMIC_RELAXED) >> device & 1)) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && device <= 63) __atomic_fetch_or(&granted, 1ull << device, __ATOMIC_RELAXED);
    return (int)e;
}

template <int D>
static int launch_prefix(const PrefixParams& p, long long items, cudaStream_t stream) {
    const size_t smem = (size_t)4 * PFX_TILE * (D + 8) * sizeof(bf16);
    static unsigned long long granted = 0;
    const int rc = grant_shared(prefix_attention_kernel<D>, smem, granted);
    if (rc) return rc;
    return launch_kernel(prefix_attention_kernel<D>, dim3((unsigned)items), dim3(PFX_WARPS * 32), smem, stream, p);
}

// --------------------------------------------------------------------------- heads of 64 and 128: tcgen05, one walk
//
// Rows of a group (or rows that belong to none) are taken `tile_rows` at a time: up to 256 (row, head) pairs of a unit, two tiles of 128, one pair a
// tensor-memory lane.  Their walk goes in steps of 128 keys: first the group's prefix, which all pairs see, then the rows' own keys, laid end to end a page (or
// 128 keys of one) a slot, where a pair sees its own row's keys only; a step holds own keys of one tile, and the tiles take turns.  An item is a range of steps
// of such a walk; it leaves o and m + log2 l of its keys for every pair (-inf where a pair saw none), and a second kernel joins the ranges of a row.  Own keys
// that way cost their bytes and little else: attended over by the decode kernel behind a kernel for the prefixes, 64 rows of up to 512 own keys behind 8,000
// took 62 us, 256 rows of up to 96 behind 16,384 143 us, of which 40 and 54 were the decode kernel's.  (Rows of many hundred own keys behind short prefixes are not
// what the walk is for: 32 heads of 64 on 4, 256 rows of up to 900 behind 400 94 us, ordinary decode attention 58; kernels/attention.py: sharing_weight.)
//
// Two chains of work run side by side, each with four softmax warps, a thread that issues its products, and its own S, P and O in tensor memory:
//   S = Q K^T; the chain's threads move their rows of S into registers, write P = 2^(s - m), rounded to bfloat16, back, and
//   O += P V with P as the left operand out of tensor memory and V as it lies.
// (m follows the running maximum in jumps of 2^8 only: the sums take the weights unrounded, and the greatest weight, which need not be 1, is rounded like the others.)
// Such a chain takes 4,000 cycles a step (heads of 128), four times what its products take; two fill one another's gaps.  With two tiles of pairs a chain owns a tile, and a
// step of the prefix serves both; with one the chains take the steps in turns over the same queries and leave a result each.
// Keys and values come by TMA, a slot a copy, keys and values each with barriers of their own: keys of a later step arrive as soon as S is formed.
// Tensor memory: heads of 64 S 2 x 128 columns, P 2 x 64, O 2 x 64; S of the next step is issued as soon as the rows are in registers.  Heads of 128: O takes
// 2 x 128, and P lies over the S that it came from.  A step's S, P and product with the values then go in halves of 64 keys: S of the next step's first half is
// formed under the softmax of this one's second (whole steps, S behind the product with the values: 51 -> 45 us for 64 rows behind 8,000 keys, 124 -> 110 for 256
// behind 16,384; 43 and 113 now).
//
// Values of one row must not reach another's output: slots' keys that are nobody's (in front of a row's own keys, behind its context) are made zero in
// shared memory, and so are own values that are not finite, since 0 times those is not 0; the row is marked, and the joining kernel adds them to its output.
#define PT_THREADS 384
#define PT_ROWS 128
#define PT_KEYS 128
#define PT_COST_START 7            // what starting and ending an item costs, in steps (3: 131 us for 256 rows behind 16,384 keys instead of 124)
#define PT_WALK_PAIRS 128          // pairs on a key head up to which the kernel for any head size takes over (see mie_prefix_layout) ...
#define PT_WALK_BYTES (16 << 20)   // ... unless heads are of 128 and there is this much to read
#define PT_MOST_TILES 512          // tiles of rows that a launch can plan for ...
#define PT_MOST_SEGMENTS 63        // ... and groups with the rows between them

struct WalkParams {
    PrefixParams b;
    int2* row_info; int* marks;                            // row_info: a row's first slot and its ranges; marks: 0, or the query heads of a (row, key head) with values that are not finite
};

template <int D> constexpr int PT_STAGES = D == 64 ? 4 : 2;
template <int D> constexpr size_t PT_SMEM = (size_t)PT_ROWS * D * 2 * 2 + (size_t)PT_STAGES<D> * 2 * PT_KEYS * D * 2 + 1024;

// What a block needs to know of the step's plan, and the scratch it is worked out in.
struct WalkPlan {
    int first[PT_MOST_SEGMENTS], rows[PT_MOST_SEGMENTS], keys[PT_MOST_SEGMENTS], tile0[PT_MOST_SEGMENTS];      // segments: rows, shared keys, first tile of rows
    int segments, tiles;
    int slots[2 * PT_MOST_TILES];                          // own slots of a tile of pairs
    int steps[PT_MOST_TILES], seg[PT_MOST_TILES];          // steps of a tile of rows' walk; its segment
    unsigned long long best;
    int young;                                             // some row's step writes a key of its prefix
    int found, splits, item0, slot0;                       // the item's tile of rows (-1: none), its ranges, first item and slot
    int own_first[2 * PT_ROWS + 1], ctx[2 * PT_ROWS];      // of the tile's rows: first own slot; context (0: not a row of one new token)
};

// Keys of an own slot as a shift, and a row's own slots: slots are whole pages, or 128 keys of a longer page.
#define PT_KEYS_SHIFT 7
__device__ __forceinline__ int slot_shift(int page_shift) { return min(page_shift, PT_KEYS_SHIFT); }
__device__ __forceinline__ int own_slots(int ctx, int prefix, int ss) { return ctx > prefix ? ((ctx + (1 << ss) - 1) >> ss) - (prefix >> ss) : 0; }

// By the whole block.  Afterwards w.found is the item's tile of rows.
template <int T>
__device__ __forceinline__ void walk_plan(WalkPlan& w, const WalkParams& q, int item) {
    const PrefixGroups& p = q.b.groups;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ss = slot_shift(q.b.page_shift), half = p.tile_rows / 2;
    // segments: the rows in front of the first group, the groups, the rows behind the last
    if (tid < p.groups + 2) {
        auto at = [&](int k) { return max(0, min(p.start[k], p.num_rows)); };
        const int a = tid == 0 ? 0 : at(tid - 1), b = tid == p.groups + 1 ? p.num_rows : at(tid);
        w.first[tid] = a;
        w.rows[tid] = max(0, b - a);
        w.keys[tid] = tid >= 1 && tid <= p.groups ? max(0, min(p.prefix[tid - 1], p.most_keys)) : 0;
    }
    if (item == 0 && tid < p.groups) check_group(p, tid, q.b.report);
    if (tid == 0) { w.segments = p.groups + 2; w.best = ~0ull; w.found = -1; w.young = 0; }
    // this thread's first row (the others are asked for where there are more rows than threads)
    const int r_len = tid < p.num_rows ? q.b.row_q_len[tid] : 0, r_ctx = tid < p.num_rows ? q.b.row_ctx_len[tid] : 0;
    __syncthreads();
    if (warp == 0) {                                       // first tiles of the segments
        int at = 0;
        for (int g0 = 0; g0 < w.segments; g0 += 32) {
            const int g = g0 + lane, n = g < w.segments ? (w.rows[g] + p.tile_rows - 1) / p.tile_rows : 0;
            int sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += up; }
            if (g < w.segments) {
                w.tile0[g] = at + sum - n;
                for (int i = 0; i < n && at + sum - n + i < PT_MOST_TILES; ++i) w.seg[at + sum - n + i] = g;
            }
            at += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) w.tiles = min(at, PT_MOST_TILES);
        const int tiles = min(at, PT_MOST_TILES);
        for (int t = lane; t < 2 * tiles; t += 32) w.slots[t] = 0;
    }
    __syncthreads();
    const int tiles = w.tiles;
    for (int r = tid; r < p.num_rows; r += T) {            // own slots of the tiles of pairs
        int g = 0;
        while (g + 1 < w.segments && !(r >= w.first[g] && r < w.first[g] + w.rows[g])) ++g;
        const int in_seg = r - w.first[g], t = w.tile0[g] + in_seg / p.tile_rows;
        const int len = r == tid ? r_len : q.b.row_q_len[r], ctx = r == tid ? r_ctx : q.b.row_ctx_len[r];
        if (in_seg >= 0 && writes_prefix(len, ctx, w.keys[g])) w.young = 1;
        if (in_seg >= 0 && t < tiles && len == 1) atomicAdd(&w.slots[2 * t + (in_seg % p.tile_rows) / half], own_slots(min(ctx, p.most_keys), w.keys[g], ss));
    }
    __syncthreads();
    const int ws = PT_KEYS_SHIFT - ss, W = 1 << ws;        // own slots a step
    for (int t = tid; t < tiles; t += T)
        w.steps[t] = (w.keys[w.seg[t]] + PREFIX_STEP - 1) / PREFIX_STEP + ((w.slots[2 * t] + W - 1) >> ws) + ((w.slots[2 * t + 1] + W - 1) >> ws);
    __syncthreads();
    // How many ranges the longest walk is cut into: a candidate a lane (prefix_plan.cuh says what is weighed).
    if (warp < PREFIX_MAX_SPLITS / 32) {
        int most = 1;
        for (int t = lane; t < tiles; t += 32) most = max(most, w.steps[t]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int s = warp * 32 + lane + 1;
        if (s <= most) {
            const int c = (most + s - 1) / s;
            unsigned items = 0;
            for (int t = 0; t < tiles; ++t) items += p.units * prefix_splits(w.steps[t], c);
            if (s == 1 || items <= 2u * p.places) {
                const unsigned long long cost = (unsigned long long)((items + p.places - 1) / p.places) * (c + PT_COST_START);
                atomicMin(&w.best, cost << 32 | (0xffffffffu - (unsigned)c));
            }
        }
    }
    __syncthreads();
    if (warp == 0) {
        const int c = max(1, (int)(0xffffffffu - (unsigned)w.best));
        int items = 0, slots = 0;
        for (int t0 = 0; t0 < tiles; t0 += 32) {
            const int t = t0 + lane, splits = t < tiles ? prefix_splits(w.steps[t], c) : 0;
            int rows = 0;
            if (t < tiles) rows = min(p.tile_rows, w.rows[w.seg[t]] - (t - w.tile0[w.seg[t]]) * p.tile_rows);
            const int n = p.units * splits, k = rows * splits * (rows > half ? 1 : 2);      // (a tile of pairs alone: a result a chain)
            int ni = n, ki = k;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, ni, o), b = __shfl_up_sync(0xffffffffu, ki, o);
                if (lane >= o) { ni += a; ki += b; }
            }
            const unsigned hit = __ballot_sync(0xffffffffu, item >= items + ni - n && item < items + ni);
            if (hit) {
                if (lane == __ffs(hit) - 1) { w.found = t; w.splits = splits; w.item0 = items + ni - n; w.slot0 = slots + ki - k; }
                break;
            }
            items += __shfl_sync(0xffffffffu, ni, 31);
            slots += __shfl_sync(0xffffffffu, ki, 31);
        }
    }
    __syncthreads();
}

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 1)
prefix_walk_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const WalkParams wp) {
    constexpr int PARTS = D / 64, STAGES = PT_STAGES<D>;
    constexpr uint32_t SUB = 128 * 64 * 2;                 // one [128 x 64] part of a tile
    constexpr uint32_t TILE = PARTS * SUB;
    constexpr bool OVER = D == 128;                        // P lies over S, and a step goes in halves of 64 keys
    constexpr int HALVES = OVER ? 2 : 1, HK = PT_KEYS / HALVES;
    constexpr uint32_t TMEM_S = 0, TMEM_P = OVER ? 0 : 256, TMEM_O = OVER ? 256 : 384, S_STEP = 128, P_STEP = OVER ? 128 : 64, O_STEP = D, HALF = 64;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t q_full[2], k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2][HALVES], s_free[2], p_full[2][HALVES], pv_done[2], o_full[2], exp_done[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ WalkPlan plan;
    const PrefixParams& p = wp.b;
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char* tiles = smem_dyn + (base - smem_u32(smem_dyn));
    auto q_off = [&](int u) { return (uint32_t)u * TILE; };
    auto k_off = [&](int st) { return 2 * TILE + (uint32_t)st * 2 * TILE; };
    auto v_off = [&](int st) { return 2 * TILE + (uint32_t)st * 2 * TILE + TILE; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    walk_plan<PT_THREADS>(plan, wp, (int)blockIdx.x);
    if (plan.found < 0) {
        pdl_wait();                                        // a block without work waits too: see common.cuh
        return;
    }
    const int t = plan.found, splits = plan.splits, seg = plan.seg[t], in_seg = t - plan.tile0[seg];
    const int index = (int)blockIdx.x - plan.item0, split = index % splits, unit = index / splits;
    const int G = p.num_heads / p.num_kv_heads, kvh = unit / p.chunks, h0 = (unit - kvh * p.chunks) * p.chunk_heads;
    const int heads = min(p.chunk_heads, G - h0);          // of this unit
    const int half = p.groups.tile_rows / 2;               // rows of a tile of pairs
    const int leader = plan.first[seg], row0 = leader + in_seg * p.groups.tile_rows, rows = min(p.groups.tile_rows, leader + plan.rows[seg] - row0);
    const bool both = rows > half;                         // two tiles of pairs, a chain each; else one, both chains over it
    const int prefix = plan.keys[seg], ss = slot_shift(p.page_shift), sk = 1 << ss, ws = PT_KEYS_SHIFT - ss, W = 1 << ws;
    const int pre_steps = (prefix + PREFIX_STEP - 1) / PREFIX_STEP;
    int x0, J;                                             // this item's steps: x0 .. x0 + J - 1 of the walk
    prefix_range(plan.steps[t], splits, split, x0, J);
    // the rows' own slots, one behind another
    if (warp == 0) {
        int at = 0;
        for (int i0 = 0; i0 < rows; i0 += 32) {
            const int i = i0 + lane, r = row0 + i;
            const bool on = i < rows && p.row_q_len[r] == 1;
            const int all = on ? p.row_ctx_len[r] : 0, ctx = min(all, p.groups.most_keys);
            if (on && unit == 0 && split == 0 && (all < prefix || all > p.groups.most_keys))         // a context that ends inside its prefix, or beyond its block table
                range_report(p.report, MIE_RANGE_POSITION, MIE_K_ATTENTION_PREFIX, r, all);
            const int n = own_slots(ctx, prefix, ss);
            int sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += up; }
            if (i < rows) { plan.own_first[i] = at + sum - n; plan.ctx[i] = on ? max(1, ctx) : 0; }
            at += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) plan.own_first[rows] = at;
    }
    if (threadIdx.x == 32) {
        abort_flag = 0;
        for (int u = 0; u < 2; ++u) {
            for (int h = 0; h < HALVES; ++h) { mbar_init(&s_full[u][h], 1); mbar_init(&p_full[u][h], 4); }
            mbar_init(&q_full[u], 4); mbar_init(&s_free[u], 4);
            mbar_init(&pv_done[u], 1); mbar_init(&o_full[u], 1); mbar_init(&exp_done[u], 4);
        }
        for (int st = 0; st < STAGES; ++st) {              // (a stage is given back by both chains' products, or twice by those of the one that uses it)
            mbar_init(&k_full[st], 1); mbar_init(&v_full[st], 1); mbar_init(&k_empty[st], 2); mbar_init(&v_empty[st], 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    volatile int* abort_p = &abort_flag;
    const int npre = max(0, min(J, pre_steps - x0));       // the first npre of this item's steps are the prefix's
    // own slots go by lists, one a tile of pairs: list l's begin at list0[l], and take list_steps[l] steps, turn by turn while both have some
    const int list0[2] = {0, both ? plan.own_first[half] : 0}, list_end[2] = {both ? plan.own_first[half] : plan.own_first[rows], plan.own_first[rows]};
    const int steps0 = (list_end[0] + W - 1) >> ws, steps1 = both ? (list_end[1] - list0[1] + W - 1) >> ws : 0;
    const WalkSteps steps = {J, npre, x0 - pre_steps, steps0, steps1, both};
    auto own_step = [&](int j) { return walk_own_step(steps, j); };
    auto active = [&](int c, int j) { return walk_takes_part(steps, c, j); };
    // the row of the tile of rows that an own slot belongs to
    auto owner = [&](int slot) {
        int lo = 0, hi = rows - 1;                         // the last row whose first slot is not behind it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (plan.own_first[mid] <= slot) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    const int own_begin = prefix >> ss << ss;                // where every row's first own slot begins

    // ---- the keys and values: lane c copies slot c of a step
    const int* table = p.block_tables + (int64_t)leader * p.table_stride;                // the prefix lies where the group's first row says
    auto copies_of = [&](int j) {
        if (j < npre) return (min((x0 + j + 1) * PT_KEYS, prefix) - (x0 + j) * PT_KEYS + sk - 1) >> ss;
        const OwnStep o = own_step(j);
        return min(W, (o.list ? list_end[1] : list_end[0]) - (o.list ? list0[1] : 0) - o.k * W);
    };
    // Where this lane's copy of step j begins: the entry of a block table, fetched long before it is asked for, and the key's place in that page.
    struct Place { int entry, page, offset; };
    auto place_of = [&](int j) {
        Place at = {0, 0, -1};
        if (j >= J || lane >= copies_of(j)) return at;
        int key;
        const int* from = table;
        if (j < npre) key = (x0 + j) * PT_KEYS + lane * sk;
        else {
            const OwnStep o = own_step(j);
            const int slot = (o.list ? list0[1] : 0) + o.k * W + lane, i = owner(slot);
            key = own_begin + (slot - plan.own_first[i]) * sk;
            from = p.block_tables + (int64_t)(row0 + i) * p.table_stride;
        }
        at.entry = key >> p.page_shift;
        at.page = from[at.entry];
        at.offset = key & (p.page_size - 1);
        return at;
    };
    auto row_of = [&](const Place& at) {                   // the cache's key row
        if (at.offset < 0) return 0;
        return (checked_page(at.page, p.num_pages, p.report, MIE_K_ATTENTION_PREFIX, at.entry) * p.num_kv_heads + kvh) * p.page_size + at.offset;
    };
    auto load = [&](int j, uint64_t* full, const CUtensorMap* map, uint32_t to, int src_row) {
        const int copies = copies_of(j);
        if (lane == 0) mbar_expect_tx(full, (uint32_t)copies * sk * 128u * PARTS);
        __syncwarp();
        if (lane < copies) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) tma_load_2d(tiles + to + part * SUB + (uint32_t)lane * sk * 128u, map, full, part * 64, src_row);
        }
    };
    // Warp 0 fetches keys, warp 11 values: neither waits for places of the other's.
    const bool fetches = warp == 0 || warp == 11;
    uint64_t* full = warp == 0 ? k_full : v_full;
    uint64_t* empty = warp == 0 ? k_empty : v_empty;
    const CUtensorMap* map = warp == 0 ? &map_k : &map_v;
    auto to = [&](int st) { return warp == 0 ? k_off(st) : v_off(st); };
    const int ahead = min(STAGES, J), early = plan.young ? 0 : min(ahead, npre);      // a prefix older than the step: its first keys are on their way before the wait
    Place later;                                           // of the step behind those that shared memory has places for
    if (fetches) {
        Place at[STAGES];
#pragma unroll
        for (int j = 0; j < STAGES; ++j) at[j] = place_of(j);
#pragma unroll
        for (int j = 0; j < STAGES; ++j) if (j < early) load(j, &full[j], map, to(j), row_of(at[j]));
        pdl_wait();
#pragma unroll
        for (int j = 0; j < STAGES; ++j) if (j >= early && j < ahead) load(j, &full[j], map, to(j), row_of(at[j]));
        later = place_of(STAGES);
    }
    // Softmax warps 2..5 (chain 0) and 6..9 (chain 1), a thread a pair: which, and its query, under the copies and the hand-out of tensor memory.  A query's 16-byte
    // pieces go to neighbouring lanes (a lane its own query, behind the hand-out: 4 us more).
    const int u = warp >= 6 ? 1 : 0, q = warp & 3, r = q * 32 + lane;      // (the lanes of tensor memory that a warp reaches go by its number)
    const int in_tile = (both ? u * half : 0) + r / heads, my_row = row0 + in_tile, head = kvh * G + h0 + r % heads;
    const bool softmax = warp >= 2 && warp <= 9, pair = softmax && r / heads < half && in_tile < rows && plan.ctx[min(in_tile, rows - 1)] > 0;
    if (softmax && (both || u == 0)) {
        constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;             // lanes a query, queries an instruction
        const int64_t mine = pair ? (int64_t)p.row_q_start[my_row] * p.q_stride + (int64_t)head * D : -1;
        pdl_wait();
        uint4 v[LANES];
#pragma unroll
        for (int i = 0; i < LANES; ++i) {                  // (where there is no pair the first query is read, and zeros are stored: a branch a load put them one behind another, 5 us)
            const int64_t src = __shfl_sync(0xffffffffu, mine, i * AT_ONCE + lane / LANES);
            v[i] = *reinterpret_cast<const uint4*>(p.q + max((int64_t)0, src) + lane % LANES * 8);
        }
#pragma unroll
        for (int i = 0; i < LANES; ++i) {
            const int to_r = q * 32 + i * AT_ONCE + lane / LANES, c = lane % LANES;
            if (__shfl_sync(0xffffffffu, mine, i * AT_ONCE + lane / LANES) < 0) v[i] = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(tiles + q_off(u) + (c >> 3) * SUB + to_r * 128 + (((c & 7) ^ (to_r & 7)) << 4)) = v[i];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[u]);
    }
    // Tensor memory is taken behind the wait, and the next kernel let in behind that: a block that held it before the kernels in front are done could keep
    // it from a block of theirs, and one that came later from this one.
    pdl_wait();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int per_row = splits * (both ? 1 : 2);           // results of a row
    if (unit == 0 && split == 0)                           // where the joining kernel finds them
        for (int i = threadIdx.x; i < rows; i += PT_THREADS) wp.row_info[row0 + i] = make_int2(plan.slot0 + i * per_row, plan.ctx[i] ? per_row : 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem_base = tmem_base_slot;

    if (fetches) {
        // the rest of the steps
        // (asking L2 for later steps as well gained nothing: 53 -> 57 us for 64 rows behind 8,000 keys.  A copy's instruction takes 100 cycles for every lane that
        // issues one, and sixteen a step are two thirds of what a step may take already.)
        for (int j = STAGES; j < J; ++j) {
            const int st = j % STAGES, src_row = row_of(later);
            later = place_of(j + 1);
            int ok = 1;
            if (lane == 0) ok = mbar_wait(&empty[st], ((j / STAGES) & 1) ^ 1, abort_p) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            load(j, &full[st], map, to(st), src_row);
        }
    } else if (warp == 1 || warp == 10) {
        const int mu = warp == 1 ? 0 : 1;
        {
            // ---- the warp that issues for chain mu: it walks its loop as a whole, so that what feeds the instructions stays uniform, and one lane issues
            const bool issuer = elect_one();               // (one lane alone in the loop: 740 cycles for the eight products of P V instead of 300)
            auto wait_for = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_p)) != 0; };
            const uint32_t idesc_s = umma_idesc_bf16(PT_ROWS, HK), idesc_o = umma_idesc_bf16(PT_ROWS, D) | (1u << 16);
            constexpr int KS = D / 16, KV = HK / 16;
            const int qt = both ? mu : 0;
            uint64_t dq[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dq[ks] = umma_desc_sw128(base + q_off(qt) + (ks / 4) * SUB + (ks % 4) * 32);
            const uint64_t dk0 = umma_desc_sw128(base + k_off(0)), dv0 = umma_desc_sw128_mn(base + v_off(0), SUB);
            constexpr uint64_t STAGE_STEP = (2 * TILE) >> 4;       // descriptors of another stage differ in the address field only
            const uint32_t s_at = tmem_base + TMEM_S + S_STEP * mu, p_at = tmem_base + TMEM_P + P_STEP * mu, o_at = tmem_base + TMEM_O + O_STEP * mu;
            bool ok = wait_for(&q_full[qt], 0);
            auto next_of = [&](int j) {                    // the chain's next step
                for (++j; j < J && !active(mu, j);) ++j;
                return j;
            };
            auto give_back = [&](uint64_t* empty, int j) {
                umma_commit(empty);
                if (!(both && j < npre)) umma_commit(empty);
            };
            auto scores = [&](int j, int h) {              // S of half h of step j, once its keys are here
                const int st = j % STAGES;
                // (behind steps of the other chain alone: once that is done with all of its own, what lay here before has come; the values' waits lie behind this one)
                if (h == 0) ok = (!walk_behind_other(steps, mu, j, STAGES) || wait_for(&o_full[mu ^ 1], 0)) && wait_for(&k_full[st], (j / STAGES) & 1);
                if (!ok) return;
                tc_fence_after();
                if (issuer) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
                        umma_bf16(s_at + h * HALF, dq[ks], dk0 + STAGE_STEP * st + (uint64_t)(((ks / 4) * SUB + h * HK * 128 + (ks % 4) * 32) >> 4), idesc_s, ks > 0 ? 1u : 0u);
                    umma_commit(&s_full[mu][h]);
                    if (h == HALVES - 1) give_back(&k_empty[st], j);
                }
                __syncwarp();
            };
            int used = 0;                                  // steps that the chain has taken part in
            int j = next_of(-1);
            if (j < J)
                for (int h = 0; h < HALVES && ok; ++h) scores(j, h);
            while (j < J && ok) {
                const int st = j % STAGES, next = next_of(j);
                if (!OVER && next < J) {                   // the next scores, as soon as the rows of these are in registers
                    ok = wait_for(&s_free[mu], used & 1);
                    if (ok) scores(next, 0);
                    if (!ok) break;
                }
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    ok = wait_for(&p_full[mu][h], used & 1) && (h > 0 || wait_for(&v_full[st], (j / STAGES) & 1));      // P is written, O rescaled
                    if (!ok) break;
                    tc_fence_after();
                    if (issuer) {
#pragma unroll
                        for (int kk = 0; kk < KV; ++kk)
                            umma_bf16_ts(o_at, p_at + h * HALF + kk * 8, dv0 + STAGE_STEP * st + (uint64_t)(((h * KV + kk) * 2048) >> 4), idesc_o, (used > 0 || h > 0 || kk > 0) ? 1u : 0u);
                        umma_commit(&pv_done[mu]);         // P may be overwritten, O rescaled
                        if (h == HALVES - 1) {
                            if (next >= J) umma_commit(&o_full[mu]);
                            give_back(&v_empty[st], j);
                        }
                    }
                    __syncwarp();
                    // (products run in the order they were issued: where P lies over S, it has been read when the next S overwrites it)
                    if (OVER && next < J) scores(next, h);
                    if (!ok) break;
                }
                ++used;
                j = next;
            }
        }
        __syncwarp();
    } else {
        // ---- softmax
        const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16);
        const uint32_t S_AT = lane_addr + TMEM_S + S_STEP * u, P_AT = lane_addr + TMEM_P + P_STEP * u, O_AT = lane_addr + TMEM_O + O_STEP * u;
        bool ok = true;
        // own keys that this pair sees, counted from its list's first: [seen_lo, seen_hi)
        int seen_lo = 0, seen_hi = 0;
        if (pair && plan.own_first[in_tile + 1] > plan.own_first[in_tile]) {
            const int at = (plan.own_first[in_tile] - (both && u ? list0[1] : 0)) << ss;
            seen_lo = at + (prefix - own_begin);
            seen_hi = at + (plan.ctx[in_tile] - own_begin);
        }
        // The chains take turns at the exponentials of the steps that both take part in (118 us for 256 rows without): half n of chain 0 behind half n - 1 of chain 1,
        // that behind half n of chain 0.  Every half takes its turn, one without keys too: a chain that went on without would complete a second phase of its
        // barrier, and the other, if it had not asked for the first by then, would wait for a parity that does not come again.
        auto take_turn = [&](int j, int n) {
            const int turn = u == 0 ? n - 1 : n;
            return !(both && j < npre) || turn < 0 || __all_sync(0xffffffffu, mbar_wait(&exp_done[u ^ 1], turn & 1, abort_p)) != 0;
        };
        float m_run = -INFINITY, l_run = 0.f;
        int used = 0;
        for (int j = 0; j < J && ok; ++j) {
            if (!active(u, j)) continue;
            const int st = j % STAGES;
            // the keys of the step that this pair sees: [lo, hi)
            int lo = 0, hi = min(PT_KEYS, prefix - (x0 + j) * PT_KEYS);
            unsigned char* v_row = tiles + v_off(st) + r * 128;            // the values of key r of the step (its 16-byte pieces in the swizzle's order)
            bool valid = j < npre && r < hi;               // key r of the step: is it anybody's?  (key `owned` of the tile's row, of own keys)
            int owned = 0;
            if (j >= npre) {
                const OwnStep o = own_step(j);
                lo = max(0, min(PT_KEYS, seen_lo - o.k * PT_KEYS));
                hi = max(lo, min(PT_KEYS, seen_hi - o.k * PT_KEYS));
                const int slot = (o.list ? list0[1] : 0) + o.k * W + (r >> ss);
                if (slot < (o.list ? list_end[1] : list_end[0])) {
                    owned = owner(slot);
                    const int key = own_begin + ((slot - plan.own_first[owned]) << ss) + (r & (sk - 1));
                    valid = key >= prefix && key < plan.ctx[owned];
                }
            }
#pragma unroll 1
            for (int h = 0; h < HALVES; ++h) {
            const int key0 = h * HK, from = max(0, min(HK, lo - key0)), end = max(from, min(HK, hi - key0)), n = used * HALVES + h;      // (n: halves before this one)
            ok = __all_sync(0xffffffffu, mbar_wait(&s_full[u][h], used & 1, abort_p));
            if (!ok) break;
            tc_fence_after();
            float alpha = 1.f;
            if (__any_sync(0xffffffffu, end > from)) {
                uint32_t sv[HK];
#pragma unroll
                for (int c = 0; c < HK; c += 32) tmem_ld32_async(S_AT + h * HALF + c, sv + c);
#pragma unroll
                for (int c = 0; c < HK; c += 32) tmem_ld_wait(sv + c);
                tc_fence_before();
                __syncwarp();
                if (!OVER && lane == 0) mbar_arrive(&s_free[u]);
                if (__any_sync(0xffffffffu, from > 0 || end < HK)) {
                    const unsigned keys = end - from;
#pragma unroll
                    for (int i = 0; i < HK; ++i) if ((unsigned)(i - from) >= keys) sv[i] = __float_as_uint(-INFINITY);
                }
                // the reference point of the exponent moves only when a score would exceed 2^8 against the one in use
                {
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < HK; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(sv[i]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2e;
                    if (mx > -INFINITY && (m_run == -INFINITY || mx - m_run > 8.0f)) {
                        alpha = m_run == -INFINITY ? 1.f : ex2_approx(m_run - mx);
                        m_run = mx;
                    }
                }
                // (where P lies over S, scores that are here say that the product which read the P before them is done)
                if (!OVER && n > 0 && !__all_sync(0xffffffffu, mbar_wait(&pv_done[u], (n - 1) & 1, abort_p))) { ok = false; break; }
                if (!take_turn(j, n)) { ok = false; break; }
                const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
                float sm[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ch = 0; ch < HK / 32; ++ch) {
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float p0 = ex2_approx(fmaf(__uint_as_float(sv[ch * 32 + i]), p.scale_log2e, neg_m));
                        const float p1 = ex2_approx(fmaf(__uint_as_float(sv[ch * 32 + i + 1]), p.scale_log2e, neg_m));
                        sm[(i >> 1) & 3] += p0 + p1;
                        packed[i >> 1] = pack2_bf16(p0, p1);
                    }
                    tmem_st16(P_AT + h * HALF + ch * 16, packed);
                }
                l_run = l_run * alpha + ((sm[0] + sm[1]) + (sm[2] + sm[3]));
                __syncwarp();
                if (both && j < npre && lane == 0) mbar_arrive(&exp_done[u]);
            } else {                                       // own keys of other warps' rows (of a prefix: none behind its end): weights of zero
                if (!OVER && lane == 0) mbar_arrive(&s_free[u]);
                if (!OVER && n > 0 && !__all_sync(0xffffffffu, mbar_wait(&pv_done[u], (n - 1) & 1, abort_p))) { ok = false; break; }
                if (!take_turn(j, n)) { ok = false; break; }
                if (both && j < npre && lane == 0) mbar_arrive(&exp_done[u]);
                uint32_t none[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) none[i] = 0;
#pragma unroll
                for (int ch = 0; ch < HK / 32; ++ch) tmem_st16(P_AT + h * HALF + ch * 16, none);
            }
            // The values' turn comes behind the weights, under whose making they arrive (before: 5,250 cycles a step of own keys instead of 3,600).
            if (h == 0 && !__all_sync(0xffffffffu, valid && j < npre)) {
                ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (j / STAGES) & 1, abort_p));
                if (!ok) break;
                if (!valid) {                              // nobody's: zeros (of a prefix's last step both chains write the same)
#pragma unroll
                    for (int c = 0; c < 8 * PARTS; ++c) *reinterpret_cast<uint4*>(v_row + (c >> 3) * SUB + ((c ^ r) & 7) * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                } else if (j >= npre) {
                    uint32_t bad = 0;                      // an exponent of all ones carries into its number's highest bit
#pragma unroll
                    for (int c = 0; c < 8 * PARTS; ++c) {
                        const uint4 v = *reinterpret_cast<const uint4*>(v_row + (c >> 3) * SUB + ((c ^ r) & 7) * 16);
                        bad |= ((v.x & 0x7f807f80u) + 0x00800080u) | ((v.y & 0x7f807f80u) + 0x00800080u) | ((v.z & 0x7f807f80u) + 0x00800080u) | ((v.w & 0x7f807f80u) + 0x00800080u);
                    }
                    if (bad & 0x80008000u) {
                        for (int c = 0; c < 8 * PARTS * 4; ++c) {
                            uint32_t* at = reinterpret_cast<uint32_t*>(v_row + (c >> 5) * SUB + (c & 31) * 4);
                            uint32_t x = *at;
                            if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
                            if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
                            *at = x;
                        }
                        wp.marks[(int64_t)(row0 + owned) * p.num_kv_heads + kvh] = G;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                }
            }
            if (n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                if (OVER && !__all_sync(0xffffffffu, mbar_wait(&pv_done[u], (n - 1) & 1, abort_p))) { ok = false; break; }
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    float v[16];
                    tmem_ld16(O_AT + c, v);
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * alpha);
                    tmem_st8(O_AT + c, w);
                    tmem_st8(O_AT + c + 8, w + 8);
                }
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[u][h]);
            }
            if (!ok) break;
            ++used;
        }
        if (ok && used > 0) ok = mbar_wait(&o_full[u], 0, abort_p);
        tc_fence_after();
        __syncwarp();
        if (__all_sync(0xffffffffu, ok)) {
            const float inv = l_run > 0.f ? 1.0f / l_run : l_run == 0.f ? 0.f : NAN;      // a sum that is no number stays none
            const int64_t slot = plan.slot0 + (int64_t)in_tile * per_row + (both ? split : 2 * split + u);
            const bool writes = pair && slot < p.most_slots;       // (the host sizes the scratch memory for every plan)
            if (writes) p.part_lse[slot * p.num_heads + head] = l_run != 0.f ? m_run + __log2f(l_run) : -INFINITY;
            // O goes through shared memory a quarter of its columns at a time, so that a pair's entries leave side by side (written out of the registers, 128 bytes
            // apart a lane, they took 10,000 cycles a block).  The queries' place is free: this chain's, or the half of the unused one.
            constexpr int COLS = D / 4, PIECES = COLS / 4;         // entries and 16-byte pieces of a pass
            float* stage = reinterpret_cast<float*>(tiles + (both ? q_off(u) : q_off(1) + u * (TILE / 2))) + q * 32 * COLS;
            auto piece = [&](int row, int c) { return row * PIECES + (PIECES == 8 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)); };
            const int to = writes && l_run != 0.f ? (int)(slot * p.num_heads + head) : -1;
            if (__any_sync(0xffffffffu, to >= 0)) {
#pragma unroll 1
                for (int pass = 0; pass < 4; ++pass) {
#pragma unroll
                    for (int c = 0; c < COLS; c += 16) {
                        float v[16];
                        tmem_ld16(O_AT + pass * COLS + c, v);
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            *reinterpret_cast<float4*>(stage + piece(lane, (c + i) / 4) * 4) = make_float4(v[i] * inv, v[i + 1] * inv, v[i + 2] * inv, v[i + 3] * inv);
                    }
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < PIECES; ++k) {
                        const int row = k * (32 / PIECES) + lane / PIECES, c = lane % PIECES, dst = __shfl_sync(0xffffffffu, to, row);
                        if (dst >= 0) *reinterpret_cast<float4*>(p.part_o + (int64_t)dst * D + pass * COLS + c * 4) = *reinterpret_cast<const float4*>(stage + piece(row, c) * 4);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
        }
    }

    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        if (threadIdx.x == 0) atomicExch(p.error, 1);
        for (int i = 0; i < 64; ++i) __nanosleep(2000);    // let copies that are still in flight land
    }
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

// Joins the ranges of a row's walk: out = sum_s 2^(L_s - max L) o_s / sum_s 2^(L_s - max L).  A warp a head, a lane D / 32 entries of it.
#define JOIN_WARPS 8
template <int D>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
prefix_join_kernel(const WalkParams wp, bf16* __restrict__ out, float* __restrict__ out32) {
    constexpr int E = D / 32;
    pdl_enter();
    const PrefixParams& p = wp.b;
    const int row = blockIdx.x, lane = threadIdx.x & 31, head = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5);
    const int2 info = __ldcg(wp.row_info + row);
    const int S = min(info.y, 2 * PREFIX_MAX_SPLITS);
    if (p.row_q_len[row] != 1 || head >= p.num_heads) return;      // (a row of more than one new token is left alone)
    const int64_t at = ((int64_t)p.row_q_start[row] * p.num_heads + head) * D + lane * E;
    auto write = [&](const float* acc) {
        if (out32) {
#pragma unroll
            for (int e = 0; e < E; ++e) out32[at + e] = acc[e];
        } else {
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<__nv_bfloat162*>(out + at + e) = __floats2bfloat162_rn(acc[e], acc[e + 1]);
        }
    };
    if (p.row_ctx_len[row] <= 0) {                         // no keys at all: no range may have been planned for the row
        const float none[E] = {};
        write(none);
        return;
    }
    if (S <= 0 || (int64_t)info.x + S > p.most_slots) return;
    const int kvh = head / (p.num_heads / p.num_kv_heads);
    int* mark = wp.marks + (int64_t)row * p.num_kv_heads + kvh;
    const int marked = __ldcg(mark);
    const float* lse = p.part_lse + (int64_t)info.x * p.num_heads + head;
    const float* from = p.part_o + ((int64_t)info.x * p.num_heads + head) * D + lane * E;
    const int64_t step = (int64_t)p.num_heads * D;
    constexpr int WORDS = 2 * PREFIX_MAX_SPLITS / 32;
    float w[WORDS], mm = -INFINITY, sum = 0.f;
#pragma unroll
    for (int h = 0; h < WORDS; ++h) {
        w[h] = h * 32 + lane < S ? __ldcg(lse + (int64_t)(h * 32 + lane) * p.num_heads) : -INFINITY;
        mm = fmaxf(mm, w[h]);
    }
    mm = warp_max(mm);
    const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int h = 0; h < WORDS; ++h) { w[h] = exp2_fast(w[h] - ref); sum += w[h]; }
    sum = warp_sum(sum);
    const float inv = sum > 0.f ? __frcp_rn(sum) : sum == 0.f ? 0.f : sum;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    // results of ranges in which the pair saw no key hold nothing: they are passed over; eight of the others are asked for at a time
#pragma unroll
    for (int h = 0; h < WORDS; ++h) {
        if (h * 32 >= S) break;
        unsigned left = __ballot_sync(0xffffffffu, w[h] != 0.f);
        while (left) {
            float v[8][E], wk[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int l = left ? __ffs(left) - 1 : 0;
                wk[k] = left ? __shfl_sync(0xffffffffu, w[h], l) * inv : 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] = 0.f;
                if (left) {
                    left &= left - 1;
                    const float* src = from + (int64_t)(h * 32 + l) * step;
                    if constexpr (E == 4) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
                        v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
                    } else {
                        const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
                        v[k][0] = x.x; v[k][1] = x.y;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(wk[k], v[k][e], acc[e]);
        }
    }
    if (marked) {                                          // own values that are not finite: each reaches the output as it is (its weight is positive)
        int prefix = 0;
        for (int g = 0; g < p.groups.groups; ++g) {
            const PrefixPart t = prefix_group(p.groups, g);
            if (row >= t.first_row && row < t.first_row + t.rows) { prefix = t.keys; break; }
        }
        const int ctx = min(p.row_ctx_len[row], p.groups.most_keys);
        for (int key = prefix; key < ctx; ++key) {
            const int entry = key >> p.page_shift;
            const int page = checked_page(p.block_tables[(int64_t)row * p.table_stride + entry], p.num_pages, p.report, MIE_K_ATTENTION_PREFIX, entry);
            const bf16* v = p.v_cache + (((int64_t)page * p.num_kv_heads + kvh) * p.page_size + (key & (p.page_size - 1))) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = __bfloat162float(v[e]);
                if (!isfinite(x)) acc[e] += x;
            }
        }
        __syncwarp();
        if (lane == 0) atomicSub(mark, 1);                 // the last of the key head's query heads leaves it 0
    }
    write(acc);
}

static int prefix_map(CUtensorMap* map, const void* ptr, uint64_t rows, int head_dim, int box_rows) {
    cuuint64_t gdim[2] = {(cuuint64_t)head_dim, rows};
    cuuint64_t gstride[1] = {(cuuint64_t)head_dim * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 1000 + (int)r;
}

template <int D>
static int launch_walk(WalkParams p, void* out, bool out_f32, long long items, cudaStream_t stream) {
    int rc = tc_setup();
    if (rc) return rc;
    p.b.error = g_error_dev;
    CUtensorMap mk, mv;
    const uint64_t rows = (uint64_t)p.b.num_pages * p.b.num_kv_heads * p.b.page_size;
    const int box = p.b.page_size < PT_KEYS ? p.b.page_size : PT_KEYS;
    if ((rc = prefix_map(&mk, p.b.k_cache, rows, D, box)) || (rc = prefix_map(&mv, p.b.v_cache, rows, D, box))) return rc;
    static unsigned long long granted = 0;
    if ((rc = grant_shared(prefix_walk_kernel<D>, PT_SMEM<D>, granted))) return rc;
    if ((rc = launch_kernel(prefix_walk_kernel<D>, dim3((unsigned)items), dim3(PT_THREADS), PT_SMEM<D>, stream, mk, mv, p))) return rc;
    return launch_kernel(prefix_join_kernel<D>, dim3(p.b.groups.num_rows, (p.b.num_heads + JOIN_WARPS - 1) / JOIN_WARPS), dim3(JOIN_WARPS * 32), 0, stream, p,
                         out_f32 ? nullptr : (bf16*)out, out_f32 ? (float*)out : nullptr);
}

// The arguments of attention over shared prefixes as the caller keeps them (kernels/ops.py).  How pairs are cut (mie_prefix_layout): chunk_heads query heads
// a unit, `chunks` units a key head, tile_rows rows an item, `places` items side by side, walk 1: the walk above, 0: the kernel for any head size, and
// attention_decode_shared.cu behind it.
#include "prefix_args.cuh"

// Fills in the layout, and most_slots: the most slots of partial results (num_heads x head_dim float32, and num_heads float32) that a launch writes.
// Non-zero: a size that is not taken.
extern "C" int mie_prefix_layout(SharedArgs* a, int sms) {
    if (a->num_rows < 0 || a->num_kv_heads <= 0 || a->num_heads <= 0 || a->num_heads % a->num_kv_heads || a->head_dim < 16 || a->head_dim > 128 || a->head_dim % 16
        || sms <= 0 || a->page_size < 1 || (a->page_size & (a->page_size - 1))) return MIE_ERR_BAD_ARG;
    const int G = a->num_heads / a->num_kv_heads;
    // Few pairs leave the walk's tiles of 128 empty, and it takes longer to begin; what it gains grows with the keys and values that there are.  Us, walk : the other
    // two kernels -- 32 heads of 64 on 4, 8 rows behind 2,048 15.4 : 13.1, 16 16.0 : 14.3, 32 19.6 : 30; 32 on 32, 16 rows behind
    // 3,000 35.9 : 30.2.  Heads of 128, 32 on 8: 16 rows behind 1,000 19.5 : 17.2, behind 4,000 21.2 : 21.6, behind 16,000 35 : 48, 64 behind 8,000 45 : 84;
    // 32 on 32: 8 rows behind 2,000 21.4 : 23.5, 33 rows in five groups 69 : 74.
    const double bytes = 4.0 * a->num_kv_heads * a->head_dim * (a->most_prefix + 0.5 * a->num_rows * a->most_own);
    for (a->walk = a->num_rows * (long long)G > PT_WALK_PAIRS || (a->head_dim == 128 && bytes > PT_WALK_BYTES); a->walk >= 0; --a->walk) {
        const int pairs = a->walk ? PT_ROWS : PFX_PAIRS;
        a->chunks = (G + pairs - 1) / pairs;
        a->chunk_heads = (G + a->chunks - 1) / a->chunks;
        a->tile_rows = pairs / a->chunk_heads * (a->walk ? 2 : 1);
        a->places = a->walk ? sms : 2 * sms;
        if ((a->head_dim == 64 || a->head_dim == 128) && a->page_size >= 8 && a->groups + 2 <= PT_MOST_SEGMENTS
            && (a->num_rows + a->tile_rows - 1) / a->tile_rows + a->groups + 2 <= PT_MOST_TILES) break;
        if (!a->walk) break;
    }
    a->most_slots = prefix_most_slots(a->num_rows, a->num_kv_heads * a->chunks, a->tile_rows, a->places);
    return 0;
}

extern "C" int mie_prefix_attention(const SharedArgs* a, cudaStream_t stream) {
    if (a->num_rows <= 0) return 0;
    if (a->groups <= 0 || (!a->walk && !a->own_keys)) return MIE_ERR_BAD_ARG;
    if (a->num_rows > 65535) return MIE_ERR_TOO_LARGE;
    WalkParams w = {};
    PrefixParams& p = w.b;
    p.q = (const bf16*)a->q; p.q_stride = a->q_stride; p.k_cache = (const bf16*)a->k_cache; p.v_cache = (const bf16*)a->v_cache;
    p.block_tables = a->block_tables; p.table_stride = a->table_stride; p.row_q_start = a->row_q_start; p.row_q_len = a->row_q_len;
    p.part_o = a->pre_o; p.part_lse = a->pre_lse; p.most_slots = a->most_slots; p.chunk = a->pre_chunk;
    p.num_heads = a->num_heads; p.num_kv_heads = a->num_kv_heads; p.page_size = a->page_size;
    while ((1 << p.page_shift) < a->page_size) ++p.page_shift;
    p.chunk_heads = a->chunk_heads; p.chunks = a->chunks;
    p.scale_log2e = a->scale * 1.4426950408889634f;
    p.num_pages = a->num_pages; p.report = g_range_report;
    p.groups = shared_groups_of(*a);
    p.row_ctx_len = a->row_ctx_len;
    w.row_info = (int2*)a->row_info; w.marks = a->marks;
    const long long items = prefix_most_items(a->num_rows, a->walk ? a->groups + 2 : a->groups, p.groups.units, p.groups.tile_rows, p.groups.places);
    if (items > 0x7fffffffll) return MIE_ERR_TOO_LARGE;
    if (a->walk) return a->head_dim == 64 ? launch_walk<64>(w, a->out, a->out_f32 != 0, items, stream) : launch_walk<128>(w, a->out, a->out_f32 != 0, items, stream);
    int rc = MIE_ERR_BAD_ARG;
    switch (a->head_dim) {
        case 16: rc = launch_prefix<16>(p, items, stream); break;
        case 32: rc = launch_prefix<32>(p, items, stream); break;
        case 48: rc = launch_prefix<48>(p, items, stream); break;
        case 64: rc = launch_prefix<64>(p, items, stream); break;
        case 80: rc = launch_prefix<80>(p, items, stream); break;
        case 96: rc = launch_prefix<96>(p, items, stream); break;
        case 112: rc = launch_prefix<112>(p, items, stream); break;
        case 128: rc = launch_prefix<128>(p, items, stream); break;
    }
    return rc ? rc : a->own_keys(a, stream);
}

// Non-zero when a block of any launch so far gave up a bounded wait.
extern "C" int mie_prefix_attention_error(void) { return g_error_host ? *g_error_host : 0; }
extern "C" void mie_prefix_attention_clear_error(void) { if (g_error_host) *g_error_host = 0; }
