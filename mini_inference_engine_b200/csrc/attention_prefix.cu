// Attention of decoding rows over keys that they share: every (row, query head) pair of a group against the group's prefix, computed once for
// all rows, in bfloat16 with float32 scores, softmax statistics and sums.  Leaves, for a pair and a range of the prefix,
//     o = sum_j 2^(s_j - m) v_j / l   and   m + log2 l,     l = sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j
// which the kernel for the rows' own keys (attention_decode_shared.cu) joins with its own.  prefix_plan.cuh says how the work is cut.
//
// Two kernels.  Heads of 64 and 128 on pages of 8 positions or more: tcgen05, below.  Any head size in steps of 16: a block takes 64 pairs, 16 a warp
// (mma.sync m16n8k16), and walks its range of keys in tiles of 64 that arrive by cp.async, two in flight; a tile serves all 64 pairs.
#include "mma_common.cuh"
#include "tcgen05_common.cuh"
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
    load_tile(0, 0);                                       // the prefix is older than the step: before the wait
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

template <int D>
static int launch_prefix(const PrefixParams& p, long long items, cudaStream_t stream) {
    const size_t smem = (size_t)4 * PFX_TILE * (D + 8) * sizeof(bf16);
    cudaError_t e = cudaFuncSetAttribute(prefix_attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return launch_kernel(prefix_attention_kernel<D>, dim3((unsigned)items), dim3(PFX_WARPS * 32), smem, stream, p);
}

// --------------------------------------------------------------------------- heads of 64 and 128: tcgen05
//
// A block holds up to 256 pairs as two tiles of 128 (one pair a tensor-memory lane) and walks its keys in tiles of 128 that TMA brings a page a copy; a
// tile of keys and values serves both tiles of pairs.  Two groups of four softmax warps, one a tile of pairs, and a thread that issues for each: while a
// group takes its scores through the softmax the tensor pipe works on the other's products.
//   S_u = Q_u K^T into tensor memory; the group's threads move their rows of S into registers, write P = 2^(s - m), rounded to bfloat16, back, and
//   O_u += P_u V with P as the left operand out of tensor memory and V as it lies.
// Tensor memory: heads of 64 S 2 x 128 columns, P 2 x 64, O 2 x 64; S of the next tile is issued as soon as the rows are in registers.  Heads of 128: O takes
// 2 x 128, and P lies over the S that it came from, so that S of the next tile is issued behind this tile's product with the values.
// Queries are fetched by the threads whose rows they are (any rows, any stride) and written to shared memory as the products want them; the first keys are on
// their way before the wait for the kernel in front (the prefix is older than the step).
#define PT_THREADS 352
#define PT_ROWS 128
#define PT_KEYS 128

template <int D> constexpr int PT_STAGES = D == 64 ? 4 : 2;
template <int D> constexpr size_t PT_SMEM = (size_t)PT_ROWS * D * 2 * 2 + (size_t)PT_STAGES<D> * 2 * PT_KEYS * D * 2 + 1024;

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 1)
prefix_attention_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixParams p) {
    constexpr int PARTS = D / 64, STAGES = PT_STAGES<D>;
    constexpr uint32_t SUB = 128 * 64 * 2;                 // one [128 x 64] part of a tile
    constexpr uint32_t TILE = PARTS * SUB;
    constexpr bool OVER = D == 128;                        // P lies over S
    constexpr uint32_t TMEM_S = 0, TMEM_P = OVER ? 0 : 256, TMEM_O = OVER ? 256 : 384, S_STEP = 128, P_STEP = OVER ? 128 : 64, O_STEP = D;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t q_full[2], kv_full[STAGES], kv_empty[STAGES], s_full[2], s_free[2], p_full[2], pv_done[2], o_full[2], exp_done[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ PrefixPart s_part;
    __shared__ int s_chunk;
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char* tiles = smem_dyn + (base - smem_u32(smem_dyn));
    auto q_off = [&](int u) { return (uint32_t)u * TILE; };
    auto k_off = [&](int st) { return 2 * TILE + (uint32_t)st * 2 * TILE; };
    auto v_off = [&](int st) { return 2 * TILE + (uint32_t)st * 2 * TILE + TILE; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
    const int half = p.groups.tile_rows / 2;               // rows of a tile of pairs
    const int row0 = t.first_row + tile * p.groups.tile_rows, rows = min(p.groups.tile_rows, t.first_row + t.rows - row0);
    const int nsub = rows > half ? 2 : 1;
    int step0, steps;
    prefix_range(t.steps, t.splits, split, step0, steps);
    const int key_lo = step0 * PREFIX_STEP, key_hi = min(t.keys, (step0 + steps) * PREFIX_STEP);
    const int J = (key_hi - key_lo + PT_KEYS - 1) / PT_KEYS;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int u = 0; u < 2; ++u) {
            mbar_init(&q_full[u], 4); mbar_init(&s_full[u], 1); mbar_init(&s_free[u], 4); mbar_init(&p_full[u], 4);
            mbar_init(&pv_done[u], 1); mbar_init(&o_full[u], 1); mbar_init(&exp_done[u], 4);
        }
        for (int st = 0; st < STAGES; ++st) { mbar_init(&kv_full[st], 1); mbar_init(&kv_empty[st], nsub); }      // every issuing thread gives a stage back
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    volatile int* abort_p = &abort_flag;
    // ---- the keys and values (warp 0): lane c copies page c of a tile
    const int* table = p.block_tables + (int64_t)t.first_row * p.table_stride;           // the prefix lies where the group's first row says
    const int rows_per_copy = min(p.page_size, PT_KEYS);
    auto copies_of = [&](int j) { return (min(key_lo + (j + 1) * PT_KEYS, key_hi) - (key_lo + j * PT_KEYS) + rows_per_copy - 1) / rows_per_copy; };
    auto page_of = [&](int j) {
        if (j >= J || lane >= copies_of(j)) return 0;
        const int entry = (key_lo + j * PT_KEYS + lane * rows_per_copy) >> p.page_shift;
        return checked_page(table[entry], p.num_pages, p.report, MIE_K_ATTENTION_PREFIX, entry);
    };
    auto load_tile = [&](int j, int st, int page) {
        const int copies = copies_of(j);
        if (lane == 0) mbar_expect_tx(&kv_full[st], (uint32_t)copies * rows_per_copy * 128u * PARTS * 2u);
        __syncwarp();
        if (lane < copies) {
            const int key = key_lo + j * PT_KEYS + lane * rows_per_copy;
            const int src_row = (page * p.num_kv_heads + kvh) * p.page_size + (key & (p.page_size - 1));
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint32_t off = part * SUB + (uint32_t)lane * rows_per_copy * 128u;
                tma_load_2d(tiles + k_off(st) + off, &map_k, &kv_full[st], part * 64, src_row);
                tma_load_2d(tiles + v_off(st) + off, &map_v, &kv_full[st], part * 64, src_row);
            }
        }
    };
    const int ahead = min(STAGES, J);
    if (warp == 0) {
        int pages[STAGES];
#pragma unroll
        for (int j = 0; j < STAGES; ++j) pages[j] = page_of(j);
#pragma unroll
        for (int j = 0; j < STAGES; ++j) if (j < ahead) load_tile(j, j, pages[j]);
    }
    // Tensor memory is taken behind the wait, and the next kernel let in behind that: a block that held it before the kernels in front are done could keep
    // it from a block of theirs, and one that came later from this one.
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.chunk = s_chunk;
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem_base = tmem_base_slot;

    if (warp == 0) {
        // the rest of the tiles, their pages looked up a tile ahead
        int page_next = page_of(ahead);
        for (int j = ahead; j < J; ++j) {
            const int st = j % STAGES, round = j / STAGES, page = page_next;
            page_next = page_of(j + 1);
            int ok = 1;
            if (lane == 0) ok = mbar_wait(&kv_empty[st], (round & 1) ^ 1, abort_p) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            load_tile(j, st, page);
        }
    } else if (warp == 1 || warp == 10) {
        const int mu = warp == 1 ? 0 : 1;
        if (lane == 0 && mu < nsub) {
            // ---- the thread that issues for group mu
            const uint32_t idesc_s = umma_idesc_bf16(PT_ROWS, PT_KEYS), idesc_o = umma_idesc_bf16(PT_ROWS, D) | (1u << 16);
            constexpr int KS = D / 16, KV = PT_KEYS / 16;
            uint64_t dq[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dq[ks] = umma_desc_sw128(base + q_off(mu) + (ks / 4) * SUB + (ks % 4) * 32);
            const uint64_t dk0 = umma_desc_sw128(base + k_off(0)), dv0 = umma_desc_sw128_mn(base + v_off(0), SUB);
            constexpr uint64_t STAGE_STEP = (2 * TILE) >> 4;       // descriptors of another stage differ in the address field only
            const uint32_t s_at = tmem_base + TMEM_S + S_STEP * mu, p_at = tmem_base + TMEM_P + P_STEP * mu, o_at = tmem_base + TMEM_O + O_STEP * mu;
            auto issue_s = [&](int st) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    umma_bf16(s_at, dq[ks], dk0 + STAGE_STEP * st + (uint64_t)(((ks / 4) * SUB + (ks % 4) * 32) >> 4), idesc_s, ks > 0 ? 1u : 0u);
                umma_commit(&s_full[mu]);
            };
            bool ok = mbar_wait(&q_full[mu], 0, abort_p);
            if (ok) ok = mbar_wait(&kv_full[0], 0, abort_p);
            if (ok) { tc_fence_after(); issue_s(0); }
            int st = 0, round = 0;
            for (int j = 0; j < J && ok; ++j) {
                const int st_next = st + 1 == STAGES ? 0 : st + 1, round_next = st + 1 == STAGES ? round + 1 : round;
                if (!OVER && j + 1 < J) {                  // the next scores, as soon as the rows of these are in registers
                    ok = mbar_wait(&s_free[mu], j & 1, abort_p) && mbar_wait(&kv_full[st_next], round_next & 1, abort_p);
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(st_next);
                }
                ok = mbar_wait(&p_full[mu], j & 1, abort_p);       // P(j) is written, O rescaled
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < KV; ++kk)
                    umma_bf16_ts(o_at, p_at + kk * 8, dv0 + STAGE_STEP * st + (uint64_t)((kk * 2048) >> 4), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
                umma_commit(&pv_done[mu]);                 // P may be overwritten, O rescaled
                if (j + 1 == J) umma_commit(&o_full[mu]);
                umma_commit(&kv_empty[st]);
                if (OVER && j + 1 < J) {                   // (products run in the order they were issued: P has been read when S overwrites it)
                    ok = mbar_wait(&kv_full[st_next], round_next & 1, abort_p);
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(st_next);
                }
                st = st_next; round = round_next;
            }
        }
        __syncwarp();
    } else {
        // ---- softmax group u = 0 (warps 2..5) or 1 (warps 6..9): a thread a pair
        const int u = warp >= 6 ? 1 : 0, q = warp & 3, r = q * 32 + lane;      // (the lanes of tensor memory that a warp reaches go by its number)
        const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16);
        const uint32_t S_AT = lane_addr + TMEM_S + S_STEP * u, P_AT = lane_addr + TMEM_P + P_STEP * u, O_AT = lane_addr + TMEM_O + O_STEP * u;
        bool ok = true;
        if (u < nsub) {
            const int in_tile = r / heads, my_row = row0 + u * half + in_tile, head = kvh * G + h0 + r - in_tile * heads;
            const bool pair = in_tile < half && u * half + in_tile < rows;
            {
                const bf16* src = pair && p.row_q_len[my_row] == 1 ? p.q + (int64_t)p.row_q_start[my_row] * p.q_stride + (int64_t)head * D : nullptr;
                uint4 v[D / 8];
#pragma unroll
                for (int i = 0; i < D / 8; ++i) v[i] = src ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *reinterpret_cast<uint4*>(tiles + q_off(u) + (i >> 3) * SUB + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = v[i];
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[u]);
            }
            float m_run = -INFINITY, l_run = 0.f;
            for (int j = 0; j < J && ok; ++j) {
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[u], j & 1, abort_p));
                if (!ok) break;
                tc_fence_after();
                const int left = key_hi - (key_lo + j * PT_KEYS);      // keys of the tile that there are
                uint32_t sv[128];
                tmem_ld32_async(S_AT, sv);
                tmem_ld32_async(S_AT + 32, sv + 32);
                tmem_ld32_async(S_AT + 64, sv + 64);
                tmem_ld32_async(S_AT + 96, sv + 96);
                if (left < PT_KEYS && r >= left) {         // values of keys that there are not (their weights are 0, and 0 * NaN is NaN): both groups write the same zeros
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4*>(tiles + v_off(j % STAGES) + part * SUB + r * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                tmem_ld_wait(sv); tmem_ld_wait(sv + 32); tmem_ld_wait(sv + 64); tmem_ld_wait(sv + 96);
                tc_fence_before();
                __syncwarp();
                if (!OVER && lane == 0) mbar_arrive(&s_free[u]);
                if (left < PT_KEYS) {
#pragma unroll
                    for (int i = 0; i < 128; ++i) if (i >= left) sv[i] = __float_as_uint(-INFINITY);
                }
                // the reference point of the exponent moves only when a score would exceed 2^8 against the one in use
                float alpha = 1.f, sum;
                {
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 128; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(sv[i]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2e;
                    if (mx > -INFINITY && (m_run == -INFINITY || mx - m_run > 8.0f)) {
                        alpha = m_run == -INFINITY ? 1.f : ex2_approx(m_run - mx);
                        m_run = mx;
                    }
                }
                if (j > 0 && !__all_sync(0xffffffffu, mbar_wait(&pv_done[u], (j - 1) & 1, abort_p))) { ok = false; break; }
                if (nsub == 2) {                           // the groups take turns at the exponentials
                    const int turn = u == 0 ? j - 1 : j;
                    if (turn >= 0 && !__all_sync(0xffffffffu, mbar_wait(&exp_done[u ^ 1], turn & 1, abort_p))) { ok = false; break; }
                }
                {
                    const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
                    float sm[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ch = 0; ch < 4; ++ch) {
                        uint32_t packed[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float p0 = ex2_approx(fmaf(__uint_as_float(sv[ch * 32 + i]), p.scale_log2e, neg_m));
                            const float p1 = ex2_approx(fmaf(__uint_as_float(sv[ch * 32 + i + 1]), p.scale_log2e, neg_m));
                            sm[(i >> 1) & 3] += p0 + p1;
                            packed[i >> 1] = pack2_bf16(p0, p1);
                        }
                        tmem_st16(P_AT + ch * 16, packed);
                    }
                    sum = (sm[0] + sm[1]) + (sm[2] + sm[3]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&exp_done[u]);
                l_run = l_run * alpha + sum;
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
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
                if (lane == 0) mbar_arrive(&p_full[u]);
            }
            if (ok) ok = mbar_wait(&o_full[u], 0, abort_p);
            tc_fence_after();
            __syncwarp();
            if (__all_sync(0xffffffffu, ok)) {
                const float inv = l_run > 0.f ? 1.0f / l_run : l_run == 0.f ? 0.f : NAN;      // a sum that is no number stays none
                const int64_t slot = t.slot0 + (int64_t)(my_row - t.first_row) * t.splits + split;
                const bool writes = pair && slot < p.most_slots;       // (the host sizes the scratch memory for every plan)
                float* op = p.part_o + (slot * p.num_heads + head) * D;
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    float v[16];
                    tmem_ld16(O_AT + c, v);
                    if (!writes) continue;
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4*>(op + c + i) = make_float4(v[i] * inv, v[i + 1] * inv, v[i + 2] * inv, v[i + 3] * inv);
                }
                if (writes) p.part_lse[slot * p.num_heads + head] = l_run != 0.f ? m_run + __log2f(l_run) : -INFINITY;
                tc_fence_before();
            }
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

static int prefix_map(CUtensorMap* map, const void* ptr, uint64_t rows, int head_dim, int box_rows) {
    cuuint64_t gdim[2] = {(cuuint64_t)head_dim, rows};
    cuuint64_t gstride[1] = {(cuuint64_t)head_dim * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 1000 + (int)r;
}

template <int D>
static int launch_prefix_tc(PrefixParams p, long long items, cudaStream_t stream) {
    int rc = tc_setup();
    if (rc) return rc;
    p.error = g_error_dev;
    CUtensorMap mk, mv;
    const uint64_t rows = (uint64_t)p.num_pages * p.num_kv_heads * p.page_size;
    const int box = p.page_size < PT_KEYS ? p.page_size : PT_KEYS;
    if ((rc = prefix_map(&mk, p.k_cache, rows, D, box)) || (rc = prefix_map(&mv, p.v_cache, rows, D, box))) return rc;
    const cudaError_t e = cudaFuncSetAttribute(prefix_attention_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PT_SMEM<D>);
    if (e != cudaSuccess) return (int)e;
    return launch_kernel(prefix_attention_tc_kernel<D>, dim3((unsigned)items), dim3(PT_THREADS), PT_SMEM<D>, stream, mk, mv, p);
}

// How a launch on `sms` SMs cuts (row, head) pairs: out[0] query heads a unit, out[1] units a key head, out[2] rows an item, out[3] items side by side,
// out[4] 1: the tcgen05 kernel (heads of 64 and 128, pages of 8 positions or more), 0: the other.  Also the most slots (rows of num_heads x head_dim
// float32, and num_heads float32) that it writes, as the return value; -1: a size it does not take.
extern "C" long long mie_prefix_layout(int num_rows, int num_heads, int num_kv_heads, int head_dim, int page_size, int sms, int* out) {
    if (num_rows < 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads || head_dim < 16 || head_dim > 128 || head_dim % 16 || sms <= 0) return -1;
    const int G = num_heads / num_kv_heads, tc = (head_dim == 64 || head_dim == 128) && page_size >= 8, pairs = tc ? PT_ROWS : PFX_PAIRS;
    out[1] = (G + pairs - 1) / pairs;
    out[0] = (G + out[1] - 1) / out[1];
    out[2] = pairs / out[0] * (tc ? 2 : 1);
    out[3] = tc ? sms : 2 * sms;
    out[4] = tc;
    return prefix_most_slots(num_rows, num_kv_heads * out[1], out[2], out[3]);
}

extern "C" int mie_prefix_attention(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, const int* block_tables, int table_stride,
                                    const int* row_q_start, const int* row_q_len, int num_rows, const int* group_start, const int* group_prefix, int groups,
                                    int num_heads, int num_kv_heads, int head_dim, int page_size, float scale, const int* layout, float* part_o,
                                    float* part_lse, int* chunk, long long most_slots, long long num_pages, cudaStream_t stream) {
    if (num_rows <= 0 || groups <= 0) return 0;
    if (num_kv_heads <= 0 || num_heads % num_kv_heads) return MIE_ERR_BAD_ARG;
    if (page_size < 1 || (page_size & (page_size - 1))) return MIE_ERR_BAD_ARG;
    PrefixParams p = {};
    p.q = (const bf16*)q; p.q_stride = q_stride; p.k_cache = (const bf16*)k_cache; p.v_cache = (const bf16*)v_cache;
    p.block_tables = block_tables; p.table_stride = table_stride; p.row_q_start = row_q_start; p.row_q_len = row_q_len;
    p.part_o = part_o; p.part_lse = part_lse; p.most_slots = most_slots; p.chunk = chunk;
    p.num_heads = num_heads; p.num_kv_heads = num_kv_heads; p.page_size = page_size;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.chunk_heads = layout[0]; p.chunks = layout[1];
    p.scale_log2e = scale * 1.4426950408889634f;
    p.num_pages = num_pages; p.report = g_range_report;
    const int64_t covered = (int64_t)table_stride * page_size;
    p.groups = PrefixGroups{group_start, group_prefix, groups, num_rows, (int)(covered < 0x7fffff00ll ? covered : 0x7fffff00ll), num_kv_heads * layout[1], layout[2], layout[3]};
    const long long items = prefix_most_items(num_rows, groups, p.groups.units, p.groups.tile_rows, p.groups.places);
    if (items > 0x7fffffffll) return MIE_ERR_TOO_LARGE;
    if (layout[4]) return head_dim == 64 ? launch_prefix_tc<64>(p, items, stream) : launch_prefix_tc<128>(p, items, stream);
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

// Non-zero when a block of any launch so far gave up a bounded wait.
extern "C" int mie_prefix_attention_error(void) { return g_error_host ? *g_error_host : 0; }
extern "C" void mie_prefix_attention_clear_error(void) { if (g_error_host) *g_error_host = 0; }
