// Rules on a row of float32 logits: penalties for tokens that its text holds already, biases on single tokens, and the mask of a grammar.
//
//   x_i' = x_i / rep  (x_i > 0)  or  x_i rep  (otherwise)   for tokens i in the prompt or the answer so far
//   x_i' -= freq count_i + pres [count_i > 0]               count_i: how often i stands in the answer so far
//   x_i' += the biases listed for i, in the list's order
//   x_i' = -inf                                             where the mask's bit i is 0 (whatever stood there: NaN and inf too)
//
// Two forms.  `apply` writes x'.  `choose` writes nothing of that size: it picks the row's token from x' as it passes by (greedy, or with
// temperature by the noise of sampling.cu: argmax x' / t + g) and, where asked, leaves log softmax(x') at that token.
//
// A block owns a slice of a row's vocabulary and keeps one 32-bit word an entry of it in shared memory: a count, a bit "in the prompt", a
// bit "has a bias".  It walks the row's whole text once, counting the tokens that fall into its slice (integer atomics: their order changes nothing),
// marks the biased ones, and then reads its logits, which meet their words there.  An entry marked as biased walks the list for its own
// token, so biases add up in the list's order however often a token is named.  A slice larger than the table takes several turns.
// Choosing: the slices of a row are a thread-block cluster whose first block joins the winners and the sums out of the others' shared
// memory (the maximum of x' and the sum of exp(x' - maximum), in float32, joined pairwise).
//
// Bound: the bytes of the logits (read once, written once by `apply`) for many rows, the chain of text -> table -> logits for few.
#include "choice.cuh"
#include "range_check.cuh"

#define MIE_K_LOGIT_RULES 15       // this kernel's number in the range report (csrc/range_check.cuh)
#define RULES_MAX_THREADS 512
#define RULES_PARTS 8              // slices of a row whose token is chosen: the blocks of a cluster
#define IN_PROMPT 0x80000000u
#define HAS_BIAS 0x40000000u
#define COUNT_BITS 0x3fffffffu

struct RuleParams {
    const float* logits; int64_t logits_stride;
    float* out; int64_t out_stride;                       // apply
    int rows, vocab, table;                               // table: words of shared memory for a slice (or a turn of one)
    const int* history; int64_t history_stride; int slots, width;       // text of every slot, [slots][width]
    const int* slot; const int* prompt_len; const int* total_len;       // of a row: its slot (-1: none), tokens of its prompt, of prompt and answer
    const float* repetition; const float* presence; const float* frequency;      // of a row; null: off
    const int* bias_tokens; const float* bias_values; int bias_width; const int* bias_len;      // [slots][bias_width], used entries of a row's list
    const int* mask; int64_t mask_stride; int masks; const int* mask_row;        // bits [masks][mask_stride words], a row's mask (-1: none)
    int* report;
    // choose
    const float* temperature; const int64_t* request; const int* position; uint64_t seed;
    int* token; float* logprob; int* append;              // append: the slots' text, which takes the token at place total_len (or null)
    int* host_out; const int* host_turn; int host_stride;
};

// A running maximum m and the sum s of exp(x - m): joined with another such pair.  Nothing seen yet: m = -inf, s = 0.
__device__ __forceinline__ void join_sums(float& m, float& s, float om, float os) {
    const float mn = fmaxf(m, om);
    if (mn == -INFINITY) { s += os; return; }             // (both sums are 0, or NaN)
    s = s * __expf(m - mn) + os * __expf(om - mn);
    m = mn;
}

template <bool CHOOSE, bool CLUSTER>
__global__ void __launch_bounds__(RULES_MAX_THREADS)
logit_rules_kernel(const RuleParams p) {
    extern __shared__ uint32_t words[];
    pdl_enter();
    const int row = blockIdx.y, part = blockIdx.x, parts = gridDim.x, T = blockDim.x, tid = threadIdx.x;
    const float* lg = p.logits + (int64_t)row * p.logits_stride;
    float* og = CHOOSE ? nullptr : p.out + (int64_t)row * p.out_stride;
    auto complain = [&](int code, int value) {
        if (part == 0 && tid == 0) range_report(p.report, code, MIE_K_LOGIT_RULES, row, value);
    };
    // ---- what holds for this row
    int slot = p.slot ? p.slot[row] : -1;
    if (slot >= p.slots) { complain(MIE_RANGE_ROW, slot); slot = -1; }
    float rep = 1.f, pres = 0.f, freq = 0.f;
    int total = 0, prompt = 0;
    if (slot >= 0 && p.history) {
        rep = p.repetition ? p.repetition[row] : 1.f;
        pres = p.presence ? p.presence[row] : 0.f;
        freq = p.frequency ? p.frequency[row] : 0.f;
        total = p.total_len[row];
        prompt = p.prompt_len[row];
        if (total < 0 || total > p.width) { complain(MIE_RANGE_POSITION, total); total = total < 0 ? 0 : p.width; }
    }
    const bool text_counts = total > 0 && (rep != 1.f || pres != 0.f || freq != 0.f);
    const int* text = text_counts ? p.history + (int64_t)slot * p.history_stride : nullptr;
    int biases = 0;
    if (slot >= 0 && p.bias_tokens) {
        biases = p.bias_len ? p.bias_len[row] : p.bias_width;
        if (biases < 0 || biases > p.bias_width) { complain(MIE_RANGE_POSITION, biases); biases = biases < 0 ? 0 : p.bias_width; }
    }
    const int* bias_tokens = biases ? p.bias_tokens + (int64_t)slot * p.bias_width : nullptr;
    const float* bias_values = biases ? p.bias_values + (int64_t)slot * p.bias_width : nullptr;
    int mask_row = p.mask && p.mask_row ? p.mask_row[row] : -1;
    if (mask_row >= p.masks) { complain(MIE_RANGE_ROW, mask_row); mask_row = -1; }
    const int* mask = mask_row >= 0 ? p.mask + (int64_t)mask_row * p.mask_stride : nullptr;
    const int last_word = (p.vocab - 1) >> 5;
    const bool marked = text_counts || biases > 0;        // some entries have words

    float temperature = 0.f;
    uint64_t key = 0;
    if (CHOOSE) {
        temperature = p.temperature[row];
        if (temperature > 0.f) key = noise_key(p.seed, p.request[row], p.position[row]);
    }
    float bv = -INFINITY, bx = -INFINITY, m = -INFINITY, s = 0.f;       // the winner's score, its logit; the running maximum and sum
    int bi = 0x7fffffff;

    // ---- this block's slice.  Slices begin where the row's 16-byte groups do (`off` entries before the row's first whole group).
    const int off = (int)((4 - ((reinterpret_cast<uintptr_t>(lg) >> 2) & 3)) & 3);
    const bool wide = CHOOSE || ((reinterpret_cast<uintptr_t>(lg) ^ reinterpret_cast<uintptr_t>(og)) & 15) == 0;      // 16-byte groups of the output too
    const int per = ((p.vocab + parts - 1) / parts + 3) & ~3;
    const int64_t lo64 = part ? (int64_t)part * per + off : 0, hi64 = (int64_t)(part + 1) * per + off;
    const int lo = (int)min((int64_t)p.vocab, lo64), hi = part + 1 == parts ? p.vocab : (int)min((int64_t)p.vocab, hi64);

    for (int c0 = lo; c0 < hi; ) {
        const int c1 = marked ? min(hi, c0 == 0 ? off + p.table - 4 : c0 + p.table) : hi;      // (a first turn is shorter, so that the next begins on a group)
        if (marked) {
            __syncthreads();                              // the turn before is done with the words
            for (int i = tid; i < c1 - c0; i += T) words[i] = 0;
            __syncthreads();
            if (text_counts) {
                for (int j = tid; j < total; j += T) {
                    const int t = text[j];
                    if (t >= c0 && t < c1) {
                        if (j < prompt) atomicOr(&words[t - c0], IN_PROMPT);
                        else atomicAdd(&words[t - c0], 1u);
                    } else if (c0 == 0 && (t < 0 || t >= p.vocab)) {
                        range_report(p.report, MIE_RANGE_TOKEN, MIE_K_LOGIT_RULES, row, t);
                    }
                }
            }
            for (int j = tid; j < biases; j += T) {
                const int t = bias_tokens[j];
                if (t >= c0 && t < c1) atomicOr(&words[t - c0], HAS_BIAS);
                else if (c0 == 0 && (t < 0 || t >= p.vocab)) range_report(p.report, MIE_RANGE_TOKEN, MIE_K_LOGIT_RULES, row, t);
            }
            __syncthreads();
        }
        auto ruled = [&](float x, int i, bool allowed) {
            if (marked) {
                const uint32_t w = words[i - c0];
                if (w) {
                    const uint32_t count = w & COUNT_BITS;
                    if (count | (w & IN_PROMPT)) x = x > 0.f ? x / rep : x * rep;
                    if (count) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)count), pres));
                    if (w & HAS_BIAS) for (int j = 0; j < biases; ++j) if (bias_tokens[j] == i) x = __fadd_rn(x, bias_values[j]);
                }
            }
            return allowed ? x : -INFINITY;
        };
        auto consider = [&](float x, int i) {
            const float v = temperature > 0.f ? noisy_score(x, temperature, key, i) : x;
            if (v > bv || (v == bv && i < bi)) { bv = v; bi = i; bx = x; }
        };
        auto one = [&](int i) {
            const float x = ruled(lg[i], i, !mask || ((mask[i >> 5] >> (i & 31)) & 1));
            if (CHOOSE) {
                consider(x, i);
                if (p.logprob) join_sums(m, s, x, x == -INFINITY ? 0.f : x != x ? NAN : 1.f);
            } else og[i] = x;
        };
        const int first = min(c1, c0 == 0 ? off : c0);    // whole groups from here on
        const int groups = wide ? (c1 - first) >> 2 : 0;
        for (int i = c0 + tid; i < first; i += T) one(i);
        for (int i = first + groups * 4 + tid; i < c1; i += T) one(i);
        constexpr int AHEAD = 4;                          // groups that a thread asks for before it works on the first
        for (int g0 = tid; g0 < groups; g0 += AHEAD * T) {
            float4 x4[AHEAD];
            uint32_t bits[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int g = g0 + u * T, i = first + g * 4;
                bits[u] = 0xffffffffu;
                if (g < groups) {
                    x4[u] = __ldcs(reinterpret_cast<const float4*>(lg + i));
                    if (mask) {
                        const int w = i >> 5;
                        bits[u] = __funnelshift_r((uint32_t)mask[w], (uint32_t)mask[min(w + 1, last_word)], i & 31);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int g = g0 + u * T, i = first + g * 4;
                if (g >= groups) continue;
                float x[4] = {x4[u].x, x4[u].y, x4[u].z, x4[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = ruled(x[e], i + e, (bits[u] >> e) & 1);
                if (CHOOSE) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) consider(x[e], i + e);
                    if (p.logprob) {
                        const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        if (mx > m) { s *= __expf(m - mx); m = mx; }
                        if (m > -INFINITY) s += (__expf(x[0] - m) + __expf(x[1] - m)) + (__expf(x[2] - m) + __expf(x[3] - m));
                        else s += (x[0] + x[1]) + (x[2] + x[3]) == -INFINITY ? 0.f : NAN;       // nothing but -inf and NaN so far
                    }
                } else {
                    __stcs(reinterpret_cast<float4*>(og + i), make_float4(x[0], x[1], x[2], x[3]));
                }
            }
        }
        c0 = c1;
    }
    if (!CHOOSE) return;

    // ---- the block's winner and sums, then the row's
    __shared__ float w_v[RULES_MAX_THREADS / 32], w_x[RULES_MAX_THREADS / 32], w_m[RULES_MAX_THREADS / 32], w_s[RULES_MAX_THREADS / 32];
    __shared__ int w_i[RULES_MAX_THREADS / 32];
    __shared__ float part_v, part_x, part_m, part_s;
    __shared__ int part_i;
    auto reduce_warp = [&]() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o), ox = __shfl_xor_sync(0xffffffffu, bx, o);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; bx = ox; }
            const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
            join_sums(m, s, om, os);
        }
    };
    const int lane = tid & 31, warp = tid >> 5;
    reduce_warp();
    if (lane == 0) { w_v[warp] = bv; w_x[warp] = bx; w_i[warp] = bi; w_m[warp] = m; w_s[warp] = s; }
    __syncthreads();
    if (warp == 0) {
        const bool on = lane < T / 32;
        bv = on ? w_v[lane] : -INFINITY; bx = on ? w_x[lane] : -INFINITY; bi = on ? w_i[lane] : 0x7fffffff;
        m = on ? w_m[lane] : -INFINITY; s = on ? w_s[lane] : 0.f;
        reduce_warp();
        if (lane == 0) { part_v = bv; part_x = bx; part_i = bi; part_m = m; part_s = s; }
    }
    auto finish = [&]() {
        const int tok = bi < p.vocab ? bi : 0;            // nothing but -inf (entry 0 wins that tie) or NaN
        p.token[row] = tok;
        if (p.logprob) p.logprob[row] = m == -INFINITY && s == 0.f ? -INFINITY : (bx - m) - logf(s);
        if (p.append && slot >= 0 && total < p.width) p.append[(int64_t)slot * p.history_stride + total] = tok;
        if (p.host_out) p.host_out[(p.host_turn ? *p.host_turn : 0) * p.host_stride + row] = tok;
    };
    if (!CLUSTER) {
        if (tid == 0) finish();
        return;
    }
    cluster_sync_all();                                   // every slice's share is in its block's shared memory
    if (part == 0 && warp == 0) {
        bv = -INFINITY; bx = -INFINITY; bi = 0x7fffffff; m = -INFINITY; s = 0.f;
        if (lane < parts) {
            auto of = [&](const void* at) { return ld_cluster_f32(cluster_addr((uint32_t)__cvta_generic_to_shared(at), lane)); };
            bv = of(&part_v); bx = of(&part_x); bi = __float_as_int(of(&part_i)); m = of(&part_m); s = of(&part_s);
        }
        reduce_warp();
        if (lane == 0) finish();
    }
    cluster_sync_all();                                   // nobody leaves while its shared memory is being read
}

static int launch_rules(RuleParams& p, bool choose, int parts, cudaStream_t stream) {
    if (p.rows <= 0) return 0;
    if (p.vocab <= 0 || p.slots < 0 || p.width < 0 || p.bias_width < 0 || p.masks < 0) return MIE_ERR_BAD_ARG;
    if (p.rows > 65535 || p.width > (int)COUNT_BITS) return MIE_ERR_TOO_LARGE;
    if ((p.history || p.bias_tokens) && !p.slot) return MIE_ERR_BAD_ARG;
    if (p.history && (!p.total_len || !p.prompt_len)) return MIE_ERR_BAD_ARG;
    if (p.bias_tokens && !p.bias_values) return MIE_ERR_BAD_ARG;
    if (p.mask && p.mask_stride < (p.vocab + 31) / 32) return MIE_ERR_BAD_ARG;
    const int per = ((p.vocab + parts - 1) / parts + 3) & ~3;
    p.table = per + 4 < 16384 ? per + 4 : 16384;
    const size_t smem = p.history || p.bias_tokens ? (size_t)p.table * 4 : 0;
    const dim3 grid(parts, p.rows), block(per > 8192 ? 512 : 256);
    auto kernel = !choose ? logit_rules_kernel<false, false> : parts > 1 ? logit_rules_kernel<true, true> : logit_rules_kernel<true, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 16384 * 4);
    if (e != cudaSuccess) return (int)e;
    return launch_kernel_cluster(kernel, grid, block, smem, stream, dim3(choose ? parts : 1, 1, 1), p);
}

static void set_rules(RuleParams& p, const int* history, int64_t history_stride, int slots, int width, const int* slot, const int* prompt_len,
                      const int* total_len, const float* repetition, const float* presence, const float* frequency, const int* bias_tokens,
                      const float* bias_values, int bias_width, const int* bias_len, const int* mask, int64_t mask_stride, int masks, const int* mask_row) {
    p.history = history; p.history_stride = history_stride; p.slots = slots; p.width = width;
    p.slot = slot; p.prompt_len = prompt_len; p.total_len = total_len;
    p.repetition = repetition; p.presence = presence; p.frequency = frequency;
    p.bias_tokens = bias_tokens; p.bias_values = bias_values; p.bias_width = bias_width; p.bias_len = bias_len;
    p.mask = mask; p.mask_stride = mask_stride; p.masks = masks; p.mask_row = mask_row;
    p.report = g_range_report;
}

#define RULE_ARGS const int* history, int64_t history_stride, int slots, int width, const int* slot, const int* prompt_len, const int* total_len,             \
                  const float* repetition, const float* presence, const float* frequency, const int* bias_tokens, const float* bias_values, int bias_width,   \
                  const int* bias_len, const int* mask, int64_t mask_stride, int masks, const int* mask_row
#define RULE_NAMES history, history_stride, slots, width, slot, prompt_len, total_len, repetition, presence, frequency, bias_tokens, bias_values, bias_width, \
                   bias_len, mask, mask_stride, masks, mask_row

// out[r] = the logits of row r under its rules (out may be the logits).  `parts`: blocks a row.
extern "C" int mie_apply_logit_rules(RULE_ARGS, const float* logits, int64_t logits_stride, float* out, int64_t out_stride, int rows, int vocab, int parts,
                                     cudaStream_t stream) {
    RuleParams p = {};
    set_rules(p, RULE_NAMES);
    p.logits = logits; p.logits_stride = logits_stride; p.out = out; p.out_stride = out_stride; p.rows = rows; p.vocab = vocab;
    if (parts < 1 || (rows > 0 && !out)) return MIE_ERR_BAD_ARG;
    return launch_rules(p, false, parts, stream);
}

// The token of every row under its rules; see mie_sample (sampling.cu) for the noise and the host's copy.  `logprob` (or null): log softmax of the
// ruled logits at the token, -inf where the rules leave nothing (the token is 0 there).  `append` (or null, else the history): the token
// joins the row's text.
extern "C" int mie_sample_rules(RULE_ARGS, const float* logits, int64_t logits_stride, const float* temperature, const int64_t* request, const int* position,
                                uint64_t seed, int* token, float* logprob, int* append, int rows, int vocab, int* host_out, const int* host_turn,
                                int host_stride, cudaStream_t stream) {
    RuleParams p = {};
    set_rules(p, RULE_NAMES);
    p.logits = logits; p.logits_stride = logits_stride; p.rows = rows; p.vocab = vocab;
    p.temperature = temperature; p.request = request; p.position = position; p.seed = seed;
    p.token = token; p.logprob = logprob; p.append = append; p.host_out = host_out; p.host_turn = host_turn; p.host_stride = host_stride;
    return launch_rules(p, true, vocab < 4096 ? 1 : RULES_PARTS, stream);
}
