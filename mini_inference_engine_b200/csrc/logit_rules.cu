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
// A block owns a slice of a row's vocabulary and keeps a word an entry of it in shared memory: a count, a bit "in the prompt", a bit "has a
// bias"; 16 bits for texts of up to 16,383 tokens, 32 for longer ones.  It walks the row's whole text once, counting the tokens that fall into its
// slice (integer atomics: their order changes nothing), marks the biased ones, and then reads its logits; entries with a word are passed over
// (choose) or written as they are (apply).  They are settled afterwards, thread by token: the text is walked again, and the first thread to take an
// entry's word applies the penalties; an entry of the biases' list belongs to the first that names it, which adds up all of them in the list's
// order.  (Penalties worked out where the logits pass by: some lane of nearly every warp met a marked entry, and the warp went through the divisions of all
// four of its group; 256 rows of 128,256 entries on texts of up to 8,000 tokens 97 us.)  A slice larger than the table takes several turns.
// Which thread takes an entry differs from run to run, and the same call is to give the same bits: the settled entries of a round (4 tokens a thread) are
// summed as integers, relative to the round's greatest, which no order changes (34.9 us for the choice of 200 rows; each thread to its own sum 32.6).
// Choosing: the slices of a row are a thread-block cluster whose first block joins the winners and the sums that the others write into its shared
// memory (the maximum of x' and the sum of exp(x' - maximum), in float32, joined pairwise).
//
// Bound: the bytes of the logits (read once, written once by `apply`) for many rows, the chain row -> text -> table -> logits -> list -> cluster for few:
// slices are cut by what a round of blocks costs (rules_cut).
#include <limits.h>

#include "choice.cuh"
#include "range_check.cuh"

#define MIE_K_LOGIT_RULES 15       // this kernel's number in the range report (csrc/range_check.cuh)
#define RULES_MAX_PARTS 8          // slices of a row whose token is chosen: the blocks of a cluster
#define RULES_SM_THREADS 1024      // threads that share an SM, at 64 registers each
#define RULES_TABLE 32776          // words of a block's table at most: a slice of 65,536 entries of 16 bits, and its ragged ends
#define IN_PROMPT 0x80000000u      // an entry's word as 32 bits; as 16, the flags are the two highest bits too
#define HAS_BIAS 0x40000000u
#define COUNT_BITS 0x3fffffffu
#define NARROW_MOST 0x3fff
#define SUM_BITS 40                // 4 x 1,024 entries of a round, each at most 1 and off by at most 2^-40: 2^52 fits the word, and what is lost is below 2^-28 of the sum

struct RuleParams {
    const float* logits; int64_t logits_stride;
    float* out; int64_t out_stride;                       // apply
    int rows, vocab, table;                               // table: 32-bit words of shared memory for a slice (or a turn of one)
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

// exp by the hardware's 2^x (two units in the last place; -inf gives 0)
__device__ __forceinline__ float exp_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
// A running maximum m and the sum s of exp(x - m); nothing seen yet, or nothing but -inf: m = -inf, s = 0.  An x that is no number leaves m
// alone and makes s one too.  The sums' reference point:
__device__ __forceinline__ float exp_base(float m) { return m == -INFINITY ? 0.f : m; }

// Numbers as unsigned words of the same order (and back); 0 is below them all.
__device__ __forceinline__ unsigned ordered_bits(float x) {
    const unsigned u = __float_as_uint(x);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered_bits(unsigned k) { return k == 0 ? -INFINITY : __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

template <int T, bool CHOOSE, bool CLUSTER>
__global__ void __launch_bounds__(T, RULES_SM_THREADS / T)
logit_rules_kernel(const RuleParams p) {
    extern __shared__ __align__(16) uint32_t words[];
    __shared__ int s_twice;
    __shared__ unsigned s_top[2];                         // of a round of settled entries: the greatest logit, as ordered_bits (0: none) ...
    __shared__ unsigned long long s_sum[2];               // ... and the sum of exp(x' - greatest), in steps of 2^-SUM_BITS
    pdl_enter();
    if (CLUSTER) cluster_arrive_relaxed();                // (the wait for it: before the first block is written to)
    const int row = blockIdx.y, part = blockIdx.x, parts = gridDim.x, tid = threadIdx.x;
    const float* lg = p.logits + (int64_t)row * p.logits_stride;
    float* og = CHOOSE ? nullptr : p.out + (int64_t)row * p.out_stride;
    auto complain = [&](int code, int value) {
        if (part == 0 && tid == 0) range_report(p.report, code, MIE_K_LOGIT_RULES, row, value);
    };
    // ---- what holds for this row (all asked for at once: a chain of loads here is in front of everything)
    int slot = p.slot ? p.slot[row] : -1;
    int total = p.history ? p.total_len[row] : 0, prompt = p.history ? p.prompt_len[row] : 0;
    const float rep = p.repetition ? p.repetition[row] : 1.f, pres = p.presence ? p.presence[row] : 0.f, freq = p.frequency ? p.frequency[row] : 0.f;
    int biases = p.bias_len ? p.bias_len[row] : p.bias_width;
    int mask_row = p.mask_row ? p.mask_row[row] : -1;
    float temperature = CHOOSE ? p.temperature[row] : 0.f;
    const int64_t request = CHOOSE ? p.request[row] : 0;
    const int position = CHOOSE ? p.position[row] : 0;
    if (slot >= p.slots) {
        if (p.slot) complain(MIE_RANGE_ROW, slot);
        slot = -1;
    }
    if (slot < 0) total = prompt = biases = 0;
    if (total < 0 || total > p.width) { complain(MIE_RANGE_POSITION, total); total = total < 0 ? 0 : p.width; }
    if (biases < 0 || biases > p.bias_width) { complain(MIE_RANGE_POSITION, biases); biases = biases < 0 ? 0 : p.bias_width; }
    if (mask_row >= p.masks) { complain(MIE_RANGE_ROW, mask_row); mask_row = -1; }
    const bool text_counts = total > 0 && (rep != 1.f || pres != 0.f || freq != 0.f);
    const int* text = text_counts ? p.history + (int64_t)slot * p.history_stride : nullptr;
    const int* bias_tokens = biases ? p.bias_tokens + (int64_t)slot * p.bias_width : nullptr;
    const float* bias_values = biases ? p.bias_values + (int64_t)slot * p.bias_width : nullptr;
    const int* mask = mask_row >= 0 ? p.mask + (int64_t)mask_row * p.mask_stride : nullptr;
    const int last_word = (p.vocab - 1) >> 5;
    const bool marked = text_counts || biases > 0;        // some entries have words
    const bool narrow = !text_counts || total <= NARROW_MOST;
    const int room = narrow ? p.table * 2 : p.table;      // entries of a turn
    // the word of entry `at` of the turn: bits joined to it (returned: what it was), added to it, read
    auto join_word = [&](int at, uint32_t bits) {
        if (!narrow) return atomicOr(&words[at], bits);
        const int shift = (at & 1) * 16;
        return (atomicOr(&words[at >> 1], (bits >> 16) << shift) >> shift) << 16;
    };
    auto count_word = [&](int at) { atomicAdd(&words[narrow ? at >> 1 : at], narrow ? 1u << ((at & 1) * 16) : 1u); };
    auto widen = [](uint32_t w) { return ((w & 0xc000u) << 16) | (w & 0x3fffu); };
    auto word = [&](int at) { return narrow ? widen(words[at >> 1] >> ((at & 1) * 16)) : words[at]; };
    auto take_word = [&](int at) {                        // an unbiased entry's word, for the one thread that gets it; 0 for the others
        if (!narrow) return words[at] & HAS_BIAS ? 0u : atomicExch(&words[at], 0u);
        const int shift = (at & 1) * 16;
        const uint32_t now = words[at >> 1] >> shift;
        if ((now & 0xffffu) == 0 || (now & 0x4000u)) return 0u;
        return widen(atomicAnd(&words[at >> 1], ~(0xffffu << shift)) >> shift);
    };
    auto marks = [&](int at) -> uint32_t {                // which entries of a group (at % 4 == 0) have a word
        if (narrow) {
            const uint2 w = *reinterpret_cast<const uint2*>(words + (at >> 1));
            if (!(w.x | w.y)) return 0;
            return (w.x & 0xffffu ? 1 : 0) | (w.x >> 16 ? 2 : 0) | (w.y & 0xffffu ? 4 : 0) | (w.y >> 16 ? 8 : 0);
        }
        const uint4 w = *reinterpret_cast<const uint4*>(words + at);
        return (w.x ? 1 : 0) | (w.y ? 2 : 0) | (w.z ? 4 : 0) | (w.w ? 8 : 0);
    };

    const uint64_t key = CHOOSE && temperature > 0.f ? noise_key(p.seed, request, position) : 0;
    float bv = -INFINITY, bx = -INFINITY, m = -INFINITY, s = 0.f;       // the winner's score, its logit; the running maximum and sum
    int bi = 0x7fffffff;
    float gv = -INFINITY;                                 // the same of the groups that are read four at a time: the best group's score, its logits and place
    float4 gx;
    int gi = -1;

    // ---- this block's slice.  Slices begin where the row's 16-byte groups do (`off` entries before the row's first whole group).
    const int off = (int)((4 - ((reinterpret_cast<uintptr_t>(lg) >> 2) & 3)) & 3);
    const bool wide = CHOOSE || ((reinterpret_cast<uintptr_t>(lg) ^ reinterpret_cast<uintptr_t>(og)) & 15) == 0;      // 16-byte groups of the output too
    const int per = ((p.vocab + parts - 1) / parts + 3) & ~3;
    const int64_t lo64 = part ? (int64_t)part * per + off : 0, hi64 = (int64_t)(part + 1) * per + off;
    const int lo = (int)min((int64_t)p.vocab, lo64), hi = part + 1 == parts ? p.vocab : (int)min((int64_t)p.vocab, hi64);

    // the slice's logits are asked for ahead: they come into L2 while the table is made (256 rows 79 -> 77 us; the choice for 64 rows does not gain, 18.8 -> 19.1)
    if (!CHOOSE && marked && tid == 0) {
        const int first = (lo == 0 ? off : lo), n = (hi - first) & ~3;
        if (n > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(lg + first), "r"(n * 4) : "memory");
    }
    const int my_bias = tid < biases ? bias_tokens[tid] : -1;           // the first T entries of the list: a thread each
    const float my_value = tid < biases ? bias_values[tid] : 0.f;
    const float my_logit = CHOOSE && my_bias >= 0 && my_bias < p.vocab ? lg[my_bias] : 0.f;
    auto bias_token = [&](int j) { return j == tid ? my_bias : bias_tokens[j]; };
    for (int c0 = lo; c0 < hi; ) {
        // Entry i's word is words[i - base], so that a group's four words lie on 16 bytes as its logits do.  (A first turn is shorter for that.)
        const int base = c0 == 0 ? off - 4 : c0;
        const int c1 = marked ? min(hi, base + room) : hi;
        if (marked) {
            __syncthreads();                              // the turn before is done with the words
            for (int i = tid * 4; i < (narrow ? (c1 - base + 1) >> 1 : c1 - base); i += T * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
            if (tid == 0) { s_twice = 0; s_top[0] = s_top[1] = 0; s_sum[0] = s_sum[1] = 0; }
            __syncthreads();
            if (text_counts) {
                constexpr int AT_ONCE = 8;                // tokens that a thread asks for before it counts the first
                for (int j0 = tid; j0 < total; j0 += AT_ONCE * T) {
                    int t[AT_ONCE];
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u) t[u] = j0 + u * T < total ? text[j0 + u * T] : INT_MAX;
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u) {
                        const int j = j0 + u * T;
                        if (j >= total) break;
                        if (t[u] >= c0 && t[u] < c1) {
                            if (j < prompt) join_word(t[u] - base, IN_PROMPT);
                            else count_word(t[u] - base);
                        } else if (c0 == 0 && (t[u] < 0 || t[u] >= p.vocab)) {
                            range_report(p.report, MIE_RANGE_TOKEN, MIE_K_LOGIT_RULES, row, t[u]);
                        }
                    }
                }
            }
            for (int j = tid; j < biases; j += T) {
                const int t = bias_token(j);
                if (t >= c0 && t < c1) {
                    if (join_word(t - base, HAS_BIAS) & HAS_BIAS) s_twice = 1;
                } else if (c0 == 0 && (t < 0 || t >= p.vocab)) range_report(p.report, MIE_RANGE_TOKEN, MIE_K_LOGIT_RULES, row, t);
            }
            __syncthreads();
        }
        auto penalised = [&](float x, uint32_t w) {       // an entry's logit under the penalties
            const uint32_t count = w & COUNT_BITS;
            if (count | (w & IN_PROMPT)) x = x > 0.f ? x / rep : x * rep;
            if (count) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)count), pres));
            return x;
        };
        auto allows = [&](int i) { return !mask || ((mask[i >> 5] >> (i & 31)) & 1); };
        auto consider = [&](float x, int i) {
            const float v = temperature > 0.f ? noisy_score(x, temperature, key, i) : x;
            if (v > bv || (v == bv && i < bi && v > -INFINITY)) { bv = v; bi = i; bx = x; }
        };
        auto settle = [&](float x, int i) {               // one entry's last value
            if (!allows(i)) x = -INFINITY;
            if (CHOOSE) {
                consider(x, i);
                const float mn = fmaxf(m, x), ref = exp_base(mn);
                s = s * exp_fast(m - ref) + exp_fast(x - ref);
                m = mn;
            } else og[i] = x;
        };
        const int first = min(c1, c0 == 0 ? off : c0);    // whole groups from here on
        const int groups = wide ? (c1 - first) >> 2 : 0;
        auto one = [&](int i) {
            if (!(marked && word(i - base))) settle(lg[i], i);
            else if (!CHOOSE) og[i] = lg[i];
        };
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
                x4[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (g < groups) {
                    x4[u] = __ldcs(reinterpret_cast<const float4*>(lg + i));
                    if (mask) {
                        const int w = i >> 5;
                        bits[u] = __funnelshift_r((uint32_t)mask[w], (uint32_t)mask[min(w + 1, last_word)], i & 31);
                    }
                }
            }
            float most = -INFINITY;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int g = g0 + u * T, i = first + g * 4;
                float x[4] = {x4[u].x, x4[u].y, x4[u].z, x4[u].w};
                if (CHOOSE && marked && g < groups) bits[u] &= ~marks(i - base);      // (those are not in the running yet)
                if (CHOOSE ? bits[u] != 0xffffffffu : mask != nullptr) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (!((bits[u] >> e) & 1)) x[e] = -INFINITY;
                }
                if (CHOOSE) {
                    x4[u] = make_float4(x[0], x[1], x[2], x[3]);
                    most = fmaxf(most, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
                } else if (g < groups) {
                    __stcs(reinterpret_cast<float4*>(og + i), make_float4(x[0], x[1], x[2], x[3]));
                }
            }
            if (CHOOSE) {
                // the best so far as a value and the group that holds it; which of its four it is, is asked once, at the end
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int i = first + (g0 + u * T) * 4;
                    float4 v = x4[u];
                    if (temperature > 0.f) {
                        v.x = noisy_score(v.x, temperature, key, i); v.y = noisy_score(v.y, temperature, key, i + 1);
                        v.z = noisy_score(v.z, temperature, key, i + 2); v.w = noisy_score(v.w, temperature, key, i + 3);
                    }
                    const float top = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
                    if (top > gv) {
                        gv = top;
                        gx = x4[u];
                        gi = i;
                    }
                }
                if (p.logprob) {
                    const float mn = fmaxf(m, most), ref = exp_base(mn);
                    if (mn > m) { s *= exp_fast(m - ref); m = mn; }
                    float sum[AHEAD];
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u)
                        sum[u] = (exp_fast(x4[u].x - ref) + exp_fast(x4[u].y - ref)) + (exp_fast(x4[u].z - ref) + exp_fast(x4[u].w - ref));
                    s += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                }
            }
        }
        if (CHOOSE && gi >= 0) {                          // the entries of the best group (a group of -inf alone is no candidate)
            consider(gx.x, gi); consider(gx.y, gi + 1); consider(gx.z, gi + 2); consider(gx.w, gi + 3);
            gi = -1;
        }
        if (marked) {
            __syncthreads();                              // (choose) nobody asks for marks any more; (apply) the output holds the marked entries' logits
            if (text_counts) {
                constexpr int AT_ONCE = 4;                // (choosing for 200 and 64 rows 34.9 and 19.6 us; 2: 36.6 and 20.4, 8: 34.2 and 20.9, and 9.4 for 8 rows instead of 8.3)
                for (int r0 = 0, turn = 0; r0 < total; r0 += AT_ONCE * T, turn ^= 1) {
                    const int j0 = r0 + tid;
                    int t[AT_ONCE];
                    uint32_t w[AT_ONCE];
                    float x[AT_ONCE];
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u) t[u] = j0 + u * T < total ? text[j0 + u * T] : INT_MAX;
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u) w[u] = t[u] >= c0 && t[u] < c1 ? take_word(t[u] - base) : 0;
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u) x[u] = !w[u] ? 0.f : CHOOSE ? lg[t[u]] : og[t[u]];
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u) {
                        if (w[u]) {
                            x[u] = penalised(x[u], w[u]);
                            if (!allows(t[u])) x[u] = -INFINITY;
                            if (CHOOSE) consider(x[u], t[u]);
                            else og[t[u]] = x[u];
                        } else x[u] = -INFINITY;
                    }
                    if (CHOOSE && p.logprob) {            // (the same for every thread of the block)
                        unsigned top = 0;
#pragma unroll
                        for (int u = 0; u < AT_ONCE; ++u) {
                            if (x[u] != x[u]) s = x[u];   // no number: nor is the sum
                            else top = max(top, ordered_bits(x[u]));
                        }
                        top = __reduce_max_sync(0xffffffffu, top);
                        if ((tid & 31) == 0) atomicMax(&s_top[turn], top);
                        __syncthreads();                  // the greatest is known, and every word of this round is taken
                        const float most = from_ordered_bits(s_top[turn]), ref = exp_base(most);
                        unsigned long long sum = 0;
#pragma unroll
                        for (int u = 0; u < AT_ONCE; ++u) {
                            const float e = exp_fast(x[u] - ref);
                            if (e != e) s = e;            // inf - inf
                            else sum += (unsigned long long)(e * (float)(1ull << SUM_BITS));
                        }
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                        if ((tid & 31) == 0) atomicAdd(&s_sum[turn], sum);
                        __syncthreads();
                        if (tid == 0) {
                            const float mn = fmaxf(m, most), join = exp_base(mn);
                            s = s * exp_fast(m - join) + (float)s_sum[turn] * (1.f / (float)(1ull << SUM_BITS)) * exp_fast(most - join);
                            m = mn;
                            s_top[turn] = 0;              // (asked for again two rounds on)
                            s_sum[turn] = 0;
                        }
                    }
                }
            }
            const bool twice = s_twice != 0;              // a token of this turn is named more than once: the list is walked for it
            for (int j = tid; j < biases; j += T) {
                const int t = bias_token(j);
                if (t < c0 || t >= c1) continue;
                float x = penalised(CHOOSE ? j == tid ? my_logit : lg[t] : og[t], word(t - base));
                if (!twice) x = __fadd_rn(x, j == tid ? my_value : bias_values[j]);
                else {
                    bool earlier = false;                 // the first that names it adds up all of them, in the list's order
                    for (int k = 0; k < j && !earlier; ++k) earlier = bias_tokens[k] == t;
                    if (earlier) continue;
                    for (int k = j; k < biases; ++k) if (bias_tokens[k] == t) x = __fadd_rn(x, bias_values[k]);
                }
                settle(x, t);
            }
        }
        c0 = c1;
    }
    if (!CHOOSE) return;

    // ---- the block's winner and sums, then the row's
    __shared__ float w_v[T / 32], w_x[T / 32], w_m[T / 32], w_s[T / 32];
    __shared__ int w_i[T / 32];
    __shared__ float parts_of[5][RULES_MAX_PARTS];                      // the first block's: every slice's winner, its logit and index, maximum and sum
    auto reduce_warp = [&]() {
        const float ref = exp_base(warp_max(m));
        s = warp_sum(s * exp_fast(m - ref));
        m = warp_max(m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o), ox = __shfl_xor_sync(0xffffffffu, bx, o);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; bx = ox; }
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
    }
    auto finish = [&]() {
        const int tok = bi < p.vocab ? bi : 0;            // nothing but -inf and NaN
        p.token[row] = tok;
        if (p.logprob) p.logprob[row] = m == -INFINITY && s == 0.f ? -INFINITY : (bx - m) - logf(s);
        if (p.append && slot >= 0 && total < p.width) p.append[(int64_t)slot * p.history_stride + total] = tok;
        if (p.host_out) p.host_out[(p.host_turn ? *p.host_turn : 0) * p.host_stride + row] = tok;
    };
    if (!CLUSTER) {
        if (tid == 0) finish();
        return;
    }
    cluster_wait();                                       // every block of the cluster runs: the first may be written to
    if (warp == 0 && lane < 5) {
        const float v = lane == 0 ? bv : lane == 1 ? bx : lane == 2 ? __int_as_float(bi) : lane == 3 ? m : s;
        st_cluster_f32(cluster_addr((uint32_t)__cvta_generic_to_shared(&parts_of[lane][part]), 0), v);
    }
    __syncwarp();
    cluster_sync_all();                                   // every slice's share is in the first block's shared memory
    if (part == 0 && warp == 0) {
        const bool on = lane < parts;
        bv = on ? parts_of[0][lane] : -INFINITY; bx = on ? parts_of[1][lane] : -INFINITY; bi = on ? __float_as_int(parts_of[2][lane]) : 0x7fffffff;
        m = on ? parts_of[3][lane] : -INFINITY; s = on ? parts_of[4][lane] : 0.f;
        reduce_warp();
        if (lane == 0) finish();
    }
}

// Words of a block's table for slices of `per` entries: 16 bits each, whole groups, and the row's ragged ends.
static int rules_table(int per) {
    const int words = (per / 2 + 8 + 3) & ~3;
    return words < RULES_TABLE ? words : RULES_TABLE;
}
// Slices a row and threads a block: the cut whose rounds of blocks are over first, a round counted as 2 for its chain of loads and barriers and 0.4 for every 256
// threads more in those, 0.3 for 16 entries a thread and 3 for eight tokens of text a thread (a row's text is taken as half as long as the slots are wide).  These
// weights take, of twelve cuts measured for thirty shapes (1 to 500 rows, 32,000 to 151,936 entries, texts of 64 to 12,000), one that is 6% behind the best on the
// average; 6, 0.4, 0.6 and 1.5 one 8% behind.  Us, slices x threads: the choice for 200 rows of 50,001 entries, 1 x 1,024 32.8, 1 x 512 35.0, 2 x 512 35.3, 8 x 256
// 53; for 8 rows of 32,000, 8 x 256 7.8, 8 x 512 8.2, 1 x 1,024 11.1; 64 rows of 128,256 written, texts of up to 2,000, 4 x 512 18.3, 8 x 256 19.4, 2 x 1,024 18.5.
struct RuleCut { int parts, threads; };
static RuleCut rules_cut(int rows, int vocab, int width, bool choose) {
    RuleCut best = {1, 1024};
    double least = 1e30;
    const int sms = device_sm_count();
    for (int threads = 256; threads <= 1024; threads *= 2) {
        for (int parts = 1; parts <= (choose ? RULES_MAX_PARTS : 64); parts *= 2) {
            const int per = ((vocab + parts - 1) / parts + 3) & ~3;
            int fit = (int)(232448 / ((size_t)rules_table(per) * 4 + 2048));
            if (fit > RULES_SM_THREADS / threads) fit = RULES_SM_THREADS / threads;
            const int64_t places = (int64_t)fit * sms, rounds = ((int64_t)rows * parts + places - 1) / places;
            const double cost = (double)rounds * (2.0 + 0.4 * (threads / 256 - 1) + 0.3 * per / (16.0 * threads) + 3.0 * (width / 2) / (8.0 * threads));
            if (cost < least) { least = cost; best = RuleCut{parts, threads}; }
        }
    }
    return best;
}

template <int T>
static int launch_rules_threads(const RuleParams& p, bool choose, int parts, cudaStream_t stream) {
    const size_t smem = p.history || p.bias_tokens ? (size_t)p.table * 4 : 0;
    auto kernel = !choose ? logit_rules_kernel<T, false, false> : parts > 1 ? logit_rules_kernel<T, true, true> : logit_rules_kernel<T, true, false>;
    static unsigned long long allowed[3] = {0, 0, 0};      // a kernel's devices on which it may have that much shared memory
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    unsigned long long* on = &allowed[!choose ? 0 : parts > 1 ? 1 : 2];
    if (device > 63 || !(__atomic_load_n(on, __ATOMIC_RELAXED) >> device & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RULES_TABLE * 4);
        if (e != cudaSuccess) return (int)e;
        if (device <= 63) __atomic_fetch_or(on, 1ull << device, __ATOMIC_RELAXED);
    }
    return launch_kernel_cluster(kernel, dim3(parts, p.rows), dim3(T), smem, stream, dim3(choose ? parts : 1, 1, 1), p);
}

static int launch_rules(RuleParams& p, bool choose, cudaStream_t stream) {
    if (p.rows <= 0) return 0;
    if (p.vocab <= 0 || p.slots < 0 || p.width < 0 || p.bias_width < 0 || p.masks < 0) return MIE_ERR_BAD_ARG;
    if (p.rows > 65535 || p.width > (int)COUNT_BITS) return MIE_ERR_TOO_LARGE;
    if ((p.history || p.bias_tokens) && !p.slot) return MIE_ERR_BAD_ARG;
    if (p.history && (!p.total_len || !p.prompt_len)) return MIE_ERR_BAD_ARG;
    if (p.bias_tokens && !p.bias_values) return MIE_ERR_BAD_ARG;
    if (p.mask && p.mask_stride < (p.vocab + 31) / 32) return MIE_ERR_BAD_ARG;
    const RuleCut cut = rules_cut(p.rows, p.vocab, p.history ? p.width : 0, choose);
    p.table = rules_table(((p.vocab + cut.parts - 1) / cut.parts + 3) & ~3);
    switch (cut.threads) {
        case 256: return launch_rules_threads<256>(p, choose, cut.parts, stream);
        case 512: return launch_rules_threads<512>(p, choose, cut.parts, stream);
        default: return launch_rules_threads<1024>(p, choose, cut.parts, stream);
    }
}

// The rules' arguments as the caller lays them out once for many calls (kernels/ops.py: LogitRules).
struct RuleArgs {
    const int* history; const int* slot; const int* prompt_len; const int* total_len;
    const float* repetition; const float* presence; const float* frequency;
    const int* bias_tokens; const float* bias_values; const int* bias_len;
    const int* mask; const int* mask_row;
    long long history_stride, mask_stride;
    int slots, width, bias_width, masks;
};
static void set_rules(RuleParams& p, const RuleArgs& a) {
    p.history = a.history; p.history_stride = a.history_stride; p.slots = a.slots; p.width = a.width;
    p.slot = a.slot; p.prompt_len = a.prompt_len; p.total_len = a.total_len;
    p.repetition = a.repetition; p.presence = a.presence; p.frequency = a.frequency;
    p.bias_tokens = a.bias_tokens; p.bias_values = a.bias_values; p.bias_width = a.bias_width; p.bias_len = a.bias_len;
    p.mask = a.mask; p.mask_stride = a.mask_stride; p.masks = a.masks; p.mask_row = a.mask_row;
    p.report = g_range_report;
}

// out[r] = the logits of row r under its rules (out may be the logits).
extern "C" int mie_apply_logit_rules(const RuleArgs* rules, const float* logits, long long logits_stride, float* out, long long out_stride, int rows, int vocab,
                                     cudaStream_t stream) {
    RuleParams p = {};
    set_rules(p, *rules);
    p.logits = logits; p.logits_stride = logits_stride; p.out = out; p.out_stride = out_stride; p.rows = rows; p.vocab = vocab;
    if (rows > 0 && !out) return MIE_ERR_BAD_ARG;
    return launch_rules(p, false, stream);
}

// The token of every row under its rules; see mie_sample (sampling.cu) for the noise and the host's copy.  `logprob` (or null): log softmax of the
// ruled logits at the token, -inf where the rules leave nothing (the token is 0 there).  `append`: the token joins the row's text.
extern "C" int mie_sample_rules(const RuleArgs* rules, const float* logits, long long logits_stride, const float* temperature, const int64_t* request,
                                const int* position, uint64_t seed, int* token, float* logprob, int append, int rows, int vocab, int* host_out,
                                const int* host_turn, int host_stride, cudaStream_t stream) {
    RuleParams p = {};
    set_rules(p, *rules);
    p.logits = logits; p.logits_stride = logits_stride; p.rows = rows; p.vocab = vocab;
    p.temperature = temperature; p.request = request; p.position = position; p.seed = seed;
    p.token = token; p.logprob = logprob; p.append = append ? const_cast<int*>(p.history) : nullptr;
    p.host_out = host_out; p.host_turn = host_turn; p.host_stride = host_stride;
    return launch_rules(p, true, stream);
}
