// How the work on shared prefixes is cut up, decided on the device from the step's groups alone, so that a captured step follows whatever groups
// and lengths its inputs hold.  The kernel that attends over the prefixes decides and leaves the length of its ranges (`chunk`) to the one that joins its
// results with the rows' own keys.
//
// Group g is the rows start[g] .. start[g + 1] - 1; they share their first prefix[g] keys.  For a unit (a key head, or a part of its query heads)
// the (row, head) pairs of a group go in tiles of up to `tile_rows` rows, and the prefix, counted in steps of PREFIX_STEP keys, is cut
// into `splits` ranges.  An item is one (group, unit, tile, range); its result goes to slot (slot0 + row within the group * splits + range).
#pragma once
#include "common.cuh"

#define MIE_K_ATTENTION_PREFIX 16      // what reads prefixes, in the range report (csrc/range_check.cuh)

#define PREFIX_STEP 128
#define PREFIX_MAX_SPLITS 64
#define PREFIX_COST_START 3        // what starting and ending an item costs, in steps

struct PrefixGroups {
    const int* start; const int* prefix; int groups;      // [groups + 1], [groups]
    int num_rows, most_keys;                              // rows of the step; keys that a block table covers
    int units, tile_rows, places;                         // rows a tile; items that run side by side
};
struct PrefixPart { int first_row, rows, keys, tiles, steps, splits, slot0, item0; };       // a group and how it is cut (rows 0: there is none)

__host__ __device__ __forceinline__ int prefix_splits(int steps, int chunk) { return (steps + chunk - 1) / chunk; }
// The steps of range s of a prefix: [first, first + n).  All ranges are as long as one another, or a step longer.
__host__ __device__ __forceinline__ void prefix_range(int steps, int splits, int s, int& first, int& n) {
    const int base = steps / splits, more = steps - base * splits;
    first = s * base + min(s, more);
    n = base + (s < more ? 1 : 0);
}

// The steps of an item of the walk over prefix and own keys (attention_prefix.cu): J of them, the first npre the prefix's.  With two tiles of pairs (`both`) a chain owns a tile:
// both chains take part in a step of the prefix; the own keys of a tile are a list (steps0 and steps1 steps), and the lists take turns while both have steps left.
// With one tile the chains take the steps in turns.
struct WalkSteps { int J, npre, own0, steps0, steps1; bool both; };        // own0 + j: own step j's place among those of the whole walk
struct OwnStep { int list, k; };                                           // the k-th step of a list
__host__ __device__ __forceinline__ OwnStep walk_own_step(const WalkSteps& w, int j) {
    const int x = w.own0 + j, turns = min(w.steps0, w.steps1);
    if (x < 2 * turns) return OwnStep{x & 1, x >> 1};
    return OwnStep{w.steps1 > w.steps0 ? 1 : 0, x - turns};
}
// Does chain c take part in step j?
__host__ __device__ __forceinline__ bool walk_takes_part(const WalkSteps& w, int c, int j) {
    if (!w.both) return (j & 1) == c;
    return j < w.npre || walk_own_step(w, j).list == c;
}
// Step j lies where step j - stages lay.  A chain that took part in that one knows that its keys and values have come; where the other chain alone did (the lists' turns have just
// ended), a wait for step j's could take the phase before it for its own.  The other chain has no step behind j then.
__host__ __device__ __forceinline__ bool walk_behind_other(const WalkSteps& w, int c, int j, int stages) {
    return w.both && j - stages >= w.npre && walk_own_step(w, j - stages).list != c;
}

__host__ __device__ __forceinline__ PrefixPart prefix_group(const PrefixGroups& p, int g) {
    PrefixPart t = {};
    const int a = max(0, min(p.start[g], p.num_rows)), b = max(a, min(p.start[g + 1], p.num_rows));
    t.first_row = a;
    t.rows = b - a;
    t.keys = max(0, min(p.prefix[g], p.most_keys));
    t.steps = (t.keys + PREFIX_STEP - 1) / PREFIX_STEP;
    t.tiles = t.steps ? (t.rows + p.tile_rows - 1) / p.tile_rows : 0;
    return t;
}
__host__ __device__ __forceinline__ long long prefix_items(const PrefixGroups& p, int chunk) {
    long long n = 0;
    for (int g = 0; g < p.groups; ++g) {
        const PrefixPart t = prefix_group(p, g);
        n += (long long)p.units * t.tiles * prefix_splits(t.steps, chunk);
    }
    return n;
}
__host__ __device__ __forceinline__ int prefix_most_steps(const PrefixGroups& p) {
    int most = 1;
    for (int g = 0; g < p.groups; ++g) {
        const PrefixPart t = prefix_group(p, g);
        if (t.tiles) most = max(most, t.steps);
    }
    return most;
}
// What cutting the longest prefix into `splits` ranges would cost: rounds of items times the steps of the longest.  -1: not allowed (so many items
// that neither the grid nor the scratch memory holds them).
__host__ __device__ __forceinline__ long long prefix_cost(const PrefixGroups& p, int most_steps, int splits, int& chunk) {
    chunk = (most_steps + splits - 1) / splits;
    const long long items = prefix_items(p, chunk);
    if (splits > 1 && items > 2ll * p.places) return -1;
    return ((items + p.places - 1) / p.places) * (chunk + PREFIX_COST_START);
}
// The most items and slots that a plan can come to (the host sizes grid and scratch memory by them).
__host__ __device__ __forceinline__ long long prefix_most_items(int rows, int groups, int units, int tile_rows, int places) {
    const long long whole = (long long)units * ((rows + tile_rows - 1) / tile_rows + groups);
    return whole > 2ll * places ? whole : 2ll * places;
}
__host__ __device__ __forceinline__ long long prefix_most_slots(int rows, int units, int tile_rows, int places) {
    return 2ll * rows + 2ll * places * tile_rows / units + tile_rows;      // (a walk's results come in twos where its pairs fill one tile only)
}

#ifdef __CUDACC__
#include "range_check.cuh"

// Does a row's step write a key of its prefix (its newest key is the prefix's last, say)?
__device__ __forceinline__ bool writes_prefix(int len, int ctx, int keys) { return len > 0 && ctx - len < keys; }
// Reports a group whose rows are none of the step's, or go back, and a prefix that is negative or longer than a block table.
__device__ __forceinline__ void check_group(const PrefixGroups& p, int g, int* report) {
    const int a = p.start[g], b = p.start[g + 1], keys = p.prefix[g];
    if (a < 0 || a > b || b > p.num_rows) range_report(report, MIE_RANGE_ROW, MIE_K_ATTENTION_PREFIX, g, a < 0 || a > b ? a : b);
    else if (b > a && (keys < 0 || keys > p.most_keys)) range_report(report, MIE_RANGE_POSITION, MIE_K_ATTENTION_PREFIX, a, keys);
}

// Steps a range, for every lane the same; by a whole warp: lane l weighs up cutting the longest prefix into l + 1 and l + 33 ranges.  A lane holds a
// group (of up to 32: the host's arithmetic above for more); 13.3 -> 11.7 us for the two launches of a step of two rows behind 208 keys against every
// lane reading every group.
__device__ __forceinline__ int prefix_chunk(const PrefixGroups& p) {
    const int lane = threadIdx.x & 31;
    const bool few = p.groups <= 32;
    PrefixPart mine = {};
    if (few && lane < p.groups) mine = prefix_group(p, lane);
    int most;
    if (few) {
        most = mine.tiles ? mine.steps : 1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    } else most = prefix_most_steps(p);
    const unsigned whole = mine.tiles ? (unsigned)p.units * mine.tiles : 0u;
    unsigned best = 0xffffffffu;
    int chunk = most;
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
        const int s = lane + 1 + 32 * turn;
        if (turn && most <= 32) break;
        unsigned cost = 0xffffffffu;
        int c = max(1, (most + s - 1) / s);
        if (few) {
            unsigned long long items = 0;
            for (int g = 0; g < p.groups; ++g) {
                const int steps = __shfl_sync(0xffffffffu, mine.steps, g);
                items += (unsigned long long)__shfl_sync(0xffffffffu, whole, g) * prefix_splits(steps, c);
            }
            const unsigned n = (unsigned)min(items, 0x3fffffffull);
            if (s == 1 || n <= 2u * p.places) cost = ((n + p.places - 1) / p.places) * (unsigned)(c + PREFIX_COST_START);
        } else {
            const long long l = prefix_cost(p, most, s, c);
            if (l >= 0) cost = (unsigned)min(l, 0xfffffffell);
        }
        if (s < most + 32 && cost < best) { best = cost; chunk = c; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oc = __shfl_xor_sync(0xffffffffu, chunk, o);
        if (ob < best || (ob == best && oc > chunk)) { best = ob; chunk = oc; }
    }
    return chunk;
}
// The group that item `item` (or, with by_row, row `item`) belongs to; rows 0 where there is none.  By a whole warp, for every lane the same.
__device__ __forceinline__ PrefixPart prefix_find(const PrefixGroups& p, int chunk, int item, bool by_row) {
    const int lane = threadIdx.x & 31;
    int items = 0, slots = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        PrefixPart t = {};
        if (g0 + lane < p.groups) t = prefix_group(p, g0 + lane);
        t.splits = t.tiles ? prefix_splits(t.steps, chunk) : 0;
        const int n = p.units * t.tiles * t.splits, k = t.rows * t.splits;
        int ni = n, ki = k;                                // sums up to this lane's group
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, ni, o), b = __shfl_up_sync(0xffffffffu, ki, o);
            if (lane >= o) { ni += a; ki += b; }
        }
        t.item0 = items + ni - n;
        t.slot0 = slots + ki - k;
        const unsigned hit = __ballot_sync(0xffffffffu, by_row ? item >= t.first_row && item < t.first_row + t.rows : item >= t.item0 && item < t.item0 + n);
        if (hit) {
            const int l = __ffs(hit) - 1;
            t.first_row = __shfl_sync(0xffffffffu, t.first_row, l); t.rows = __shfl_sync(0xffffffffu, t.rows, l);
            t.keys = __shfl_sync(0xffffffffu, t.keys, l); t.tiles = __shfl_sync(0xffffffffu, t.tiles, l);
            t.steps = __shfl_sync(0xffffffffu, t.steps, l); t.splits = __shfl_sync(0xffffffffu, t.splits, l);
            t.slot0 = __shfl_sync(0xffffffffu, t.slot0, l); t.item0 = __shfl_sync(0xffffffffu, t.item0, l);
            return t;
        }
        items += __shfl_sync(0xffffffffu, ni, 31);
        slots += __shfl_sync(0xffffffffu, ki, 31);
    }
    return PrefixPart{};
}
#endif
