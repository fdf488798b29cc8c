// How the work on shared prefixes is cut up, decided on the device from the step's groups alone, so that a captured step follows whatever groups
// and lengths its inputs hold.  Two kernels ask and have to agree: the one that attends over the prefixes and the one that joins its results
// with the rows' own keys.
//
// Group g is the rows start[g] .. start[g + 1] - 1; they share their first prefix[g] keys.  For a unit (a key head, or a part of its query heads)
// the (row, head) pairs of a group go in tiles of up to `tile_rows` rows, and the prefix, counted in steps of PREFIX_STEP keys, is cut
// into `splits` ranges.  An item is one (group, unit, tile, range); its result goes to slot (slot0 + row within the group * splits + range).
#pragma once
#include "common.cuh"

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
    return rows + 2ll * places * tile_rows / units + tile_rows;
}

#ifdef __CUDACC__
// Steps a range, for every lane the same; by a whole warp: lane l weighs up cutting the longest prefix into l + 1 and l + 33 ranges.
__device__ __forceinline__ int prefix_chunk(const PrefixGroups& p) {
    const int lane = threadIdx.x & 31, most = prefix_most_steps(p);
    long long best = 0x7fffffffffffffffll;
    int chunk = most;
#pragma unroll 1
    for (int s = lane + 1; s <= PREFIX_MAX_SPLITS && s < most + 32; s += 32) {
        int c;
        const long long cost = prefix_cost(p, most, s, c);
        if (cost >= 0 && cost < best) { best = cost; chunk = c; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const long long ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oc = __shfl_xor_sync(0xffffffffu, chunk, o);
        if (ob < best || (ob == best && oc > chunk)) { best = ob; chunk = oc; }
    }
    return chunk;
}
// The group that item `item` (or, with by_row, row `item`) belongs to; rows 0 where there is none.
__device__ __forceinline__ PrefixPart prefix_find(const PrefixGroups& p, int chunk, int item, bool by_row) {
    int items = 0, slots = 0;
    for (int g = 0; g < p.groups; ++g) {
        PrefixPart t = prefix_group(p, g);
        t.splits = t.tiles ? prefix_splits(t.steps, chunk) : 0;
        t.item0 = items;
        t.slot0 = slots;
        items += p.units * t.tiles * t.splits;
        slots += t.rows * t.splits;
        if (by_row ? item >= t.first_row && item < t.first_row + t.rows : item < items) return t;
    }
    return PrefixPart{};
}
#endif
