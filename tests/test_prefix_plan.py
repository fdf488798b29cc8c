"""How work on shared prefixes is cut: the arithmetic of csrc/prefix_plan.cuh, compiled for the host."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mini_inference_engine_b200", "csrc")

SOURCE = r"""
#include <algorithm>
#include <cstdint>
using std::max; using std::min;
#define __host__
#define __device__
#define __forceinline__ inline
#define MIE_HOST_ONLY
#include "prefix_plan_host.h"
extern "C" {
// out: chunk, items, slots, most items, most slots
void plan(const int* start, const int* prefix, int groups, int rows, int most_keys, int units, int tile_rows, int places, long long* out) {
    PrefixGroups p{start, prefix, groups, rows, most_keys, units, tile_rows, places};
    const int most = prefix_most_steps(p);
    long long best = -1; int chunk = most;
    for (int s = 1; s <= PREFIX_MAX_SPLITS && s < most + 32; ++s) {
        int c; const long long cost = prefix_cost(p, most, s, c);
        if (cost >= 0 && (best < 0 || cost < best || (cost == best && c > chunk))) { best = cost; chunk = c; }
    }
    long long slots = 0;
    for (int g = 0; g < groups; ++g) { const PrefixPart t = prefix_group(p, g); slots += (long long)t.rows * (t.tiles ? prefix_splits(t.steps, chunk) : 0); }
    out[0] = chunk; out[1] = prefix_items(p, chunk); out[2] = slots;
    out[3] = prefix_most_items(rows, groups, units, tile_rows, places); out[4] = prefix_most_slots(rows, units, tile_rows, places);
}
void range(int steps, int splits, int s, int* out) { prefix_range(steps, splits, s, out[0], out[1]); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    text = open(os.path.join(CSRC, "prefix_plan.cuh")).read().replace('#include "common.cuh"', "").replace("#pragma once", "")
    (d / "prefix_plan_host.h").write_text(text)
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(d / "plan.so"), str(d / "plan.cpp")], check=True)
    return ctypes.CDLL(str(d / "plan.so"))


def plan(lib, start, prefix, rows, most_keys, units, tile_rows, places):
    out = (ctypes.c_longlong * 5)()
    n = len(prefix)
    lib.plan((ctypes.c_int * (n + 1))(*start), (ctypes.c_int * max(1, n))(*prefix), n, rows, most_keys, units, tile_rows, places, out)
    return list(out)


def test_grid_and_scratch_hold_every_plan(lib):
    rng = random.Random(0)
    for _ in range(3000):
        groups = rng.randint(0, 9)
        rows = rng.choice([1, 2, rng.randint(1, 300)])
        cuts = sorted(rng.randint(0, rows) for _ in range(groups + 1))
        prefix = [rng.choice([0, 1, rng.randint(0, 40000)]) for _ in range(groups)]
        units, tile_rows, places = rng.choice([1, 2, 4, 8, 32, 40]), rng.choice([1, 2, 5, 16, 64, 128]), rng.choice([1, 148, 296])
        chunk, items, slots, most_items, most_slots = plan(lib, cuts, prefix, rows, 32768, units, tile_rows, places)
        assert chunk >= 1 and items <= most_items and slots <= most_slots, (cuts, prefix, rows, units, tile_rows, places)


def test_wild_groups_stay_within_the_rows(lib):
    """Whatever the device holds as groups, no item reads rows or keys that are not there."""
    rng = random.Random(1)
    for _ in range(500):
        groups = rng.randint(1, 5)
        cuts = [rng.choice([-5, 0, 3, 99, 2 ** 31 - 1, -2 ** 31]) for _ in range(groups + 1)]
        prefix = [rng.choice([-1, 0, 2 ** 31 - 1, 77]) for _ in range(groups)]
        out = plan(lib, cuts, prefix, 20, 4096, 8, 16, 296)
        assert out[0] >= 1 and out[1] >= 0


def test_ranges_cover_a_prefix_once(lib):
    for steps in list(range(1, 70)) + [1000]:
        for splits in sorted({1, 2, 3, min(steps, 7), steps} & set(range(1, steps + 1))):
            at = 0
            for s in range(splits):
                out = (ctypes.c_int * 2)()
                lib.range(steps, splits, s, out)
                assert out[0] == at and out[1] >= 1
                at += out[1]
            assert at == steps


def test_one_long_prefix_fills_the_gpu(lib):
    # 64 rows of one group, 8 key heads, 16 rows a tile: 32 tiles without cuts; 296 places
    chunk, items, _, _, _ = plan(lib, [0, 64], [8192], 64, 16384, 8, 16, 296)
    assert 200 <= items <= 296 and chunk == 8
