"""Which steps of the walk over shared prefixes a chain takes part in, and what it knows of the place in shared memory that a step's keys come to: the arithmetic of
csrc/prefix_plan.cuh, compiled for the host."""
import ctypes
import os
import shutil
import subprocess

import pytest

from test_launch_waits import kernels
from test_prefix_plan import CSRC

SOURCE = r"""
#include <algorithm>
#include <cstdint>
using std::max; using std::min;
#define __host__
#define __device__
#define __forceinline__ inline
#include "prefix_plan_host.h"
extern "C" {
static WalkSteps of(const int* s) { return WalkSteps{s[0], s[1], s[2], s[3], s[4], s[5] != 0}; }
int own(const int* s, int j) { const OwnStep o = walk_own_step(of(s), j); return o.list << 16 | o.k; }
int takes_part(const int* s, int c, int j) { return walk_takes_part(of(s), c, j); }
int behind_other(const int* s, int c, int j, int stages) { return walk_behind_other(of(s), c, j, stages); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("steps")
    (d / "prefix_plan_host.h").write_text(open(os.path.join(CSRC, "prefix_plan.cuh")).read().replace('#include "common.cuh"', "").replace("#pragma once", ""))
    (d / "steps.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(d / "steps.so"), str(d / "steps.cpp")], check=True)
    return ctypes.CDLL(str(d / "steps.so"))


def items():
    """(J, npre, own0, steps0, steps1, both) of ranges of walks: prefix steps, and the steps of two lists."""
    for both in (1, 0):
        for pre in (0, 1, 2, 5):
            for s0 in (0, 1, 2, 3, 6, 9):
                for s1 in (0, 1, 2, 4, 5, 9) if both else (0,):
                    total = pre + s0 + s1
                    for x0 in range(total):
                        for J in {1, 2, 3, (total - x0) // 2, total - x0} & set(range(1, total - x0 + 1)):
                            yield J, max(0, min(J, pre - x0)), x0 - pre, s0, s1, both


def test_the_lists_are_walked_in_order(lib):
    for s0 in range(8):
        for s1 in range(8):
            s = (ctypes.c_int * 6)(s0 + s1, 0, 0, s0, s1, 1)
            seen = [(o >> 16, o & 0xffff) for o in (lib.own(s, j) for j in range(s0 + s1))]
            assert [k for l, k in seen if l == 0] == list(range(s0)) and [k for l, k in seen if l == 1] == list(range(s1))


@pytest.mark.parametrize("stages", [2, 4])
def test_a_chain_knows_what_lay_where_a_step_comes_to(lib, stages):
    """A chain that waits for step j's keys has taken part in the step that lay there before, or waits for the other chain's end -- which does not wait in turn."""
    waits = 0
    for item in items():
        s, J, npre, both = (ctypes.c_int * 6)(*item), item[0], item[1], item[5]
        part = [[bool(lib.takes_part(s, c, j)) for j in range(J)] for c in range(2)]
        for j in range(J):
            assert part[0][j] + part[1][j] == (2 if both and j < npre else 1)
        waiting = set()
        for c in range(2):
            for j in (j for j in range(J) if part[c][j]):
                behind = bool(lib.behind_other(s, c, j, stages))
                assert behind == (j >= stages and not part[c][j - stages]), (item, c, j)
                if behind:
                    assert any(part[1 - c]) and not any(part[1 - c][j:]), (item, c, j)
                    waiting.add(c)
        assert len(waiting) < 2
        waits += len(waiting)
    assert waits > 100                                     # (the case is among them)


def test_the_walk_asks():
    body = next(body for _, name, body in kernels() if name == "prefix_walk_kernel")
    assert body.count("wait_for(&k_full[st]") == 1 and "(!walk_behind_other(steps, mu, j, STAGES) || wait_for(&o_full[mu ^ 1], 0)) && wait_for(&k_full[st]" in body
