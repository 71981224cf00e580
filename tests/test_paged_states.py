"""Softmax states of query rows (csrc/sa_paged_plan.h), compiled with g++: what a
row is divided by, and that a row which a kernel gave up on comes out as NaN
whatever it is joined with.  The join is the kernels' formula:
M = max m_i, L = sum 2^(m_i - M) l_i, parts with no weight left out of the O sum."""
import math
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "streaming_attention_b200", "csrc")

SRC = r"""
#include <cmath>
#include <cstdio>
#include "sa_paged_plan.h"
using namespace sa::pg;
int main() {
    int n;
    while (scanf("%d", &n) == 1) {          // n states "m l o"; "x x x": given up, its O whatever lay there (7)
        float m[8], l[8], o[8], M = -INFINITY, L = 0.f, O = 0.f;
        for (int i = 0; i < n; ++i) {
            char w[3][32];
            if (scanf("%31s %31s %31s", w[0], w[1], w[2]) != 3) return 1;
            if (w[0][0] == 'x') { m[i] = given_up().m; l[i] = given_up().l; o[i] = 7.f; }
            else { m[i] = strtof(w[0], 0); l[i] = strtof(w[1], 0); o[i] = strtof(w[2], 0); }
            M = fmaxf(M, m[i]);
        }
        if (M != -INFINITY)
            for (int i = 0; i < n; ++i) {
                const float wt = exp2f(m[i] - M);
                L += wt * l[i];
                if (wt != 0.f) O += wt * o[i];
            }
        printf("%a\n", (double)(O * row_factor(L)));
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_states")
    src, exe = d / "states.cpp", d / "states"
    src.write_text("#include <cstdlib>\n" + SRC)
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)

    def run(states):
        line = f"{len(states)} " + " ".join("x x x" if s is None else "%r %r %r" % s for s in states)
        out = subprocess.run([str(exe)], input=line, capture_output=True, text=True, check=True).stdout.strip()
        return float("nan") if "nan" in out else float.fromhex(out) if "inf" not in out else float(out)
    return run


INF = math.inf


def test_rows_are_divided_by_their_sums(ask):
    assert ask([(3.0, 4.0, 10.0)]) == 2.5
    assert ask([(0.0, 1.0, 2.0), (1.0, 1.0, 5.0)]) == 4.0           # (2/2 + 5) / (1/2 + 1)
    assert ask([(-INF, 0.0, 0.0)]) == 0.0                           # saw nothing
    assert ask([(-INF, 0.0, 0.0), (-INF, 0.0, 0.0)]) == 0.0
    assert ask([(-INF, 0.0, 0.0), (-200.0, 2.0, 3.0)]) == 1.5


@pytest.mark.parametrize("others", [[], [(0.0, 1.0, 1.0)], [(-INF, 0.0, 0.0)], [(500.0, 3.0, 1.0)], [(-500.0, 3.0, 1.0)],
                                    [(-INF, 0.0, 0.0), (120.0, 1e30, 1e30)]])
def test_a_given_up_part_makes_the_row_nan(ask, others):
    for at in range(len(others) + 1):
        assert math.isnan(ask(others[:at] + [None] + others[at:]))


def test_every_kernel_divides_by_the_shared_factor():
    """No kernel of its own makes a NaN sum a zero: the final factor is row_factor's, in the joins, the tensor-core
    kernels and the fp32 tiles."""
    for name, at_least in (("sa_paged.cuh", 1), ("sa_paged_tc.cu", 1), ("sa_paged_f32.cu", 1)):
        src = open(os.path.join(CSRC, name)).read()
        assert src.count("row_factor(") >= at_least and "> 0.f ? 1.f /" not in src, name
    tc = open(os.path.join(CSRC, "sa_paged_tc.cu")).read()
    assert "given_up().l" in tc
