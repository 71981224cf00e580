"""How the tokens of a ragged batch are cut into units (csrc/sa_paged_plan.h),
compiled with g++: every token of a right cu_q in exactly one unit, and the
ranges of a wrong one, which may overlap to more units than 31 bits count,
leading to no index outside the tensors."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "streaming_attention_b200", "csrc")

SRC = r"""
#include <cstdio>
#include <vector>
#include "sa_paged_plan.h"
using namespace sa::pg;
// `threads` runs of sequences, as a block searches for its unit
int main() {
    long long n, n_tok, per, threads, k;
    while (scanf("%lld %lld %lld %lld %lld", &n, &n_tok, &per, &threads, &k) == 5) {
        std::vector<int> cu(n + 1);
        for (auto& x : cu) if (scanf("%d", &x) != 1) return 1;
        const long long run = (n + threads - 1) / threads;
        unsigned total = 0;
        std::vector<unsigned> at, mine;
        for (long long t = 0; t < threads; ++t) {
            unsigned m = 0;
            for (long long b = t * run; b < (t + 1) * run && b < n; ++b)
                m = add_units(m, unit_count(token_count(cu[b], cu[b + 1], n_tok), per), threads);
            at.push_back(total);
            mine.push_back(m);
            if (total + m < total) return 2;               // wrapped
            total += m;
        }
        printf("%u", total);
        for (long long i = 0; i < k; ++i) {
            long long w;
            if (scanf("%lld", &w) != 1) return 1;
            const unsigned want = (unsigned)w;
            int found = 0, b = -1;
            unsigned unit = 0;
            for (long long t = 0; t < threads; ++t)
                if (want >= at[t] && want - at[t] < mine[t]) {
                    unsigned a = at[t];
                    b = unit_sequence(cu.data(), t * run, (t + 1) * run < n ? (t + 1) * run : n, n_tok, per, want, &a);
                    unit = want - a;
                    found += b >= 0;
                }
            printf(" %d %d %u", found, b, unit);
        }
        printf("\n");
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_units")
    src, exe = d / "units.cpp", d / "units"
    src.write_text(SRC)
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-fsanitize=undefined,address", "-fno-sanitize-recover", "-Wall",
                    "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)

    def run(cu, n_tok, per, threads, wants):
        line = " ".join(map(str, [len(cu) - 1, n_tok, per, threads, len(wants), *cu, *wants]))
        r = subprocess.run([str(exe)], input=line, capture_output=True, text=True, check=True)
        x = [int(v) for v in r.stdout.split()]
        return x[0], [tuple(x[1 + 3 * i:4 + 3 * i]) for i in range(len(wants))]
    return run


def test_every_token_in_one_unit(ask):
    rng = random.Random(1)
    for _ in range(40):
        new = [rng.choice([0, 0, 1, 5, 64, 65, 200]) for _ in range(rng.randint(1, 30))]
        per, lead = rng.choice([1, 8, 42, 64, 128]), rng.choice([0, 3])
        cu = [lead]
        for n in new:
            cu.append(cu[-1] + n)
        units = sum(-(-n // per) for n in new)
        total, got = ask(cu, cu[-1] + 2, per, rng.choice([1, 3, 256]), list(range(units)))
        assert total == units
        seen = []
        for found, b, unit in got:
            assert found == 1
            seen += [cu[b] + t for t in range(unit * per, min(new[b], (unit + 1) * per))]
        assert sorted(seen) == list(range(lead, cu[-1])) and len(seen) == len(set(seen))


@pytest.mark.parametrize("threads", [256, 384])
@pytest.mark.parametrize("n_tok,per", [(1 << 20, 8), ((1 << 31) - 1, 1), ((1 << 31) - 1, 128), (3 << 20, 42), (100, 64)])
def test_overlapping_ranges(ask, n_tok, per, threads):
    """All tokens, over and over: [0, n), then a range that runs backwards, and so on.  The block's sum does not wrap,
    and each of its units is one of a sequence's."""
    n = 4000
    cu = [0 if i % 2 == 0 else n_tok for i in range(n + 1)]
    each = -(-n_tok // per)
    total, _ = ask(cu, n_tok, per, threads, [])
    assert total <= n // 2 * each and (total == n // 2 * each or total > 1 << 31)
    wants = sorted({0, 1, total // 3, total // 2, total - 2, total - 1})
    for found, b, unit in ask(cu, n_tok, per, threads, wants)[1]:
        assert found == 1 and b % 2 == 0 and unit < each


def test_ranges_outside_the_tensors_count_as_none(ask):
    assert ask([0, 10, 5, 20, 21], 20, 4, 2, [0, 2, 3, 6])[0] == 3 + 4      # [10, 5) and [20, 21) are none
    assert ask([-1, 5, 9], 20, 4, 1, [0])[1] == [(1, 1, 0)]
    assert ask([2 ** 31 - 1, -2 ** 31, 0], 20, 4, 1, [])[0] == 0
