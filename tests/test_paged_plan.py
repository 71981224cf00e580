"""The paged operators' arithmetic (csrc/sa_paged_plan.h) compiled with g++ and
enumerated on the CPU: every visible row in exactly one tile, no page without a
visible row copied, the batch's tiles shared out without gap or overlap, bad
lengths and pages caught, appended tokens at their rows."""
import os
import random
import subprocess

import pytest

from _paged import sees

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "streaming_attention_b200", "csrc")

SRC = r"""
#include <cstdio>
#include <cstring>
#include "sa_paged_plan.h"
using namespace sa::pg;
int main() {
    char op[16];
    while (scanf("%15s", op) == 1) {
        if (!strcmp(op, "tiles")) {
            int len, w, s, tk;
            if (scanf("%d %d %d %d", &len, &w, &s, &tk) != 4) return 1;
            Tiles t = make_tiles(len, w, s, tk);
            printf("%d", t.n);
            for (int i = 0; i < t.n; ++i) {
                printf(" %d", t.row0(i, tk));
                for (int r = t.row0(i, tk); r < t.row0(i, tk) + tk; r += 16) printf(" %d", t.any(r, 16) | (t.all(r, 16) << 1));
                for (int r = t.row0(i, tk); r < t.row0(i, tk) + tk; ++r) printf(" %d", (int)t.sees(r));
            }
            printf("\n");
        } else if (!strcmp(op, "unit")) {
            int p0, l0, l1, w, s, tk;
            if (scanf("%d %d %d %d %d %d", &p0, &l0, &l1, &w, &s, &tk) != 6) return 1;
            UnitTiles u = make_unit(p0, l0, l1, w, s, tk);
            printf("%d %d %d", u.t.n, u.n[0], u.n[1]);
            for (int i = 0; i < u.t.n; ++i) {
                printf(" %d", u.t.row0(i, tk));
                for (int r = u.t.row0(i, tk); r < u.t.row0(i, tk) + tk; ++r) printf(" %d", (int)u.t.sees(r));
            }
            printf("\n");
        } else if (!strcmp(op, "share")) {
            long long total, n;
            if (scanf("%lld %lld", &total, &n) != 2) return 1;
            for (long long c = 0; c <= n; ++c) printf("%lld ", share_first(c, total, n));
            for (long long t = 0; t < total; ++t) printf("%d ", share_of(t, total, n));
            printf("\n");
        } else if (!strcmp(op, "row")) {
            int len, n, t, mp, pl;
            long long p0, np;
            if (scanf("%d %d %d %d %d %lld %lld", &len, &n, &t, &mp, &pl, &p0, &np) != 7) return 1;
            printf("%lld\n", append_row(len, n, t, mp, pl, p0, np));
        } else if (!strcmp(op, "cut")) {
            int len, mp, pl;
            if (scanf("%d %d %d", &len, &mp, &pl) != 3) return 1;
            printf("%d\n", cut_len(len, mp, pl));
        } else if (!strcmp(op, "page")) {
            int e, n;
            if (scanf("%d %d", &e, &n) != 2) return 1;
            printf("%d\n", (int)page_ok(e, n));
        }
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_plan")
    src, exe = d / "plan.cpp", d / "plan"
    src.write_text(SRC)
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall",
                    "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)

    def run(lines):
        r = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True)
        return [[int(x) for x in line.split()] for line in r.stdout.splitlines()]
    return run


def test_tiles_cover_what_is_seen_once(ask):
    rng = random.Random(1)
    cases = [(n, w, s, tk) for tk in (16, 32, 64, 128) for n in (0, 1, 15, 64, 65, 128, 129, 300)
             for w in (0, 1, 16, 63, 64, 100, 299, 300, 301) for s in (0, 1, 4, 64, 130, 500)]
    cases += [(rng.randint(0, 1000), rng.randint(0, 1000), rng.randint(0, 300), rng.choice([16, 32, 64, 128]))
              for _ in range(300)]
    for (n, w, s, tk), got in zip(cases, ask(f"tiles {a} {b} {c} {d}" for a, b, c, d in cases)):
        seen = [j for j in range(n) if sees(n - 1, j, w, s)]
        per, rows, starts = 1 + tk // 16 + tk, [], []
        assert len(got) == 1 + got[0] * per
        for i in range(got[0]):
            part = got[1 + i * per:1 + (i + 1) * per]
            r0, groups, flags = part[0], part[1:1 + tk // 16], part[1 + tk // 16:]
            assert r0 % tk == 0 and any(flags)            # no tile without a visible row
            starts.append(r0)
            rows += [r0 + x for x, f in enumerate(flags) if f]
            for gi, f in enumerate(groups):               # the 16-row flags agree with the rows
                part16 = flags[gi * 16:gi * 16 + 16]
                assert bool(f & 1) == any(part16) and bool(f & 2) == all(part16)
        assert rows == seen, (n, w, s, tk)
        assert starts == sorted(set(starts))


def test_units_hold_what_their_queries_see(ask):
    """Two slots of consecutive queries: every row that a slot's query sees lies in the slot's tiles, tiles come once
    and in order, and a row that no query sees is not asked for unless it lies between rows of the window."""
    rng = random.Random(2)
    cases = []
    for _ in range(400):
        n0, n1 = rng.randint(1, 40), rng.randint(0, 40)
        p0 = rng.choice([0, 0, rng.randint(-60, 400)])
        last0 = max(-1, p0 + n0 - 1)
        last1 = max(-1, p0 + n0 + n1 - 1) if n1 else -1
        cases.append((p0, last0, last1, rng.choice([0, 1, 30, 64, 200]), rng.choice([0, 1, 4, 64, 100]),
                      rng.choice([16, 64, 128]), n0, n1))
    for (p0, last0, last1, w, s, tk, n0, n1), got in zip(cases, ask("unit %d %d %d %d %d %d" % c[:6] for c in cases)):
        n = got[:3]
        per = 1 + tk
        tiles = [got[3 + i * per:3 + (i + 1) * per] for i in range(n[0])]
        starts = [x[0] for x in tiles]
        assert starts == sorted(set(starts)) and all(x % tk == 0 for x in starts) and n[0] == max(n[1:])
        asked = {x[0] + i for x in tiles for i, f in enumerate(x[1:]) if f}
        for slot, (a, b) in enumerate(((p0, p0 + n0), (p0 + n0, p0 + n0 + n1))):
            mine = {x + i for x in starts[:n[1 + slot]] for i in range(tk)}
            for p in range(a, b):
                seen = {j for j in range(max(0, p + 1)) if sees(p, j, w, s)}
                assert seen <= mine and seen <= asked
        top = max(last0, last1)
        lo = max(0, max(p0, 0) - w + 1) if w else 0
        assert all(j <= top and (j >= lo or j < s) for j in asked)


def test_tiles_of_the_longest_sequences(ask):
    big = 2 ** 31 - 1 - 512
    got = ask([f"tiles {big} 100 4 64"])[0]
    assert got[0] <= 4 and got[1] == 0 and got[1 + 1 + 4 + 64] == (big - 100) // 64 * 64


@pytest.mark.parametrize("n", [1, 2, 7, 148, 296])
def test_shares(ask, n):
    for total in [x for x in (1, 2, 7, 148, 149, 296, 297, 1000, 5003) if x >= n]:
        got = ask([f"share {total} {n}"])[0]
        first, owner = got[:n + 1], got[n + 1:]
        assert first[0] == 0 and first[-1] == total and all(a < b for a, b in zip(first, first[1:]))
        assert max(b - a for a, b in zip(first, first[1:])) <= -(-total // n)
        for c in range(n):
            assert owner[first[c]:first[c + 1]] == [c] * (first[c + 1] - first[c])


def test_rows_lengths_and_pages(ask):
    # len n t max_pages page_log2 pos0 n_pos
    assert ask(["row 10 1 0 1 4 0 100", "row 10 3 0 1 4 0 100", "row 2 3 0 1 4 0 100", "row 17 1 0 1 4 0 100",
                "row 16 1 0 1 4 0 100", "row 10 1 0 1 4 91 100", "row 10 1 0 1 4 90 100",
                "row 2147483647 1 0 134217728 4 0 1099511627776"]) == \
        [[9], [7], [-1], [-1], [15], [-1], [9], [2147483646]]
    assert ask(["cut 5 1 4", "cut 17 1 4", "cut -3 1 4", "cut 5 0 4", "cut 2147483647 134217727 4"]) == \
        [[5], [16], [0], [0], [2147483632]]
    assert ask(["page -1 4", "page 0 4", "page 3 4", "page 4 4", "page -2147483648 4"]) == [[0], [1], [1], [0], [0]]
