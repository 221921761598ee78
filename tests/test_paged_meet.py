"""The word at which the blocks of a split unit meet: the rules that the kernels go by, compiled for the host, over every order in which
the blocks can arrive, wait (to the end, or until their time is up) and go.  The word has to be zero when all have gone, and no wait may end by
itself before all have arrived."""
import os
import subprocess

import q4gpu

CSRC = os.path.join(os.path.dirname(os.path.dirname(q4gpu.LIB_PATH)), "csrc")
PROGRAM = r"""
#include <stdio.h>
#include <set>
#include <vector>
#include "q4_paged.h"
enum { BEGIN, HERE, DONE_WAITING, GONE };
struct State {
    uint32_t word;
    std::vector<int> at;
    bool operator<(const State &o) const { return word != o.word ? word < o.word : at < o.at; }
};
static std::set<State> seen;
static bool good;
static uint32_t k;
static bool first_joins, first_goes;   /* first_goes: a first that joins nothing counts as gone, as it has to */
static void walk(State s) {
    if (!seen.insert(s).second) return;
    bool over = true;
    for (uint32_t b = 0; b < k; b++) {
        State n = s;
        const bool joins = b || first_joins;
        auto add = [&](uint32_t what) {
            const uint32_t before = n.word;
            n.word += what;
            if (what >= PG_GONE && pg_last_gone(before, first_goes ? k : k - 1u)) n.word = 0;
        };
        switch (s.at[b]) {
        case BEGIN:
            add(joins || first_goes ? pg_arrival(joins) : PG_HERE);
            n.at[b] = joins ? HERE : GONE;
            walk(n);
            break;
        case HERE:
            if (pg_all_here(s.word, k))
                for (int a : s.at) good = good && a != BEGIN;
            n.at[b] = DONE_WAITING;   /* all here, or its time is up */
            walk(n);
            break;
        case DONE_WAITING:
            add(PG_GONE);
            n.at[b] = GONE;
            walk(n);
            break;
        default: continue;
        }
        over = false;
    }
    if (over) good = good && s.word == 0;
}
static bool holds(uint32_t blocks, bool joins, bool goes) {
    seen.clear();
    good = true;
    k = blocks; first_joins = joins; first_goes = goes;
    walk({0u, std::vector<int>(blocks, BEGIN)});
    return good;
}
int main() {
    for (uint32_t blocks = 2; blocks <= 7; blocks++) {
        if (pg_joiners(blocks, true) != blocks || pg_joiners(blocks, false) != blocks - 1u) return printf("joiners of %u\n", blocks), 1;
        if (!holds(blocks, false, true) || !holds(blocks, true, true) || !holds(blocks, pg_first_joins(blocks), true)) return printf("%u blocks: the word does not come back to zero\n", blocks), 1;
        if (blocks > 2u && holds(blocks, false, false)) return printf("%u blocks: the walk does not see a first block that never goes\n", blocks), 1;
    }
    if ((uint64_t)PG_MAX_BLOCKS >= PG_GONE) return printf("more blocks than the halves count\n"), 1;
    printf("ok\n");
    return 0;
}
"""


def test_the_word_comes_back_to_zero(tmp_path):
    src, exe = tmp_path / "meet.cpp", tmp_path / "meet"
    src.write_text(PROGRAM)
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-I", CSRC, "-I", "/usr/local/cuda/include", str(src), "-o", str(exe)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout


WAITS = r"""
#include <stdio.h>
#include "q4_paged.h"
int main() {
    for (uint32_t probes : {0u, 1u, 5u, 4096u})
        for (uint32_t yes : {0u, 1u, 4u, 4095u, 4096u, 0xffffffffu}) {   /* the probe that says so */
            uint32_t n = 0;
            const bool got = pg_within(probes, [&]() { return n++ == yes; });
            if (got != (yes < probes) || n != (got ? yes + 1u : probes)) return printf("%u probes, yes at %u: %d after %u\n", probes, yes, got, n), 1;
        }
    printf("ok\n");
    return 0;
}
"""


def test_a_wait_says_whether_it_ran_out(tmp_path):
    """by it the join of records knows not to store what did not come"""
    src, exe = tmp_path / "waits.cpp", tmp_path / "waits"
    src.write_text(WAITS)
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-I", CSRC, "-I", "/usr/local/cuda/include", str(src), "-o", str(exe)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout
