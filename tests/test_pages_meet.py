"""The word at which release's blocks meet twice: the rules that the kernel goes by, compiled for the host, over every order in which blocks come, find something bad, wait (to the
end, or until their time is up) and go on.  All have to decide alike, whenever they look: one that lowers a page's holders where another leaves the stack as it is
would lose the page.  They go on exactly where all came in time and none found anything bad."""
import os
import subprocess

import q4gpu

CSRC = os.path.join(os.path.dirname(os.path.dirname(q4gpu.LIB_PATH)), "csrc")
PROGRAM = r"""
#include <stdio.h>
#include <set>
#include <vector>
#include "q4_pages_scan.h"
enum { BEGIN, FIRST, BETWEEN, SECOND, WELL, ILL };
struct State {
    uint32_t word;
    bool late;                 /* somebody's time was up before all had come */
    std::vector<int> at;
    bool operator<(const State &o) const { return word != o.word ? word < o.word : late != o.late ? late < o.late : at < o.at; }
};
static std::set<State> seen;
static bool good, looks;       /* looks: one that gives up looks whether all have come in the same step, as it has to */
static uint32_t k, bad_first, bad_second, over;
static bool in_time;           /* nobody's time is up */
static void walk(State s) {
    if (!seen.insert(s).second) return;
    bool end = true;
    for (uint32_t b = 0; b < k; b++) {
        const uint32_t times = s.at[b] == FIRST ? 1u : 2u;
        const bool first = s.at[b] == FIRST;
        State n = s;
        switch (s.at[b]) {
        case BEGIN:
        case BETWEEN:
            if ((s.at[b] == BEGIN ? bad_first : bad_second) >> b & 1u) n.word |= MEET_BAD;
            n.word += MEET_HERE;
            n.at[b] = s.at[b] == BEGIN ? FIRST : SECOND;
            end = false;
            walk(n);
            break;
        case FIRST:
        case SECOND:
            if (meet_over(s.word, k, times)) {
                if (!(s.word & MEET_LATE))   /* else what has come a second time counts too, and nothing comes of the call */
                    for (int a : s.at) good = good && (first ? a != BEGIN : a >= SECOND);
                n.at[b] = first ? BETWEEN : meet_good(s.word, k) ? WELL : ILL;
                end = false;
                walk(n);
            }
            if (!in_time) {
                n = s;
                n.late |= !meet_came(s.word, k, times);
                n.word = looks ? meet_given_up(s.word, k, times) : s.word | MEET_LATE;
                n.at[b] = first ? BETWEEN : meet_good(n.word, k) ? WELL : ILL;
                end = false;
                walk(n);
            }
            break;
        default: break;
        }
    }
    if (!end) return;
    over++;
    const bool well = !s.late && !bad_first && !bad_second;
    for (int a : s.at) good = good && a == (well ? WELL : ILL);
}
static bool holds(uint32_t blocks, uint32_t first, uint32_t second, bool no_time_up, bool with_looking) {
    seen.clear();
    good = true;
    over = 0;
    k = blocks; bad_first = first; bad_second = second; in_time = no_time_up; looks = with_looking;
    walk({0u, false, std::vector<int>(blocks, BEGIN)});
    return good && over > 0;
}
int main() {
    for (uint32_t blocks = 2; blocks <= 5; blocks++)
        for (uint32_t first = 0; first < 4; first++)
            for (uint32_t second = 0; second < 4; second++)
                for (int in = 0; in < 2; in++)
                    if (!holds(blocks, first, second, in, true)) return printf("%u blocks, bad %u and %u, %s: they do not decide alike\n", blocks, first, second, in ? "in time" : "late"), 1;
    for (uint32_t blocks = 2; blocks <= 5; blocks++)
        if (holds(blocks, 0u, 0u, false, false)) return printf("%u blocks: the walk does not see one that gives up behind the others' decision\n", blocks), 1;
    if (meet_came(MEET_BAD | MEET_LATE | 2047u, 1024u, 2u) || !meet_came(MEET_BAD | MEET_LATE | 2048u, 1024u, 2u)) return printf("the flags are counted as blocks\n"), 1;
    printf("ok\n");
    return 0;
}
"""


def test_all_blocks_decide_alike(tmp_path):
    src, exe = tmp_path / "meet.cpp", tmp_path / "meet"
    src.write_text(PROGRAM)
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-I", CSRC, "-I", "/usr/local/cuda/include", str(src), "-o", str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout
