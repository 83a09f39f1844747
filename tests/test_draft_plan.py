"""The cut of a sequence's pages into segments and the room for their partial results, from the kernels' own header, compiled for
the host."""
import subprocess

from lumenllm_b200.csrc import build

PROGRAM = r"""
#include "tree_plan.cuh"
#include <cstdio>
#include <random>
#include <vector>
static int fail(const char* what, int a, int b, int c, int d) { printf("%s: %d %d %d %d\n", what, a, b, c, d); return 1; }
int main() {
    std::mt19937 rng(0);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    const int groups[] = {1, 2, 3, 4, 5, 8, 16, 40};
    for (int round = 0; round < 20000; ++round) {
        // a step as the kernels see it: lengths inside a page table, tokens inside N
        const int width = round % 3 ? pick(1, 40) : pick(1, 3000), G = groups[rng() % 8], B = pick(1, 6);
        const bool mma = rng() & 1;
        const int seg_min = mma ? TREE_MMA_MIN_SEG : TREE_MIN_SEG, seg_rows = mma ? TREE_MMA_SEG_ROWS : TREE_SEG_ROWS;
        std::vector<TreeSeq> s(B);
        int N = 0;
        for (auto& x : s) {
            x.n0 = N;
            x.q = rng() % 4 ? pick(1, 40) : pick(1, 600);
            x.start = pick(0, width * LUMEN_PAGE);
            x.end = x.q > width * LUMEN_PAGE - x.start ? width * LUMEN_PAGE : x.start + x.q;
            N += x.q;
        }
        N += pick(0, 5);
        const long long room = tree_pairs(B, N, width, G);
        long long behind = 0;                        // one past the last pair of the sequences before
        for (int b = 0; b < B; ++b) {
            const int window = rng() % 2 ? 0 : pick(1, 1 << pick(1, 18));
            const TreePlan p = tree_plan(s[b], window, G, seg_min, seg_rows);
            if (p.nseg < 1 || p.nseg > tree_max_segs(width)) return fail("segments beyond those launched", p.nseg, width, s[b].q, G);
            int next = p.pg_lo;
            for (int i = 0; i < p.nseg; ++i) {
                if (p.first(i) != next || p.count(i) < 1) return fail("a page left out, or twice", i, p.first(i), next, p.count(i));
                next += p.count(i);
            }
            if (next != p.pg_lo + p.np || next > width || p.pg_lo < 0) return fail("pages outside the table", p.pg_lo, p.np, next, width);
            if (s[b].end > 0 && next != (s[b].end - 1) / LUMEN_PAGE + 1) return fail("not to the last key", next, s[b].end, 0, 0);
            const int first_seen = window > 0 && s[b].start - window + 1 > 0 ? s[b].start - window + 1 : 0;
            if (p.pg_lo * LUMEN_PAGE > first_seen) return fail("not from the first key", p.pg_lo, s[b].start, window, 0);
            if (p.nseg == 1) continue;
            const long long base = tree_part_base(b, s[b].n0, width, G), end = base + (long long)s[b].q * p.nseg;
            if (base < behind) return fail("pairs of two sequences", b, s[b].q, p.nseg, width);
            if (end > room) return fail("pairs beyond the room", b, s[b].q, p.nseg, width);
            behind = end;
        }
    }
    return 0;
}
"""


def test_segments_fit_their_room_and_cover_every_page(tmp_path):
    """20,000 random steps of both kernels that cut a sequence by its own length."""
    (tmp_path / "plan.cu").write_text(PROGRAM)
    flags = [f for f in build.NVCC_FLAGS if f not in ("-shared", "-Xcompiler", "-fPIC")]
    made = subprocess.run([build._nvcc(), *flags, "-I", str(build.CSRC), "-o", str(tmp_path / "plan"), str(tmp_path / "plan.cu")],
                          capture_output=True, text=True)
    assert made.returncode == 0, made.stdout + made.stderr
    ran = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout
