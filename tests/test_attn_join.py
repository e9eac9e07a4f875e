"""Who does what in the workgroup that joins the parts of attention rows
(csrc/q4k_join.h), on the CPU: for every head dimension and number of parts each row has its
threads, and no thread reads LDS past the workgroup's own."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemv-q4_k-optimization_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "q4k_join.h"
using namespace q4k;
int main() {
    int cases = 0;
    for (int dim = 4; dim <= 256; dim += 4)
        for (long long parts = 1; parts <= 2048; parts += parts < 40 ? 1 : parts / 3) {
            const JoinSplit s = join_split(dim, parts);
            if (s.groups < 1 || s.rows < 1 || s.groups * s.rows * (dim / 4) > kJoinThreads) return printf("split: dim %d, parts %lld\n", dim, parts), 1;
            int rows = 0, there = 0;
            for (int t = 0; t < kJoinThreads; ++t) {
                const JoinThread me(t, dim, s.groups, s.rows);
                there += me.there;
                if (me.there && (me.which < 0 || me.which >= s.rows || me.sub >= s.groups || me.d4 >= dim / 4)) return printf("thread %d, dim %d\n", t, dim), 1;
                if (!me.collects()) continue;
                rows += me.d4 == 0;
                for (int i = 0; i < s.groups; ++i) {
                    const int at = JoinThread::place(t, dim, i);
                    if (at < 0 || at >= kJoinThreads) return printf("dim %d, %d groups, %d rows: thread %d reads place %d\n", dim, s.groups, s.rows, t, at), 1;
                    const JoinThread other(at, dim, s.groups, s.rows);
                    if (other.which != me.which || other.d4 != me.d4 || other.sub != i) return printf("dim %d: thread %d takes another row's sum\n", dim, t), 1;
                }
            }
            if (rows != s.rows || there != s.groups * s.rows * (dim / 4)) return printf("dim %d, parts %lld: %d rows of %d\n", dim, parts, rows, s.rows), 1;
            ++cases;
        }
    printf("%d cases\n", cases);
    return 0;
}
"""


def test_join_threads_stay_within_their_row(tmp_path):
    (tmp_path / "join.cpp").write_text(PROGRAM)
    exe = str(tmp_path / "join")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(tmp_path / "join.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], stdout=subprocess.PIPE, text=True, timeout=60)
    assert r.returncode == 0 and int(r.stdout.split()[0]) > 1000, r.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 48, 80, 96, 112, 200])
def test_joined_rows_where_threads_are_left_over(Q, gpu, D):
    """Many parts of few rows, of head dimensions that 256 threads do not divide among."""
    import test_gpu_kv8_attn as eight
    import test_gpu_prefix_attn as sixteen
    for prefix, suffix, lens in ((3000, 0, None), (900, 700, [700, 3, 0])):
        sixteen.Case(gpu, 3, 1, 3, 1, D, prefix, suffix, 32, lens=lens, seed=D).check(Q)
    if D % 16 == 0:
        eight.Case(gpu, 3, 1, 3, 1, D, 3000, 64, 32, lens=[3000, 700, 1], seed=D).check(Q)
