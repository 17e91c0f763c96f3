"""How linear4 cuts calls of more than 16 rows into tiles (host code, compiled here; runs without a GPU): the tensor cores' shapes, all rows taken, what is laid into tensor and shared memory in its
bounds, and the steps of the warps that make weights."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
#include <stdio.h>
#include <stdlib.h>
#include "linear4_plan.h"
int main() {
    const int fits[3][kLinear4Splits] = {{74, 33, 22, 15}, {66, 30, 20, 14}, {1, 1, 1, 1}}, outs[] = {1, 257, 1001, 4096, 10240, 18944, 120832, 1 << 30}, widths[] = {32, 160, 448, 1056, 4096, 8192, 65536};
    long n = 0;
    for (int rows = 17; rows <= 1 << 24; rows += rows < 2200 ? 1 : rows / 3)
        for (int out : outs) for (int width : widths) for (const auto &fit : fits) for (int wide = 0; wide < 2; wide++) {
            const int m_tiles = (out + 255) / 256, units = (width + 127) / 128, teams = linear4_teams(wide);
            const linear4_plan p = linear4_plan_of(rows, m_tiles, units, wide, fit);
            const int sums = (wide ? 2 : 1) * p.columns;
            const bool right = p.columns % 32 == 0 && p.columns >= 32 && p.columns <= (wide ? 128 : 256)      /* N of a product of two CTAs, M = 256, A in tensor memory */
                && p.tiles == (long long)((rows + p.columns - 1) / p.columns) * m_tiles && p.splits >= 1 && p.splits <= kLinear4Splits && p.splits <= units
                && p.steps >= teams && p.steps <= kLinear4Steps && p.steps * p.columns * 64 <= kLinear4XBytes
                && p.a_column >= sums && p.a_column + p.steps * linear4_a_columns(wide) == kLinear4Tmem;
            /* the teams' steps, through seven tiles of a pair where it has several: each step is one team's, and what a team has seen over rules out that a wait is over two phases early */
            const int steps = 2 * ((units + p.splits - 1) / p.splits), tiles = p.splits == 1 && p.tiles > fit[0] ? 7 : 1;
            if (rows % 7 == 0 && steps < 100) {
                static int taken[7 * 100];
                for (int &t : taken) t = 0;
                for (int team = 0; team < teams; team++) {
                    int s0 = team, last = -1;
                    for (int tile = 0; tile < tiles; tile++) {
                        for (int s = s0; s < steps; s += teams) {
                            const int k = tile * steps + s, gap = k - last;
                            if (last >= 0 && (gap > p.steps || gap + p.steps > 2 * kLinear4Units)) { printf("rows %d out %d width %d wide %d: steps %d apart, %d stages\\n", rows, out, width, wide, gap, p.steps); return 1; }
                            last = k;
                            taken[k]++;
                        }
                        s0 = linear4_first_step(s0, steps, teams);
                    }
                }
                for (int k = 0; k < tiles * steps; k++) if (taken[k] != 1) { printf("step %d is %d teams'\\n", k, taken[k]); return 1; }
            }
            if (!right) { printf("rows %d out %d width %d wide %d: columns %d tiles %lld splits %d steps %d a_column %d\\n", rows, out, width, wide, p.columns, p.tiles, p.splits, p.steps, p.a_column); return 1; }
            n++;
        }
    printf("%ld\\n", n);
    return 0;
}
"""


def test_tiles(tmp_path):
    source, program = tmp_path / "plan.cpp", str(tmp_path / "plan")
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", os.path.join(ROOT, "hy3_b200", "csrc"), str(source), "-o", program], check=True)
    done = subprocess.run([program], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout
    assert int(done.stdout) > 100000
