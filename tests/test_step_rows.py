"""Which rows of a step the warps of one-token attention over 8-bit pages look at, gone through on the host."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fieldrun_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "step_rows.h"

int main() {
    const int most = 64;
    for (int rows = 1; rows <= 65535; ++rows) {
        const RowGroups groups = row_groups(rows, most);
        if (groups.steps < 1 || groups.count < 1 || groups.count > most) { printf("%d rows: %d groups of %d steps\n", rows, groups.count, groups.steps); return 1; }
        std::vector<char> seen(rows, 0);
        for (int group = 0; group < groups.count; ++group)
            for (int step = 0; step < groups.steps; ++step) {
                const int b0 = 32 * (group * groups.steps + step);
                for (int lane = 0; lane < 32; ++lane) {
                    const int own = b0 + lane, beside = row_beside(b0, lane, rows);
                    if (own < rows) ++seen[own];
                    // inside the tables, and the neighbour in front of a first row or behind a last one whenever there is one
                    const int want = lane == 0 && own < rows ? own - 1 : lane == 31 && own + 1 < rows ? own + 1 : -1;
                    if (beside >= rows || beside < -1 || beside != want) {
                        printf("%d rows: lane %d of the rows from %d on looks at row %d\n", rows, lane, b0, beside);
                        return 1;
                    }
                }
            }
        for (int row = 0; row < rows; ++row)
            if (seen[row] != 1) { printf("%d rows: row %d is looked at %d times\n", rows, row, seen[row]); return 1; }
    }
    return 0;
}
"""


def test_every_row_is_looked_at_once_and_none_behind_the_last(tmp_path):
    source, program = tmp_path / "rows.cpp", tmp_path / "rows"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", CSRC, str(source), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout
