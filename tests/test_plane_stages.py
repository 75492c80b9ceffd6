"""Which rows the tile loops of plane_gemm.h read where stages end past an operand's k, or lie past it altogether: rows that there are (CPU)."""
import host_probe

SOURCE = r"""
#include <stdio.h>
#include "plane_gemm.h"
// An operand whose stored rows are k (T = 1): stage t of nk from kt0 on has its lanes at rows 0 .. bk-1 of the stage, and those past k at k's last.
int main() {
    long bad = 0, seen = 0;
    for (int bk = 32; bk <= 64; bk *= 2)
        for (int k = 1; k <= 300; k++)
            for (int kt0 = 0; kt0 < 12; kt0++)
                for (int nk = 1; nk < 12; nk++) {
                    const int there = ah::pg::stages_of(k, bk, kt0, nk);
                    if (there > nk) bad++;
                    for (int t = 0; t < nk; t++) {
                        const int kt = kt0 + t, krem = k - kt * bk;
                        if ((t < there) != (krem > 0)) bad++;   // the stages that hold something of it, and no others
                        if (t >= there) continue;
                        for (int kk = 0; kk < bk; kk++, seen++) {
                            const long row = (long)kt * bk + (kk >= krem ? krem - 1 : kk);
                            if (row < 0 || row >= k) bad++;
                        }
                    }
                }
    printf("%ld %ld\n", seen, bad);
}
"""


def test_every_row_read_is_one_of_the_operand(tmp_path):
    seen, bad = map(int, host_probe.run(tmp_path, SOURCE)[0].split())
    assert seen > 10 ** 6 and bad == 0
