"""The f16 contraction's L2 prefetch touches four bytes of its operands and nothing behind them, for ragged sizes too (CPU)."""
import host_probe

SOURCE = r"""
#include <stdio.h>
#include "gemm16_kernel.h"
// Every line of every stage of every tile: R tile rows, `rows` operand rows, K a multiple of a stage's 64, rows of `ld` halves.
template <int R, int T>
void check(long &seen, long &bad) {
    for (int rows = 8; rows <= 600; rows += 8)
        for (int K = 64; K <= 192; K += 64)
            for (int gap = 0; gap <= 8; gap += 8) {
                const long ld = (T == 0 ? K : rows) + gap, bytes = T == 0 ? ((rows - 1) * ld + K) * 2 : ((K - 1) * ld + rows) * 2;
                for (int r0 = 0; r0 < rows; r0 += R)
                    for (int k0 = 0; k0 < K; k0 += 64)
                        for (int i = 0; i < R; i++, seen++) {
                            const long at = ah::g16::prefetch_offset<R, T>(ld, r0, rows, k0, i);
                            if (at < 0 || at % 4 || at + 4 > bytes) bad++;
                        }
            }
}
int main() {
    long seen = 0, bad = 0;
    check<128, 0>(seen, bad);
    check<128, 1>(seen, bad);
    check<256, 0>(seen, bad);
    check<256, 1>(seen, bad);
    printf("%ld %ld\n", seen, bad);
}
"""


def test_the_prefetch_stays_inside(tmp_path):
    seen, bad = map(int, host_probe.run(tmp_path, SOURCE)[0].split())
    assert seen > 10 ** 5 and bad == 0
