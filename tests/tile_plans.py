"""How the linear layer's products are cut into tiles: asked of the planners themselves, in the kernels' sources, on the host alone."""
import host_probe

FORWARD = r"""
#include <stdio.h>
#include <stdlib.h>
#include "linear.hip"
int main(int n, char **v) {
    for (int i = 1; i + 3 < n; i += 4) {
        ah_linear_desc d{};
        d.dtype = atoi(v[i]);
        d.N = atoi(v[i + 1]), d.D = atoi(v[i + 2]), d.F = atoi(v[i + 3]);
        d.ldx = d.ldw = d.D;
        d.ldu = d.ldr = d.ldy = d.ldz = d.F;
        const auto l = ah::layout(d);
        if (l.few) {
            printf("few %d\n", l.few);
            continue;
        }
        const auto p = ah::plan_of(d, l);
        printf("%d %d %d %d %d\n", p.width, p.w.whole, p.w.rest, p.w.splits, l.Dp / (l.P == 1 ? 64 : 32));
    }
}
"""

BACKWARD = r"""
#include <stdio.h>
#include <stdlib.h>
#include "linear_grad.hip"
int main(int n, char **v) {
    for (int i = 1; i + 4 < n; i += 5) {
        ah_linear_grad_desc d{};
        d.dtype = atoi(v[i]), d.grad_dtype = atoi(v[i + 1]);
        d.N = atoi(v[i + 2]), d.D = atoi(v[i + 3]), d.F = atoi(v[i + 4]);
        d.act = AH_ACT_GELU;
        d.ldx = d.ldw = d.lddx = d.lddw = d.D;
        d.ldu = d.ldz = d.lddy = d.lddu = d.F;
        d.X = d.W = d.Z = d.U = d.dY = d.dX = d.dW = d.dbias = (float *)256;   // (never read)
        d.dU = d.dX;
        const auto l = ah::layout(d);
        const int bk = l.P == 1 ? 64 : 32;
        printf("%d %d %d %d %d %d %d %d\n", l.few ? 0 : l.cuts.x.width, l.cuts.x.w.splits, (d.F + bk - 1) / bk, l.cuts.w.width, l.cuts.w.w.splits, (d.N + bk - 1) / bk, l.exact,
               l.track);
    }
}
"""


def forward(tmp_path, cases):
    """(dtype, N, D, F) each: "few" or (width, whole tiles, split tiles, splits, stages)."""
    out = host_probe.run(tmp_path, FORWARD, *[x for c in cases for x in c])
    return ["few" if o.startswith("few") else tuple(map(int, o.split())) for o in out]


def backward(tmp_path, cases):
    """(dtype, grad_dtype, N, D, F) each: widths (0: few rows), splits and stages of dX and dW, and how dZ's largest magnitude is found."""
    keys = ("x_width", "x_splits", "x_stages", "w_width", "w_splits", "w_stages", "exact", "track")
    return [dict(zip(keys, map(int, o.split()))) for o in host_probe.run(tmp_path, BACKWARD, *[x for c in cases for x in c])]


# Shapes that the planners send to each kind of tile loop, with ragged ends. Forward: (dtype, N, D, F): (width, kind); whole: a tile a workgroup, split: K over
# several and joined, mixed: some of each. 256-wide tiles of f16 have 1 to 6 stages among them.
FORWARD_SHAPES = {
    (0, 156, 9, 106): (64, "whole"), (0, 194, 665, 107): (64, "split"), (0, 2738, 1419, 748): (64, "mixed"),
    (0, 196, 17, 8571): (128, "whole"), (0, 1601, 2138, 584): (128, "split"), (0, 1781, 705, 4631): (128, "mixed"),
    (0, 1079, 19, 7249): (256, "whole"), (0, 3478, 3049, 1355): (256, "split"), (0, 1941, 511, 8256): (256, "mixed"),
    (1, 146, 17, 108): (64, "whole"), (1, 138, 1950, 105): (64, "split"), (1, 895, 1958, 2321): (64, "mixed"),
    (1, 264, 21, 6596): (128, "whole"), (1, 934, 6553, 1149): (128, "split"), (1, 2397, 782, 6912): (128, "mixed"),
    (1, 2205, 7689, 1400): (256, "split"), (1, 4434, 1036, 3807): (256, "mixed"),
    **{(1, 2100, d, 4100): (256, "whole") for d in (40, 128, 190, 256, 300, 384)},
}
# Backward: (dtype, grad_dtype, N, D, F): (dX's width, whether it is split, dW's, whether); width 0: few rows.
BACKWARD_SHAPES = {
    (0, 0, 157, 24, 100): (64, False, 64, False), (0, 0, 642, 14, 109): (64, True, 64, True), (0, 0, 135, 25, 484): (64, False, 128, False),
    (0, 0, 408, 24, 100): (128, False, 64, False), (0, 0, 2571, 778, 588): (128, False, 128, True), (0, 0, 1281, 763, 1457): (128, True, 128, True),
    (0, 0, 95, 4185, 1838): (0, False, 256, False), (0, 0, 3613, 1526, 211): (256, False, 256, True), (0, 0, 1187, 2391, 3212): (256, True, 256, False),
    (1, 0, 83, 19, 103): (128, False, 128, False), (1, 0, 102, 8, 424): (128, True, 128, True), (1, 0, 1693, 3600, 169): (256, False, 256, True),
    (1, 0, 680, 1191, 4774): (256, True, 256, False),
    (1, 1, 83, 19, 103): (128, False, 128, False), (1, 1, 65, 8, 686): (128, True, 128, False), (1, 1, 571, 31, 107): (128, False, 128, True),
    (1, 1, 50, 859, 8658): (0, False, 256, False), (1, 1, 190, 1943, 7747): (256, True, 256, False), (1, 1, 250, 2244, 6524): (256, True, 256, False),
    (1, 1, 320, 3329, 6227): (256, True, 256, False), (1, 1, 380, 3346, 7581): (256, True, 256, False), (1, 1, 1545, 3385, 646): (256, False, 256, False),
    (1, 1, 1693, 3600, 169): (256, False, 256, True), (1, 1, 1693, 3600, 230): (256, False, 256, True), (1, 1, 1693, 3600, 380): (256, False, 256, True),
}
