"""The shapes that test_gpu_linear_tiles.py runs go to the tile loops that it means to test (CPU): every width, whole and split, in each direction and
type. A change to the planners' model of time that sends one elsewhere shows here."""
import tile_plans as T

F32, F16 = 0, 1


def test_forward(tmp_path):
    got = T.forward(tmp_path, T.FORWARD_SHAPES)
    for (case, want), plan in zip(T.FORWARD_SHAPES.items(), got):
        assert plan != "few", case
        width, whole, rest, splits, _ = plan
        kind = "whole" if splits == 1 else "mixed" if whole else "split"
        assert rest == 0 or splits > 1, case
        assert (width, kind) == want, (case, plan)
    kinds = {(c[0],) + k for c, k in T.FORWARD_SHAPES.items()}
    assert kinds == {(t, w, k) for t in (F32, F16) for w in (64, 128, 256) for k in ("whole", "split", "mixed")}
    stages = {p[4] for c, p in zip(T.FORWARD_SHAPES, got) if c[0] == F16 and p[0] == 256}
    assert {1, 2, 3, 4, 5, 6} <= stages


def test_backward(tmp_path):
    got = T.backward(tmp_path, T.BACKWARD_SHAPES)
    for (case, want), p in zip(T.BACKWARD_SHAPES.items(), got):
        assert (p["x_width"], p["x_splits"] > 1, p["w_width"], p["w_splits"] > 1) == want, (case, p)
    for types in ((F32, F32), (F16, F32), (F16, F16)):
        wide = {64, 128, 256} if types[0] == F32 else {128, 256}
        mine = [w for c, w in T.BACKWARD_SHAPES.items() if c[:2] == types]
        for at in (0, 2):
            assert {(w[at], w[at + 1]) for w in mine if w[at]} == {(w, s) for w in wide for s in (False, True)}, types
    assert {p["w_stages"] for c, p in zip(T.BACKWARD_SHAPES, got) if c[:2] == (F16, F16) and p["w_width"] == 256} >= {1, 3, 4, 5, 6}
    # dZ's largest magnitude is scanned for in some and bounded first in others
    assert {p["exact"] for p in got} == {0, 1} and all(p["exact"] != p["track"] for p in got)
