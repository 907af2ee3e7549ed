"""The limit of the linear block's waits: argument checks (no GPU)."""
from flashgen_b200 import _lib


def test_set_wait():
    lib = _lib.load()
    for ns, acc in ((-1, -1), (10 ** 9 + 1, -1), (0, -2), (0, 4)):
        assert lib.fg_linear_set_wait(ns, acc) == _lib.FG_EINVAL
    for ns, acc in ((1000, 3), (10 ** 9, 0), (0, -1)):
        assert lib.fg_linear_set_wait(ns, acc) == _lib.FG_OK
