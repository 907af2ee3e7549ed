"""The limit of the LM head's waits: argument checks (no GPU)."""
from flashgen_b200 import _lib


def test_set_wait():
    lib = _lib.load()
    for ns, acc in ((-1, -1), (10 ** 9 + 1, -1), (0, -2), (0, 8)):
        assert lib.fg_adapter_set_wait(ns, acc) == _lib.FG_EINVAL
    for ns, acc in ((1000, 7), (10 ** 9, 0), (0, -1)):
        assert lib.fg_adapter_set_wait(ns, acc) == _lib.FG_OK
