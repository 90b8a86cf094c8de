"""The switch that makes waits of int8 products give up, checked without a GPU: nothing is launched."""


def test_blocks_that_are_refused():
    from rexsc_b200 import _lib, build

    build.build()
    lib = _lib.load()
    for block in (-3, 1 << 31, -(1 << 40)):
        assert lib.rexsc_int8_test_waits(block) == -1
    for block in (0, 5, (1 << 31) - 1, -2, -1):
        assert lib.rexsc_int8_test_waits(block) == 0
