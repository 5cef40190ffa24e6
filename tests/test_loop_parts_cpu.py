"""Loops that are cut over a cluster's CTAs: the size is one that the device can launch (tests/csrc/loop_parts_probe.cu; no GPU)."""
import ctypes

import pytest

from dscuda_b200.library import build_directory

HELD = {1: 148, 2: 74, 3: 45, 4: 33, 5: 26, 6: 22, 7: 15, 8: 15, 16: 7}     # a whole B200, one CTA to an SM


@pytest.fixture(scope="module")
def parts():
    lib = ctypes.CDLL(str(build_directory() / "libdscuda_test_probes.so"))
    lib.dscuda_test_loop_parts.argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_double, ctypes.POINTER(ctypes.c_int)]

    def call(ctas, tiles, held, tile_us=0.75):
        return lib.dscuda_test_loop_parts(ctas, tiles, tile_us, (ctypes.c_int * 17)(*[held.get(n, 0) for n in range(17)]))
    return call


def test_a_whole_device(parts):
    assert parts(2, 63, HELD) == 16 and parts(15, 1000, HELD) in (7, 8) and parts(148, 1000, HELD) == 1 and parts(1, 1, HELD) == 1
    # 180 loops for 148 SMs: cut, over several waves
    assert parts(180, 190, HELD) > 1


@pytest.mark.parametrize("missing", [{16}, {7, 8, 16}, {2, 3, 4, 5, 6, 7, 8, 16}])
def test_sizes_that_the_device_does_not_hold(parts, missing):
    held = {n: count for n, count in HELD.items() if n not in missing}
    for ctas in (1, 2, 7, 15, 16, 40, 100, 180, 400):
        for tiles in (1, 2, 5, 8, 16, 63, 1000):
            assert parts(ctas, tiles, held) in held
    assert parts(2, 63, held) == max(held)


def test_a_small_partition(parts):
    """A few SMs: fewer clusters at a time, more waves, and never a size that waits for SMs that are not there."""
    held = {1: 14, 2: 7, 3: 4, 4: 3}
    assert parts(2, 63, held) in (2, 3, 4) and parts(14, 63, held) == 1
