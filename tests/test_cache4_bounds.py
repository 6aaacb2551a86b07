"""What the 4-bit ring's entries take and refuse at the ends of their ranges, on
the CPU against the stand-in runtime."""
import ctypes

import pytest

from igllm_amd import native
from test_cache4_host import Host, lib  # noqa: F401 (a fixture)

INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def host(lib):  # noqa: F811
    return Host(lib)


def takes(lib, span):  # noqa: F811
    c = native.Cache4(0, span, 0, 1, 64, 1.0, 1.0)
    return lib.igl_cache4_code_bytes(ctypes.byref(c)) > 0


def test_the_longest_rings_blocks_end_below_an_int(lib):  # noqa: F811
    """The attention counts slots in ints to the end of its last block, of 512 slots
    where a ring is long: past the largest int it would take that block for whole and
    read rows behind the ring."""
    low, high = 1, INT_MAX
    while low < high:
        mid = (low + high + 1) // 2
        low, high = (mid, high) if takes(lib, mid) else (low, mid - 1)
    assert low >= INT_MAX - 4096 and not takes(lib, low + 1) and not takes(lib, INT_MAX)
    lib.plan4_form.restype, lib.plan4_form.argtypes = ctypes.c_int, [ctypes.c_int] * 8
    assert lib.plan4_form(64, 1, low, 0, 1, low - 1, 0, 1) % 4 == 3  # blocks of 512
    assert (low - 1) // 512 * 512 + 512 <= INT_MAX
