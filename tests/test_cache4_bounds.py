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


def test_launches_of_too_many_threads_are_refused_before(lib, tmp_path):  # noqa: F811
    """A grid has fewer than 2^32 threads: rows of 32 dims and more are laid and read by
    a thread every eight values, attended by 256 every sixteen rows.  The last call
    that fits is launched, the next refused as unsupported, neither as the device's
    failure.  The pointers are no memory; nothing on the host follows them."""
    import os
    import shutil
    import test_cache4_host as t

    so = shutil.copy(os.path.join(t.HERE, "host4", "_build", "libhost4.so"), tmp_path / "libhost4.so")
    own = ctypes.CDLL(str(so))  # its own counts: the stand-in notes that these buffers are none
    for name, (res, args) in native.SIGNATURES.items():
        getattr(own, name).restype, getattr(own, name).argtypes = res, args
    own.audit_report.restype, own.audit_report.argtypes = ctypes.c_long, [ctypes.POINTER(ctypes.c_long)] * 2
    host = Host(own)
    at = 1 << 40
    for head, kv in ((64, 1), (512, 1), (128, 3)):
        c = native.Cache4(0, INT_MAX - 4096, 0, kv, head, 1.0, 1.0, at, at, at, at)
        width = kv * head
        most = ((1 << 24) - 1) * 256 // (width // 8)  # rows
        for lanes, code in ((most, native.IGL_OKAY), (most + 1, native.IGL_FAIL_SUPPORT)):
            before = host.launches()[0]
            assert host.lay(c, at, at, width, 0, lanes) == code
            assert host.take() == code
            assert host.read(c, 0, lanes, at, at, width) == code
            assert host.take() == code
            assert host.launches()[0] - before == (2 if code == native.IGL_OKAY else 0)
    c = native.Cache4(0, INT_MAX - 4096, 0, 1, 64, 1.0, 1.0, at, at, at, at)
    for share, lanes, code in ((16, (1 << 24) - 1, native.IGL_OKAY), (1, (1 << 28) - 16, native.IGL_OKAY),
                               (1, (1 << 28) - 15, native.IGL_FAIL_SUPPORT), (3, 89478481, native.IGL_FAIL_SUPPORT)):
        before = host.launches()[0]
        assert host.attend(c, share, at, 64 * share, 0, 0, lanes, at) == code, (share, lanes)
        assert host.take() == code
        assert (host.launches()[0] > before) == (code == native.IGL_OKAY)
        assert ((lanes * share + 15) // 16 * 256 < 1 << 32) == (code == native.IGL_OKAY)


@pytest.mark.parametrize("window,sinks,lanes", [(512, 4, 1), (512, 4, 5), (60, 0, 16), (1, 3, 1)])
def test_a_session_on_the_shortest_ring_of_a_window(host, window, sinks, lanes):
    """sink_count + window + lanes - 1 slots carry a session of blocks of `lanes` as far
    as it goes; with one less it ends where the ring wraps."""
    for span, ends in ((sinks + window + lanes - 1, False), (sinks + window + lanes - 2, True)):
        if span <= sinks:
            continue
        c = host.ring(1, span, sinks, 1, 256)
        rows, heads = host.alloc(lanes * 256 * 4), host.alloc(lanes * 2048 * 4)
        codes = []
        for place in range(0, 3 * (span + lanes), lanes):
            assert host.lay(c, rows, rows, 256, place, lanes) == native.IGL_OKAY
            codes.append(host.attend(c, 8, heads, 2048, place, window, lanes, heads))
            host.take()
        assert (native.IGL_FAIL_ARGUMENT in codes) == ends
        assert codes[0] == native.IGL_OKAY and (codes[-1] == native.IGL_OKAY) != ends
    assert host.launches()[1] == 0


def test_a_desk_without_room_for_partials_opens(lib):  # noqa: F811
    """Where the device has no 48 MiB left a desk opens as before there were any, and
    attention over the ring runs in one launch, without partials.  In a process of
    its own, whose memory is bounded; the stand-in notes the missing buffer, which the
    launch does not use."""
    import subprocess
    import sys
    import test_cache4_host as t

    script = r"""
import ctypes, resource, sys
sys.path.insert(0, sys.argv[1]); sys.path.insert(0, sys.argv[2])
import test_cache4_host as t
from igllm_amd import native
lib = ctypes.CDLL(t.os.path.join(t.HERE, "host4", "_build", "libhost4.so"))
for name, (res, args) in native.SIGNATURES.items():
    getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
lib.audit_report.restype, lib.audit_report.argtypes = ctypes.c_long, [ctypes.POINTER(ctypes.c_long)] * 2
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (32 << 20),) * 2)
host = t.Host(lib)
c = host.ring(0, 16384)
room = host.alloc(8 * 256 * 4)
before = host.launches()[0]
assert host.attend(c, 8, room, 2048, 16383, 0, 1, room) == native.IGL_OKAY
print("launches", host.launches()[0] - before)
"""
    r = subprocess.run([sys.executable, "-c", script, t.HERE, t.os.path.dirname(t.HERE)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "launches 1\n", (r.stdout, r.stderr[-1500:])


@pytest.mark.parametrize("form,plan", [
    (3, (64, 2, 131072, 0, 8, 131071, 0, 1)), (3, (128, 2, 131072, 0, 4, 131071, 0, 1)),
    (3, (128, 8, 32768, 0, 4, 32767, 0, 1)), (3, (64, 8, 32768, 0, 1, 90000, 32768, 1)),
    (3, (128, 8, 131072, 0, 4, 131071, 0, 1)), (3, (128, 8, 200000, 0, 4, 199999, 0, 1)),
    (2, (64, 8, 40000, 0, 1, 39999, 0, 1)),   # a workgroup would have more slots
    (2, (128, 8, 66000, 0, 4, 65999, 0, 1)), (2, (64, 8, 66000, 0, 4, 65999, 0, 1)),
    (2, (128, 8, 105000, 0, 4, 104999, 0, 1)),
    (2, (128, 2, 65536, 0, 4, 65535, 0, 1)),  # or one block
    (2, (256, 8, 65536, 0, 8, 65535, 0, 1))])  # wide heads fill the registers
def test_steps_over_long_contexts_take_longer_blocks(lib, form, plan):  # noqa: F811
    """Twice the slots a block where four times leave a workgroup fewer than two blocks
    or cut unevenly, small blocks where both do."""
    lib.plan4_form.restype, lib.plan4_form.argtypes = ctypes.c_int, [ctypes.c_int] * 8
    lib.plan4_check.restype, lib.plan4_check.argtypes = ctypes.c_int, [ctypes.c_int] * 8
    assert lib.plan4_form(*plan) % 4 == form
    assert lib.plan4_check(*plan) == 0


def test_sixteen_heads_at_40000_take_blocks_between(lib):  # noqa: F811
    """32 segments of five blocks of 256 slots, not 27 of three of 512."""
    lib.plan4_form.restype, lib.plan4_form.argtypes = ctypes.c_int, [ctypes.c_int] * 8
    got = lib.plan4_form(128, 16, 40000, 0, 4, 39999, 0, 1)
    assert (got % 4, got // 4) == (3, 32)
