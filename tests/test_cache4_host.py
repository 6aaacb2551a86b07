"""The host side of the 4-bit ring's entries, on the CPU: what they refuse, and
that what they launch stays inside its buffers.

The backend's own host code runs against a stand-in HIP runtime that records
every allocation and checks every launch's grid, block and buffers
(tests/host4); no kernel runs.
"""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import cache4_oracle as c4
from igllm_amd import native

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib():
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc or make absent")
    where = os.path.join(HERE, "host4")
    r = subprocess.run(["make", "-s", "-j8", "-C", where], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    lib = ctypes.CDLL(os.path.join(where, "_build", "libhost4.so"))
    for name, (res, args) in native.SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    lib.audit_report.restype = ctypes.c_long
    lib.audit_report.argtypes = [ctypes.POINTER(ctypes.c_long)] * 2
    return lib


class Host:
    """A desk on the stand-in runtime."""

    def __init__(self, lib):
        self.lib, self.desk = lib, native.Desk()
        assert lib.igl_back_open(ctypes.byref(self.desk), 0, 64, 2048, 16) == native.IGL_OKAY

    def alloc(self, nbytes):
        return self.lib.igl_dev_alloc(ctypes.byref(self.desk), nbytes)

    def ring(self, fmt=0, span=100, sinks=0, kv=1, head=256, key_scale=0.01, value_scale=0.01):
        c = native.Cache4(fmt, span, sinks, kv, head, key_scale, value_scale)
        codes, gains = (f(ctypes.byref(c)) for f in (self.lib.igl_cache4_code_bytes, self.lib.igl_cache4_gain_bytes))
        c.key_code, c.key_gain, c.value_code, c.value_gain = (self.alloc(n) for n in (codes, gains, codes, gains))
        return c

    def lay(self, c, key, value, stride, place, lanes):
        return self.lib.igl_cache4_lay_dev(ctypes.byref(self.desk), ctypes.byref(c) if c else None, key, value, stride,
                                           place, lanes)

    def read(self, c, place, lanes, key, value, stride):
        return self.lib.igl_cache4_read_dev(ctypes.byref(self.desk), ctypes.byref(c) if c else None, place, lanes, key,
                                            value, stride)

    def attend(self, c, share, query, stride, place, window, lanes, out, score=1.0):
        return self.lib.igl_attend4_lanes_dev(ctypes.byref(self.desk), ctypes.byref(c) if c else None, share, query,
                                              stride, place, window, lanes, score, out)

    def take(self):
        return self.lib.igl_desk_error_take(ctypes.byref(self.desk))

    def launches(self):
        n, k = ctypes.c_long(), ctypes.c_long()
        bad = self.lib.audit_report(ctypes.byref(n), ctypes.byref(k))
        return n.value, bad


@pytest.fixture(scope="module")
def host(lib):
    return Host(lib)


def test_bytes(lib):
    """Sizes of a side, and none for dimensions no ring has."""
    def sizes(*dims):
        c = native.Cache4(*dims, 1.0, 1.0)
        return lib.igl_cache4_code_bytes(ctypes.byref(c)), lib.igl_cache4_gain_bytes(ctypes.byref(c))

    assert sizes(0, 100, 4, 2, 256) == (100 * 256, 128 * 16)
    assert sizes(1, 1, 0, 1, 64) == (32, 128)
    assert sizes(0, 1 << 24, 0, 8, 512) == ((1 << 24) * 2048, (1 << 24) * 128)  # past 32 bits
    for dims in [(2, 100, 0, 1, 256), (-1, 100, 0, 1, 256), (0, 0, 0, 1, 256), (0, 100, 100, 1, 256),
                 (0, 100, -1, 1, 256), (0, 100, 0, 0, 256), (0, 100, 0, 1, 96), (0, 100, 0, 1, 0),
                 (0, 2 ** 31 - 1, 0, 1, 64)]:
        assert sizes(*dims) == (0, 0), dims
    assert lib.igl_cache4_code_bytes(None) == 0 and lib.igl_cache4_gain_bytes(None) == 0


ARG, SUPPORT = native.IGL_FAIL_ARGUMENT, native.IGL_FAIL_SUPPORT


@pytest.mark.parametrize("field,value,code", [
    ("format", 2, ARG), ("format", -1, ARG), ("cache_span", 0, ARG), ("cache_span", -5, ARG), ("sink_count", -1, ARG),
    ("sink_count", 100, ARG), ("kv_count", 0, ARG), ("kv_count", -1, ARG), ("head_size", 96, SUPPORT),
    ("head_size", 1024, SUPPORT), ("head_size", 0, ARG), ("key_scale", 0.0, ARG), ("value_scale", -1.0, ARG),
    ("key_scale", float("nan"), ARG), ("value_scale", float("inf"), ARG), ("key_code", None, ARG),
    ("key_gain", None, ARG), ("value_code", None, ARG), ("value_gain", None, ARG), ("key_code", 8, ARG),
    ("value_gain", 4, ARG)])
def test_every_entry_refuses_a_bad_ring(host, field, value, code):
    c = host.ring()
    if field.endswith(("_code", "_gain")) and value:
        value = getattr(c, field) + value  # off its alignment
    setattr(c, field, value)
    room = host.alloc(100 * 256 * 8 * 4)
    before = host.launches()
    for call in (lambda: host.lay(c, room, room, 256, 0, 1), lambda: host.read(c, 0, 1, room, room, 256),
                 lambda: host.attend(c, 8, room, 2048, 0, 0, 1, room)):
        assert call() == code
        assert host.take() == code  # kept until it is taken
    assert host.launches() == before


def test_bad_calls_are_refused(host):
    c = host.ring(span=100, sinks=4)
    room = host.alloc(200 * 256 * 8 * 4)
    far = 2 ** 31 - 1
    before = host.launches()
    bad = [
        lambda: host.lay(None, room, room, 256, 0, 1), lambda: host.lay(c, None, room, 256, 0, 1),
        lambda: host.lay(c, room, None, 256, 0, 1), lambda: host.lay(c, room, room, 256, 0, 0),
        lambda: host.lay(c, room, room, 256, 0, -1), lambda: host.lay(c, room, room, 256, -1, 1),
        lambda: host.lay(c, room, room, 255, 0, 2), lambda: host.lay(c, room, room, 256, far, 1),
        lambda: host.lay(c, room, room, 256, 0, 101),  # 4 + 97 positions, 4 + 96 slots
        lambda: host.lay(c, room, room, 256, 50, 97), lambda: host.lay(c, room, room, 256, 3, 98),
        lambda: host.read(None, 0, 1, room, room, 256), lambda: host.read(c, 0, 1, None, None, 256),
        lambda: host.read(c, 0, 0, room, room, 256), lambda: host.read(c, -1, 1, room, room, 256),
        lambda: host.read(c, 0, 2, room, room, 255), lambda: host.read(c, 10, 97, room, room, 256),
        lambda: host.attend(None, 8, room, 2048, 0, 0, 1, room), lambda: host.attend(c, 8, None, 2048, 0, 0, 1, room),
        lambda: host.attend(c, 8, room, 2048, 0, 0, 1, None), lambda: host.attend(c, 0, room, 2048, 0, 0, 1, room),
        lambda: host.attend(c, 8, room, 2048, 0, -1, 1, room), lambda: host.attend(c, 8, room, 2048, 0, 0, 0, room),
        lambda: host.attend(c, 8, room, 2047, 0, 0, 2, room), lambda: host.attend(c, 8, room, 2048, -1, 0, 1, room),
        lambda: host.attend(c, 8, room, 2048, far, 8, 1, room),
        lambda: host.attend(c, 8, room, 2048, 100, 0, 1, room),    # 97 positions in 96 slots
        lambda: host.attend(c, 8, room, 2048, 500, 97, 1, room),   # a window past the ring
        lambda: host.attend(c, 8, room, 2048, 500, 96, 2, room),   # its last lane's row lies on its first's oldest
    ]
    for call in bad:
        assert call() == ARG
        assert host.take() == ARG
    assert host.attend(c, 65, room, 65 * 256, 0, 0, 1, room) == SUPPORT and host.take() == SUPPORT
    assert host.attend(c, 64, room, 64 * 256, 0, 1, 1 << 22, room) == SUPPORT and host.take() == SUPPORT
    assert host.launches() == before
    assert host.lib.igl_cache4_lay_dev(None, ctypes.byref(c), room, room, 256, 0, 1) == native.IGL_FAIL_STATE
    assert host.lib.igl_cache4_read_dev(None, ctypes.byref(c), 0, 1, room, room, 256) == native.IGL_FAIL_STATE
    assert host.lib.igl_attend4_lanes_dev(None, ctypes.byref(c), 8, room, 2048, 0, 0, 1, 1.0, room) == native.IGL_FAIL_STATE


@pytest.mark.parametrize("place,lanes,window", [(0, 100, 0), (99, 1, 0), (3, 1, 1), (500, 1, 96), (500, 2, 95),
                                                (2 ** 31 - 2, 1, 96), (0, 1, 2 ** 31 - 1), (2, 50, 7)])
def test_what_just_fits_runs(host, place, lanes, window):
    c = host.ring(span=100, sinks=4)
    room = host.alloc(lanes * 2048 * 4)
    n, bad = host.launches()
    assert host.attend(c, 8, room, 2048, place, window, lanes, room) == native.IGL_OKAY
    n1, bad1 = host.launches()
    assert n1 > n and bad1 == bad


@pytest.mark.parametrize("head", [64, 128, 256, 512])
@pytest.mark.parametrize("kv,share", [(1, 8), (3, 5), (2, 16), (1, 64), (8, 1)])
def test_launches_stay_inside_their_buffers(host, head, kv, share):
    """Every launch's grid, block, rings, rows and workspace (exactly as large
    as the entry's arguments say), over lanes, places, windows and wraps."""
    for span, sinks, place, window, lanes in [(1, 0, 0, 0, 1), (1, 0, 9, 1, 1), (65, 0, 0, 0, 65), (516, 4, 700, 512, 1),
                                              (600, 17, 4000, 512, 64), (2100, 0, 0, 0, 2047), (300, 3, 0, 40, 250),
                                              (20000, 0, 19000, 0, 5), (70000, 1, 69999, 0, 1)]:
        c = host.ring(0, span, sinks, kv, head)
        width = kv * head
        rows, heads = host.alloc(lanes * width * 4), host.alloc(lanes * width * share * 4)
        assert host.lay(c, rows, rows, width, place, lanes) == native.IGL_OKAY
        assert host.read(c, place, lanes, rows, None, width) == native.IGL_OKAY
        assert host.attend(c, share, heads, width * share, place, window, lanes, heads) == native.IGL_OKAY
        for p in (rows, heads, c.key_code, c.key_gain, c.value_code, c.value_gain):
            host.lib.igl_dev_free(ctypes.byref(host.desk), p)
    assert host.launches()[1] == 0


PLANS = [  # head, kv, span, sinks, share, place, window, lanes
    (64, 1, 1, 0, 1, 0, 0, 1), (64, 1, 1, 0, 64, 9, 1, 1), (128, 2, 65, 0, 3, 0, 0, 65), (256, 1, 516, 4, 8, 700, 512, 1),
    (256, 1, 2600, 4, 8, 0, 512, 2047), (512, 1, 2047, 0, 4, 0, 0, 2047), (512, 1, 16384, 0, 8, 15000, 0, 160),
    (512, 1, 16384, 0, 8, 8000, 0, 300), (128, 8, 131072, 0, 4, 131071, 0, 1), (512, 4, 40000, 1, 8, 39990, 0, 10),
    (128, 16, 5000, 0, 8, 0, 0, 5000), (512, 16, 3000, 5, 8, 900, 700, 2000), (64, 8, 300, 299, 2, 0, 0, 300),
    (256, 1, 100000, 17, 1, 99000, 50000, 17), (128, 1, 700, 0, 64, 5000, 300, 400), (256, 2, 65, 64, 2, 900, 1, 1),
]


def random_plans(count=400):
    rng = np.random.default_rng(11)
    for _ in range(count):
        head, kv, share = int(rng.choice([64, 128, 256, 512])), int(rng.choice([1, 2, 3, 8])), int(rng.integers(1, 65))
        span = int(2 ** rng.uniform(0, 12.5))
        sinks = int(rng.integers(0, min(span, 1 + int(2 ** rng.uniform(0, 8)))))
        ring = span - sinks
        lanes = int(min(2 ** rng.uniform(0, 11), ring))
        if rng.random() < 0.5:  # everything there is
            place, window = int(rng.integers(0, span - lanes + 1)), 0
        else:
            window = int(rng.integers(1, ring - lanes + 2))
            place = int(2 ** rng.uniform(0, 24)) - 1
        yield head, kv, span, sinks, share, place, window, lanes


def test_every_plan_covers_what_its_rows_see(lib):
    """The attention's tiles, blocks, segments, masks and partials, by counting:
    each slot a lane sees lies in one block of one segment, no block is taken for
    wholly visible that is not, and the partials fit their room."""
    lib.plan4_check.restype, lib.plan4_check.argtypes = ctypes.c_int, [ctypes.c_int] * 8
    for plan in PLANS + list(random_plans()):
        assert lib.plan4_check(*plan) == 0, plan


@pytest.mark.parametrize("form,segments,plan", [
    (2, 9, (256, 1, 516, 4, 8, 5000, 512, 1)),      # eight rows
    (3, 27, (64, 16, 40000, 0, 1, 39999, 0, 1)),    # in deep blocks
    (2, 63, (64, 8, 40000, 0, 1, 39999, 0, 1)),     # of which each workgroup would have one
    (1, 84, (512, 1, 16384, 0, 8, 16000, 0, 5)),    # sixteen, one workgroup a CU
    (1, 79, (512, 1, 16384, 0, 8, 15000, 0, 12)),   # two
    (1, 1, (256, 1, 2600, 4, 8, 0, 512, 1000)),     # too few blocks for tiles
    (0, 1, (256, 1, 2600, 4, 8, 0, 512, 2047)),     # tiles of 64
    (0, 12, (512, 1, 16384, 0, 8, 15000, 0, 160)),  # one turn of the card
    (1, 1, (64, 1, 2047, 0, 8, 0, 0, 2047)),        # 64-dim heads have none
])
def test_forms(lib, form, segments, plan):
    got = lib.plan4_form(*plan)
    assert (got % 4, got // 4) == (form, segments)


def test_oracle_agrees_with_itself():
    """What is stored stands for the nearest value there is: every level of every
    gain is stored as itself, and no other code of the chosen gain is nearer."""
    rng = np.random.default_rng(5)
    for fmt in (c4.INT4, c4.E2M1):
        rows = (rng.normal(size=(40, 64)) * np.exp(rng.normal(size=(40, 1)) * 2)).astype(np.float32)
        codes, gains = c4.quantise(rows, fmt, 0.013)
        got = c4.values(codes, gains, fmt, 0.013)
        for code in range(16):
            if fmt == c4.INT4 and code == 0:
                continue
            other = c4.values(np.full_like(codes, code), gains, fmt, 0.013)
            assert np.all(np.abs(got - rows) <= np.abs(other - rows))
        again, g2 = c4.quantise(got.astype(np.float32), fmt, 0.013)
        full = np.abs(c4.LEVELS[fmt][codes]).reshape(40, 2, 32).max(-1) == c4.TOP[fmt]
        assert np.array_equal(g2[full], gains[full])


def test_mirror_matches_header(tmp_path):
    """native.Cache4 has igl_cache4's layout, field for field."""
    fields = [f for f, _ in native.Cache4._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "igl_backend.h"\nint main(void) {\n' + "".join(
        f'  printf("%zu\\n", offsetof(igl_cache4, {f}));\n' for f in fields) +
        '  printf("%zu\\n", sizeof(igl_cache4));\n  return 0;\n}\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I" + os.path.join(os.path.dirname(HERE), "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [getattr(native.Cache4, f).offset for f in fields] + [ctypes.sizeof(native.Cache4)]
