"""The host side of the entries of microscaled rows, of the choice of experts and
of the experts' blocks, on the CPU: what they refuse, their limits, and that
what they launch stays inside its buffers.

The backend's own host code runs against a stand-in HIP runtime that records
every allocation and checks every launch's grid, block and buffers
(tests/hostmx); no kernel runs.
"""
import ctypes
import fcntl
import os
import shutil
import subprocess

import numpy as np
import pytest

from igllm_amd import native

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
OKAY, ARG, SUPPORT = native.IGL_OKAY, native.IGL_FAIL_ARGUMENT, native.IGL_FAIL_SUPPORT
F32, BF16, F16 = native.IGL_STORE_F32, native.IGL_STORE_BF16, native.IGL_STORE_F16
AT = 1 << 40  # an address nothing on the host follows


def load(path):
    lib = ctypes.CDLL(path)
    for name, (res, args) in native.SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    lib.audit_report.restype = ctypes.c_long
    lib.audit_report.argtypes = [ctypes.POINTER(ctypes.c_long)] * 2
    for name, count in (("form", 4), ("slices", 5), ("steps", 1), ("room", 6), ("pieces", 2), ("banks", 2), ("lanes", 1)):
        fn = getattr(lib, "planmx_" + name)
        fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_int] * count
    lib.planmx_tiles.restype, lib.planmx_tiles.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_int]
    lib.igl_mx4_work_bytes.restype, lib.igl_mx4_work_bytes.argtypes = ctypes.c_size_t, [ctypes.c_int] * 4
    return lib


@pytest.fixture(scope="module")
def so():
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc or make absent")
    where = os.path.join(HERE, "hostmx")
    with open(os.path.join(where, "Makefile")) as lock:  # test processes side by side build once
        fcntl.flock(lock, fcntl.LOCK_EX)
        r = subprocess.run(["make", "-s", "-j8", "-C", where], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    return os.path.join(where, "_build", "libhostmx.so")


@pytest.fixture(scope="module")
def lib(so):
    return load(so)


class Host:
    """A desk on the stand-in runtime."""

    def __init__(self, lib):
        self.lib, self.desk = lib, native.Desk()
        assert lib.igl_back_open(ctypes.byref(self.desk), 0, 64, 2048, 16) == OKAY

    def call(self, name, *args):
        args = [ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args]
        code = getattr(self.lib, name)(ctypes.byref(self.desk), *args)
        assert self.lib.igl_desk_error_take(ctypes.byref(self.desk)) == code
        return code

    def alloc(self, nbytes):
        return self.lib.igl_dev_alloc(ctypes.byref(self.desk), nbytes)

    def mx4(self, rows, cols, pad=0):
        code, scale = self.alloc(rows * (cols // 2 + 16 * pad)), self.alloc(rows * (cols // 32 + pad))
        return native.Mx4(rows, cols, code, cols // 2 + 16 * pad, scale, cols // 32 + pad)

    def launches(self):
        n, k = ctypes.c_long(), ctypes.c_long()
        bad = self.lib.audit_report(ctypes.byref(n), ctypes.byref(k))
        return n.value, bad


@pytest.fixture(scope="module")
def host(lib):
    return Host(lib)


@pytest.fixture()
def loose(so, tmp_path):
    """A desk of its own, for calls whose pointers are no memory."""
    return Host(load(str(shutil.copy(so, tmp_path / "lib.so"))))


# ---- the structs -----------------------------------------------------------------

def test_mirrors_match_the_header(tmp_path):
    mirrors = [("igl_mx4", native.Mx4), ("igl_route", native.Route), ("igl_experts", native.Experts)]
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "igl_backend.h"', "int main(void) {"]
    for c, mirror in mirrors:
        lines.append(f'  printf("%zu\\n", sizeof({c}));')
        lines += [f'  printf("%zu\\n", offsetof({c}, {f[0]}));' for f in mirror._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, mirror in mirrors:
        want += [ctypes.sizeof(mirror)] + [getattr(mirror, f[0]).offset for f in mirror._fields_]
    assert got == want


# ---- what is refused -------------------------------------------------------------

def changed(s, field, value):
    t = type(s)()
    ctypes.memmove(ctypes.byref(t), ctypes.byref(s), ctypes.sizeof(s))
    setattr(t, field, value)
    return t


@pytest.mark.parametrize("field,value", [
    ("row_count", 0), ("row_count", -1), ("col_count", 0), ("col_count", 48), ("col_count", -32), ("code", None),
    ("scale", None), ("code_stride", 47), ("code_stride", 24), ("code_stride", 40), ("scale_stride", 2), ("code", 8)])
def test_bad_rows_are_refused(host, field, value):
    s = host.mx4(20, 96)
    x, out = host.alloc(20 * 96 * 4), host.alloc(20 * 20 * 4)
    bad = changed(s, field, s.code + value if field == "code" and value else value)
    before = host.launches()
    assert host.call("igl_mx4_lay_dev", bad, 0, 1, x, F32, 96) == ARG
    assert host.call("igl_mx4_read_dev", bad, 0, 1, x, F32, 96) == ARG
    assert host.call("igl_mx4_mat_mat_dev", bad, x, F32, 96, 2, out, F32, 20) == ARG
    assert host.call("igl_mx4_mat_mx4_dev", bad, s, 0, 2, out, F32, 20) == ARG
    assert host.call("igl_mx4_mat_mx4_dev", s, bad, 0, 1, out, F32, 20) == ARG
    x4 = native.Experts(1, 96, 96, 0, host.mx4(192, 96), s)
    assert host.call("igl_experts_dev", changed(x4, "down", bad), x, F32, 96, 1, x, x, 1, out, F32, 96) == ARG
    assert host.call("igl_experts_dev", changed(x4, "gate_up", bad), x, F32, 96, 1, x, x, 1, out, F32, 96) == ARG
    assert host.launches() == before


def test_bad_calls_on_rows_are_refused(host):
    s = host.mx4(20, 96)
    x, out = host.alloc(20 * 96 * 4), host.alloc(20 * 20 * 4)
    before = host.launches()
    for name in ("igl_mx4_lay_dev", "igl_mx4_read_dev"):
        for first, count, at, kind, stride, code in (
                (0, 0, x, F32, 96, ARG), (0, 21, x, F32, 96, ARG), (-1, 2, x, F32, 96, ARG), (19, 2, x, F32, 96, ARG),
                (2 ** 31 - 1, 2, x, F32, 96, ARG), (0, 2, None, F32, 96, ARG), (0, 2, x, F32, 95, ARG),
                (0, 2, x, F32, -96, ARG), (0, 2, x + 2, F32, 96, ARG), (0, 2, x + 1, BF16, 96, ARG), (0, 2, x, F16, 96, SUPPORT),
                (0, 2, x, -1, 96, SUPPORT), (0, 2, x, 99, 96, SUPPORT)):
            assert host.call(name, s, first, count, at, kind, stride) == code, (first, count, kind, stride)
        assert host.call(name, None, 0, 1, x, F32, 96) == ARG
    for at, kind, stride, lanes, to, out_kind, out_stride, code in (
            (None, F32, 96, 2, out, F32, 20, ARG), (x, F32, 96, 2, None, F32, 20, ARG), (x, F32, 96, 0, out, F32, 20, ARG),
            (x, F32, 96, -3, out, F32, 20, ARG), (x, F32, 95, 2, out, F32, 20, ARG), (x, F32, 96, 2, out, F32, 19, ARG),
            (x + 2, F32, 96, 2, out, F32, 20, ARG), (x, F32, 96, 2, out + 1, BF16, 20, ARG), (x, F16, 96, 2, out, F32, 20, SUPPORT),
            (x, F32, 96, 2, out, F16, 20, SUPPORT), (x, F32, 96, 65535 * 16 + 1, out, F32, 20, SUPPORT)):
        assert host.call("igl_mx4_mat_mat_dev", s, at, kind, stride, lanes, to, out_kind, out_stride) == code
    assert host.call("igl_mx4_mat_mat_dev", None, x, F32, 96, 2, out, F32, 20) == ARG
    other = host.mx4(20, 64)
    for act, first, lanes, to, out_kind, out_stride, code in (
            (s, 0, 0, out, F32, 20, ARG), (s, 0, 21, out, F32, 20, ARG), (s, -1, 2, out, F32, 20, ARG), (s, 19, 2, out, F32, 20, ARG),
            (other, 0, 2, out, F32, 20, ARG), (None, 0, 2, out, F32, 20, ARG), (s, 0, 2, None, F32, 20, ARG),
            (s, 0, 2, out, F16, 20, SUPPORT), (s, 0, 2, out, F32, 19, ARG), (s, 0, 2, out + 2, F32, 20, ARG)):
        assert host.call("igl_mx4_mat_mx4_dev", s, act, first, lanes, to, out_kind, out_stride) == code
    assert host.launches() == before
    assert host.lib.igl_mx4_lay_dev(None, ctypes.byref(s), 0, 1, x, F32, 96) == native.IGL_FAIL_STATE


ROUTE = dict(expert_count=16, top=2, score=0, group_count=4, group_top=2, group_best=2, renorm=1, gain_scale=1.0)


@pytest.mark.parametrize("field,value,code", [
    ("expert_count", 0, ARG), ("expert_count", -4, ARG), ("expert_count", 1028, SUPPORT), ("top", 0, ARG), ("top", 17, ARG),
    ("score", 2, ARG), ("score", -1, ARG), ("group_count", 0, ARG), ("group_count", 3, ARG), ("group_count", -1, ARG),
    ("group_top", 0, ARG), ("group_top", 5, ARG), ("group_best", 0, ARG), ("group_best", 3, ARG),
    ("gain_scale", float("nan"), ARG), ("gain_scale", float("inf"), ARG)])
def test_bad_rules_are_refused(host, field, value, code):
    b = host.alloc(1 << 20)
    before = host.launches()
    assert host.call("igl_route_dev", native.Route(**dict(ROUTE, **{field: value})), b, 2000, 3, None, None, b, b) == code
    assert host.launches() == before


def test_bad_routes_are_refused(host):
    b, rule = host.alloc(1 << 20), native.Route(**ROUTE)
    before = host.launches()
    for args, code in (((None, 16, 3, None, None, b, b), ARG), ((b, 15, 3, None, None, b, b), ARG), ((b, 16, 0, None, None, b, b), ARG),
                       ((b, 16, 3, None, None, None, b), ARG), ((b, 16, 3, None, None, b, None), ARG),
                       ((b + 2, 16, 3, None, None, b, b), ARG), ((b, 16, 3, b + 1, None, b, b), ARG),
                       ((b, 16, 3, None, b + 3, b, b), ARG), ((b, 16, 3, None, None, b + 2, b), ARG),
                       ((b, 16, 3, None, None, b, b + 2), ARG), ((b, 16, 2 ** 26, None, None, b, b), SUPPORT)):
        assert host.call("igl_route_dev", rule, *args) == code, args
    assert host.call("igl_route_dev", None, b, 16, 3, None, None, b, b) == ARG
    assert host.call("igl_route_dev", native.Route(**dict(ROUTE, expert_count=130, top=65, group_count=1, group_top=1)), b, 130, 3,
                     None, None, b, b) == SUPPORT
    assert host.call("igl_route_dev", native.Route(**dict(ROUTE, expert_count=130, group_count=65)), b, 130, 3, None, None, b,
                     b) == SUPPORT
    assert host.launches() == before


def test_bad_experts_are_refused(host):
    E, hidden, inner = 3, 64, 96
    x = native.Experts(E, hidden, inner, 0, host.mx4(E * 2 * inner, hidden), host.mx4(E * hidden, inner))
    act, pick = host.alloc(4 * 64 * 10), host.alloc(4 * 10)
    good = (act, F32, 64, 2, pick, pick, 2, act, F32, 64)
    before = host.launches()
    for field, value in (("expert_count", 0), ("expert_count", 2), ("hidden", 32), ("hidden", 0), ("inner", 64), ("gate", 2),
                         ("gate", -1), ("expert_count", -3)):
        assert host.call("igl_experts_dev", changed(x, field, value), *good) == ARG, field
    for at, value, code in ((0, None, ARG), (0, act + 2, ARG), (1, F16, SUPPORT), (2, 63, ARG), (3, 0, ARG), (3, -1, ARG),
                            (4, None, ARG), (4, pick + 1, ARG), (5, None, ARG), (5, pick + 2, ARG), (6, 0, ARG), (6, -2, ARG),
                            (6, 65, SUPPORT), (7, None, ARG), (8, F16, SUPPORT), (9, 63, ARG), (3, 2 ** 31 - 1, SUPPORT),
                            (3, 524289, SUPPORT)):
        args = list(good)
        args[at] = value
        assert host.call("igl_experts_dev", x, *args) == code, (at, value)
    assert host.call("igl_experts_dev", None, *good) == ARG
    assert host.launches() == before
    many = native.Experts(1025, 32, 32, 0, host.mx4(1025 * 64, 32), host.mx4(1025 * 32, 32))
    assert host.call("igl_experts_dev", many, act, F32, 32, 1, pick, pick, 1, act, F32, 32) == SUPPORT


def test_calls_past_a_launch_are_refused_before(loose):
    """A grid has fewer than 2^32 threads a side, and 65535 workgroups of the second."""
    def rows(count, cols, stride=None):
        return native.Mx4(count, cols, AT, stride or cols // 2, AT, cols // 32)

    def both(name, good, bad):
        for args, code in ((good, OKAY), (bad, SUPPORT)):
            before = loose.launches()[0]
            assert loose.call(name, *args) == code, (name, args)
            assert (loose.launches()[0] > before) == (code == OKAY)

    most = ((1 << 24) - 1) * 256 // 4
    for name in ("igl_mx4_lay_dev", "igl_mx4_read_dev"):
        both(name, (rows(2 ** 31 - 1, 32), 0, most, AT, F32, 32), (rows(2 ** 31 - 1, 32), 0, most + 1, AT, F32, 32))
    both("igl_mx4_mat_mat_dev", (rows(1 << 27, 32), AT, F32, 32, 1, AT, F32, 1 << 27),
         (rows((1 << 27) + 1, 32), AT, F32, 32, 1, AT, F32, (1 << 27) + 1))
    both("igl_mx4_mat_mat_dev", (rows(9, 32, 1 << 24), AT, F32, 32, 1, AT, F32, 9), (rows(9, 32, (1 << 24) + 16), AT, F32, 32, 1, AT, F32, 9))
    both("igl_mx4_mat_mat_dev", (rows(16, 32), AT, BF16, 32, 65535 * 16, AT, F32, 16), (rows(16, 32), AT, BF16, 32, 65535 * 16 + 1, AT, F32, 16))
    both("igl_mx4_mat_mx4_dev", (rows(16, 32), rows(1 << 21, 32), 5, 65535 * 16, AT, F32, 16),
         (rows(16, 32), rows(1 << 21, 32), 5, 65535 * 16 + 1, AT, F32, 16))
    both("igl_mx4_mat_mx4_dev", (rows(16, 32), rows(9, 32, 1 << 24), 0, 9, AT, F32, 16), (rows(16, 32), rows(9, 32, (1 << 24) + 16), 0, 9, AT, F32, 16))
    both("igl_route_dev", (native.Route(**ROUTE), AT, 16, (1 << 26) - 64, None, None, AT, AT),
         (native.Route(**ROUTE), AT, 16, (1 << 26) - 63, None, None, AT, AT))

    def experts(count, hidden, inner):
        return native.Experts(count, hidden, inner, 1, rows(count * 2 * inner, hidden), rows(count * hidden, inner))

    both("igl_experts_dev", (experts(1024, 32, 32), AT, F32, 32, 64511 * 16, AT, AT, 1, AT, F32, 32),
         (experts(1024, 32, 32), AT, F32, 32, 64512 * 16, AT, AT, 1, AT, F32, 32))
    for wide, width in ((experts(1, 32, 32768), 32), (experts(1, 32768, 32), 32768)):
        both("igl_experts_dev", (wide, AT, BF16, width, 131071, AT, AT, 1, AT, F32, width),
             (wide, AT, BF16, width, 131072, AT, AT, 1, AT, F32, width))


# ---- what is launched --------------------------------------------------------------

def free(host, *buffers):
    for b in buffers:
        host.lib.igl_dev_free(ctypes.byref(host.desk), b)


def test_products_stay_inside_their_buffers(lib, host):
    """Every form, at its own workspace: a small desk first, so that each call grows it or fits."""
    rng = np.random.default_rng(1)
    forms, sliced = set(), 0
    cases = [(6144, 1536, 1), (262144, 1536, 5), (70000, 800, 16), (2048, 8192, 37), (8192, 2048, 2047), (1, 32, 1),
             (16, 32, 20000), (7690, 160, 1540), (6200, 96, 1000), (6150, 64, 500), (300, 8192, 16), (300, 8192, 17)]
    cases += [(int(2 ** rng.uniform(0, 14)), 32 * int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 12))) for _ in range(60)]
    for rows, cols, lanes in cases:
        pad = int(rng.integers(0, 3))
        s, a = host.mx4(rows, cols, pad), host.mx4(lanes + 2, cols, pad)
        for kind, width in ((F32, 4), (BF16, 2)):
            act, out = host.alloc(width * lanes * (cols + pad)), host.alloc(width * lanes * (rows + pad))
            assert host.call("igl_mx4_mat_mat_dev", s, act, kind, cols + pad, lanes, out, kind, rows + pad) == OKAY
            assert host.call("igl_mx4_mat_mx4_dev", s, a, 2, lanes, out, kind, rows + pad) == OKAY
            assert host.call("igl_mx4_lay_dev", a, 2, lanes, act, kind, cols + pad) == OKAY
            assert host.call("igl_mx4_read_dev", a, 2, lanes, act, kind, cols + pad) == OKAY
            free(host, act, out)
        for terms in (0, 3, 5):
            forms.add((terms, lib.planmx_form(rows, cols, lanes, terms)))
            sliced += lib.planmx_form(rows, cols, lanes, terms) == 2 and lib.planmx_slices(rows, cols, lanes, 64 if terms == 0 else 32, 256) > 1
        assert host.launches()[1] == 0, (rows, cols, lanes)
        free(host, s.code, s.scale, a.code, a.scale)
    assert forms == {(0, 0), (0, 2), (0, 3), (3, 0), (3, 1), (3, 2), (3, 3), (3, 4), (3, 5), (5, 0), (5, 1),
                     (5, 2), (5, 3), (5, 5)}
    assert sliced > 5


def test_experts_stay_inside_their_buffers(lib, host):
    rng = np.random.default_rng(2)
    cases = [(1, 32, 32, 1, 1), (128, 1536, 768, 8, 1), (64, 1536, 704, 6, 37), (128, 1536, 768, 8, 700), (4, 64, 96, 2, 1000),
             (8, 96, 128, 8, 7), (16, 8192, 32, 2, 3), (16, 32, 8192, 2, 3), (1024, 32, 32, 64, 9)]
    for _ in range(40):
        E = int(2 ** rng.uniform(0, 7))
        cases.append((E, 32 * int(2 ** rng.uniform(0, 6)), 32 * int(2 ** rng.uniform(0, 5)), int(rng.integers(1, min(E, 8) + 1)),
                      int(2 ** rng.uniform(0, 9))))
    for E, hidden, inner, top, lanes in cases:
        gate_up, down = host.mx4(E * 2 * inner, hidden, 1), host.mx4(E * hidden, inner, 2)
        x = native.Experts(E, hidden, inner, 0, gate_up, down)
        pick, weight = host.alloc(4 * lanes * top), host.alloc(4 * lanes * top)
        for kind, width in ((F32, 4), (BF16, 2)):
            act, out = host.alloc(width * lanes * (hidden + 3)), host.alloc(width * lanes * (hidden + 1))
            assert host.call("igl_experts_dev", x, act, kind, hidden + 3, lanes, pick, weight, top, out, kind, hidden + 1) == OKAY
            free(host, act, out)
        for bf16 in (0, 1):
            assert lib.planmx_room(E, hidden, inner, lanes, top, bf16) == 0
        assert host.launches()[1] == 0, (E, hidden, inner, top, lanes)
        free(host, pick, weight, gate_up.code, gate_up.scale, down.code, down.scale)


def test_routes_stay_inside_their_buffers(host):
    for E, top, groups, lanes, biased in ((1, 1, 1, 1, 0), (128, 8, 1, 5, 0), (256, 8, 8, 2048, 1), (1024, 64, 64, 300, 1),
                                          (60, 16, 4, 5000, 0), (63, 16, 1, 5000, 1), (4, 4, 1, 2049, 0), (1000, 9, 1, 2048, 0)):
        x, pick, weight, b = (host.alloc(4 * n) for n in (lanes * (E + 1), lanes * top, lanes * top, E))
        rule = native.Route(E, top, 1, groups, groups, 1, 1, 1.0)
        assert host.call("igl_route_dev", rule, x, E + 1, lanes, b if biased else None, b, pick, weight) == OKAY
        assert host.launches()[1] == 0
        free(host, x, pick, weight, b)


def test_a_second_desk_has_its_own_room(lib):
    """And a call that finds no room leaves an error, not a launch."""
    a, b = Host(lib), Host(lib)
    s = a.mx4(4096, 2048)
    act, out = a.alloc(4 * 300 * 2048), a.alloc(4 * 300 * 4096)
    for h in (a, b):
        assert h.call("igl_mx4_mat_mat_dev", s, act, F32, 2048, 300, out, F32, 4096) == OKAY
    assert a.launches()[1] == 0


# ---- plans ---------------------------------------------------------------------------

def test_slices_cover_the_columns(lib):
    rng = np.random.default_rng(3)
    for _ in range(2000):
        rows, cols, lanes = (int(2 ** rng.uniform(0, 15)), 32 * int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 12)))
        for tile in (32, 64):
            steps, n = lib.planmx_steps(cols), lib.planmx_slices(rows, cols, lanes, tile, 256)
            each = -(-steps // n)
            assert 1 <= n <= steps and (n - 1) * each < steps <= n * each  # none empty, none left out


def test_pieces_of_terms(lib):
    for terms in (3, 5):
        for lanes in (1, 2, 3, 7, 16, 37, 2047):
            assert lib.planmx_pieces(terms, lanes) == 0


def test_rows_in_lds_meet_no_bank_twice(lib):
    for width in (64, 128):
        assert lib.planmx_banks(width, 1) == 0 and lib.planmx_banks(width, 0) != 0


def test_a_slots_lane(lib):
    assert all(lib.planmx_lanes(top) == 0 for top in range(1, 65))


def test_tiles_of_experts_places(lib):
    """Tiles of an expert begin behind the last's, whatever the counts, and fill the launch."""
    rng = np.random.default_rng(4)
    for _ in range(500):
        E = int(2 ** rng.uniform(0, 8))
        count = np.ascontiguousarray(rng.integers(0, 2 ** rng.integers(1, 9), size=E) * (rng.random(E) < rng.random()), np.int32)
        for tile in (16, 32, 64):
            assert lib.planmx_tiles(count.ctypes.data, E, tile) == 0
    planted = np.array([5, 70, 0, 3], np.int32)
    assert lib.planmx_tiles(planted.ctypes.data, 4, 0x7FFFFFFF) == 0  # one tile an expert
