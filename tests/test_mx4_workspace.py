"""The workspaces of microscaled products and of experts' blocks, on the CPU (test_mx4_host's stand-in runtime): a call
asks for what its form uses, so that one which uses none is not refused for it while a replay lives."""
import ctypes

import pytest

from igllm_amd import native
from test_mx4_host import BF16, F32, OKAY, Host, lib, load, so  # noqa: F401


def frozen(lib):  # noqa: F811
    """A desk whose workspaces are as they were at its opening, and stay."""
    h = Host(lib)
    x = h.alloc(4096)
    rule = native.Route(16, 2, 0, 1, 1, 1, 1, 1.0)
    assert lib.igl_record_begin(ctypes.byref(h.desk)) == OKAY
    assert h.call("igl_route_dev", rule, x, 16, 1, None, None, x, x) == OKAY
    replay = ctypes.c_void_p()
    assert lib.igl_record_end(ctypes.byref(h.desk), ctypes.byref(replay)) == OKAY
    return h, replay


@pytest.mark.parametrize("rows,cols,lanes", [(6144, 8192, 1), (6144, 1536, 1), (6144, 1536, 3), (262144, 1536, 1), (40, 96, 2)])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_a_token_needs_no_room(lib, rows, cols, lanes, kind):  # noqa: F811
    assert lib.igl_mx4_work_bytes(rows, cols, lanes, 5 if kind == F32 else 3) == 0
    h, replay = frozen(lib)
    s, act, out = h.mx4(rows, cols), h.alloc(4 * cols * lanes), h.alloc(4 * rows * lanes)
    before = h.launches()[0]
    assert h.call("igl_mx4_mat_mat_dev", s, act, kind, cols, lanes, out, F32, rows) == OKAY
    assert h.launches() == (before + 1, 0)
    lib.igl_replay_free(ctypes.byref(h.desk), replay)


@pytest.mark.parametrize("E,hidden,inner,top,lanes", [(128, 1536, 768, 8, 1), (128, 1536, 768, 8, 4), (8, 64, 96, 2, 3), (1, 32, 32, 1, 1)])
def test_a_tokens_experts_need_their_hidden_values(lib, E, hidden, inner, top, lanes):  # noqa: F811
    lib.igl_experts_work_bytes.restype = ctypes.c_size_t
    lib.igl_experts_work_bytes.argtypes = [ctypes.POINTER(native.Experts)] + [ctypes.c_int] * 3
    x = native.Experts(E, hidden, inner)
    for bf16 in (0, 1):
        assert lib.igl_experts_work_bytes(ctypes.byref(x), lanes, top, bf16) == -(-lanes * top * inner * 4 // 256) * 256


def test_what_does_need_room_is_refused(lib):  # noqa: F811
    h, replay = frozen(lib)
    s, act, out = h.mx4(6144, 1536), h.alloc(4 * 1536 * 40), h.alloc(4 * 6144 * 40)
    before = h.launches()
    assert h.call("igl_mx4_mat_mat_dev", s, act, F32, 1536, 40, out, F32, 6144) == native.IGL_FAIL_STATE
    assert h.launches() == before
    lib.igl_replay_free(ctypes.byref(h.desk), replay)
    assert h.call("igl_mx4_mat_mat_dev", s, act, F32, 1536, 40, out, F32, 6144) == OKAY
