"""CPU: what the row operators' C entry points refuse (before anything reaches a GPU) and what the Python layer refuses without one."""
import ctypes as C

import pytest
import torch

from simhand_amd import _lib, ops

P = C.c_void_p(16)  # a pointer that nothing may follow: every call below has to be refused first


def refused(rc):
    return rc != 0 and _lib.load().simhand_last_error()


def test_c_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    N = None
    assert refused(lib.simhand_layer_norm_fwd(P, P, P, 1e-5, 0, P, P, P, 4, 8, 7, N))              # dtype
    assert refused(lib.simhand_layer_norm_fwd(P, P, P, 1e-5, 0, P, P, P, -1, 8, 0, N))             # rows
    assert refused(lib.simhand_layer_norm_fwd(P, P, P, 1e-5, 0, P, P, P, 4, 0, 0, N))              # cols
    assert refused(lib.simhand_layer_norm_fwd(P, P, P, 1e-5, 0, P, P, P, 4, 8193, 0, N))           # too wide, fp32
    assert refused(lib.simhand_layer_norm_fwd(P, P, P, 1e-5, 0, P, P, P, 4, 16385, 1, N))          # too wide, 16 bits
    assert refused(lib.simhand_layer_norm_fwd(P, P, P, -1.0, 0, P, P, P, 4, 8, 0, N))              # eps
    assert refused(lib.simhand_layer_norm_fwd(N, P, P, 1e-5, 0, P, P, P, 4, 8, 0, N))              # x
    assert refused(lib.simhand_layer_norm_bwd(P, P, N, N, P, P, P, P, 0, P, P, 4000, 8, 0, P, 4, N))  # workspace
    assert refused(lib.simhand_layer_norm_bwd(P, P, P, P, P, P, P, P, 0, P, P, 4, 8, 0, P, 1 << 20, N))  # x and codes
    assert refused(lib.simhand_layer_norm_bwd(P, N, P, N, P, P, P, P, 0, P, P, 4, 8, 0, P, 1 << 20, N))  # codes without exponents
    assert refused(lib.simhand_linear_fwd(P, P, N, 4, N, P, N, 4, 8, 8, 0, P, 1 << 30, N))                     # act
    assert refused(lib.simhand_linear_fwd(P, P, N, 0, N, P, N, 4, 0, 8, 0, P, 1 << 30, N))                     # in_dim
    assert refused(lib.simhand_linear_fwd(P, P, N, 0, N, P, N, 4, 8, 0, 0, P, 1 << 30, N))                     # out_dim
    assert refused(lib.simhand_linear_fwd(P, P, N, 0, N, P, N, 1 << 31, 8, 8, 0, P, 1 << 30, N))               # rows
    assert refused(lib.simhand_linear_fwd(P, P, N, 0, N, N, N, 4, 8, 8, 0, P, 1 << 30, N))                     # y
    assert refused(lib.simhand_linear_fwd(P, P, N, 0, N, P, N, 200000, 77, 130, 1, N, 0, N))       # workspace
    assert refused(lib.simhand_linear_act_bwd(P, N, 2, P, P, 4, 8, 0, P, 1 << 20, N))              # gelu without pre
    assert refused(lib.simhand_linear_act_bwd(P, P, 2, P, P, 4000, 8, 0, N, 0, N))                 # workspace
    assert refused(lib.simhand_linear_dgrad(P, P, P, 4, 8, 8, 0, P, 8, N))                         # workspace
    assert refused(lib.simhand_linear_wgrad(P, P, N, N, N, 4, 8, 8, 0, P, 1 << 20, N))             # dw
    assert refused(lib.simhand_linear_wgrad(P, P, N, N, P, 4, 8, 8, 2, P, 1 << 20, N))             # dtype
    assert refused(lib.simhand_linear_wgrad(P, P, N, N, P, 100000, 512, 512, 1, N, 0, N))          # workspace
    assert refused(lib.simhand_act8_pack(P, P, N, 4, 8, 0, N))                                     # exps
    assert refused(lib.simhand_act8_pack(P, P, P, 4, 0, 0, N))                                     # cols
    assert refused(lib.simhand_act8_unpack(P, P, P, -4, 8, 0, N))                                  # rows


def test_no_rows_is_no_launch():
    lib = _lib.load()
    assert lib.simhand_layer_norm_fwd(None, P, P, 1e-5, 0, None, None, None, 0, 8, 0, None) == 0
    assert lib.simhand_linear_fwd(None, P, None, 0, None, None, None, 0, 8, 8, 1, None, 0, None) == 0
    assert lib.simhand_act8_pack(None, None, None, 0, 8, 0, None) == 0
    assert lib.simhand_act8_unpack(None, None, None, 0, 8, 1, None) == 0


def test_workspace_queries():
    lib = _lib.load()
    assert lib.simhand_layer_norm_bwd_workspace_bytes(0, 8, 0) == 0  # one block: its sums are the result
    assert lib.simhand_layer_norm_bwd_workspace_bytes(4000, 8, 0) > 0
    assert lib.simhand_layer_norm_bwd_workspace_bytes(-1, 8, 0) == 0
    assert lib.simhand_linear_dgrad_workspace_bytes(4, 8, 0, 0, 0) == 0
    for rows in (0, 1, 1000, 401408, (1 << 31) - 1):
        for cols in (1, 77, 2048):
            assert 0 <= lib.simhand_linear_act_bwd_workspace_bytes(rows, cols, 1) < 1 << 28
            assert 0 <= lib.simhand_linear_wgrad_workspace_bytes(rows, cols, 512, 1) < 1 << 30


def test_python_layer_refuses_host_tensors():
    x, w, g = torch.zeros(4, 8), torch.zeros(6, 8), torch.ones(8)
    E = _lib.SimhandHipError
    for f in (lambda: ops.layer_norm_fwd(x, g, g), lambda: ops.layer_norm_bwd(x, x, g, g, g[:4], g[:4]), lambda: ops.linear_fwd(x, w),
              lambda: ops.linear_act_bwd(x), lambda: ops.linear_bwd(torch.zeros(4, 6), x, w), lambda: ops.act8_pack(x),
              lambda: ops.act8_unpack(ops.Act8(torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), torch.float32))):
        with pytest.raises(E):
            f()


def test_act8_checks_its_parts():
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    E = _lib.SimhandHipError
    ops.Act8(u8(4, 33), u8(4, 2), torch.bfloat16)
    ops.Act8(u8(2, 3, 64), u8(6, 2), torch.bfloat16)
    for codes, exps in ((u8(4, 33), u8(4, 1)), (u8(4, 33).int(), u8(4, 2)), (u8(4, 33), torch.zeros(4, 2)), (u8(4, 0), u8(0))):
        with pytest.raises(E):
            ops.Act8(codes, exps, torch.bfloat16)
