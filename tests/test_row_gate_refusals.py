"""CPU: a layer norm's kept ReLU gate without the ReLU is refused by the C entry points and by the Python layer."""
import ctypes as C

import pytest
import torch

from simhand_amd import _lib, ops

P = C.c_void_p(16)  # a pointer that nothing may follow: every call below has to be refused first


def test_a_gate_needs_the_relu():
    lib = _lib.load()
    assert lib.simhand_layer_norm_fwd_ex(P, P, P, 1e-5, 0, P, P, P, P, 4, 8, 0, None) != 0
    assert lib.simhand_layer_norm_bwd_ex(P, P, None, None, P, P, P, P, 0, P, P, P, 4, 8, 0, P, 1 << 20, None) != 0
    assert lib.simhand_layer_norm_fwd_ex(P, P, P, 1e-5, 1, P, P, P, P, 4, 8, 7, None) != 0   # dtype
    assert lib.simhand_layer_norm_bwd_ex(P, P, P, P, P, P, P, P, 1, P, P, P, 4, 8, 0, P, 1 << 20, None) != 0  # x and codes
    assert lib.simhand_layer_norm_fwd_ex(None, P, P, 1e-5, 1, None, None, None, None, 0, 8, 0, None) == 0  # no rows: no launch
    x, g = torch.zeros(4, 8), torch.ones(8)
    for f in (lambda: ops.layer_norm_fwd(x, g, g, relu=True, want_gate=True), lambda: ops.layer_norm_bwd(x, x, g, g, g[:4], g[:4], True, gate=torch.zeros(4, 2, dtype=torch.uint8))):
        with pytest.raises(_lib.SimhandHipError):
            f()


def test_limits_that_the_header_names():
    lib = _lib.load()
    big = 1 << 40
    for cin, cout in (((1 << 20) + 1, 8), (8, (1 << 20) + 1)):
        assert lib.simhand_linear_fwd(P, P, None, 0, None, P, None, 4, cin, cout, 0, P, big, None) != 0
        assert lib.simhand_linear_dgrad(P, P, P, 4, cin, cout, 0, P, big, None) != 0
        assert lib.simhand_linear_wgrad(P, P, None, None, P, 4, cin, cout, 0, P, big, None) != 0
    assert lib.simhand_linear_act_bwd(P, P, 2, P, P, 4, (1 << 20) + 1, 0, P, big, None) != 0
    for rows in (-1, 1 << 31):
        assert lib.simhand_linear_act_bwd(P, P, 2, P, P, rows, 8, 0, P, big, None) != 0
        assert lib.simhand_linear_wgrad(P, P, None, None, P, rows, 8, 8, 0, P, big, None) != 0
    assert lib.simhand_act8_pack(P, P, P, 4, (1 << 24) + 1, 0, None) != 0
    assert lib.simhand_act8_unpack(P, P, P, 4, (1 << 24) + 1, 0, None) != 0
    assert lib.simhand_layer_norm_bwd_ex(P, P, None, None, P, P, P, P, 1, P, P, P, 4, 8193, 0, P, big, None) != 0
