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
