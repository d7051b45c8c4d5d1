"""The linear forward and input gradient on both sides of the rules that choose their kernels (tests/test_row_dispatch.py says which is which), against 64-bit products."""
import pytest
import torch

from tests.test_gpu_row_ops import U, dtype, half_step, randn, test_linear_forward_many_rows as forward, tiny  # noqa: F401  (dtype is a fixture)

pytestmark = pytest.mark.gpu

# K at 191 / 193 and out at 120 / 130 (ragged rows with a residual), out at 190 / 192 (without), two k-steps of ragged rows; whole chunks at out 192 / 256
BORDERS = [(87600, 191, 192), (87600, 193, 192), (131200, 201, 120), (131200, 201, 130), (87600, 201, 190), (87600, 201, 192), (87600, 256, 192), (65600, 256, 256), (87600, 250, 250), (66001, 33, 520)]


@pytest.mark.parametrize("m,k,n", BORDERS)
@pytest.mark.parametrize("act,bias,residual,pre", [("none", False, False, False), ("relu", True, True, False), ("gelu", True, True, True), ("silu", False, False, True)])
def test_forward_at_the_borders(dtype, m, k, n, act, bias, residual, pre):
    forward(dtype, m, k, n, act, bias, residual, pre)


@pytest.mark.parametrize("m,n,k", BORDERS)  # (the product's K is out, its columns are in)
def test_input_gradient_at_the_borders(dtype, m, n, k):
    from simhand_amd import ops

    if dtype == torch.float32:
        m = m // 16 + 5
    w, dz = randn(n, k, seed=1, dtype=dtype).cuda(), randn(m, n, seed=2, dtype=dtype).cuda()
    dx = ops.linear_bwd(dz, None, w, need_dw=False)[0]
    zd, wd = dz.double(), w.double()
    want = zd @ wd
    assert bool(((dx.double() - want).abs() <= half_step(dtype) * want.abs() + 1.01 * 2 * (n + 2) * U * (zd.abs() @ wd.abs()) + tiny(dtype)).all())
