"""Infinities, NaN and far values in the activations' gradients."""
import math

import pytest
import torch

from tests.test_gpu_row_ops import dtype, slope_ref  # noqa: F401  (dtype is a fixture)

pytestmark = pytest.mark.gpu


def test_relu_gradient_is_a_gate(dtype):
    """What the ReLU closes is 0 even for an infinite or NaN incoming gradient, what it opens passes as it is; a NaN pre-activation shows in dz and in its column's sum alone."""
    from simhand_amd import ops

    inf, nan = math.inf, math.nan
    dy = torch.tensor([[inf, -inf, nan, 2.0, inf, nan, 3.0, 5.0, 7.0]] * 3).to(dtype)
    pre = torch.tensor([[-1.0, 0.0, -2.0, -0.0, 1.0, 4.0, 6.0, nan, 1e-7]] * 3).to(dtype)
    dz, db = (t.cpu().float() for t in ops.linear_act_bwd(dy.cuda(), pre.cuda(), "relu"))
    want = torch.tensor([0.0, 0.0, 0.0, 0.0, inf, nan, 3.0, nan, 7.0])
    assert torch.equal(torch.isnan(dz), torch.isnan(want).expand(3, 9)) and torch.equal(torch.nan_to_num(dz, nan=9.0), torch.nan_to_num(want, nan=9.0).expand(3, 9))
    assert torch.equal(torch.nan_to_num(db, nan=9.0), torch.nan_to_num(3 * want, nan=9.0))


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_nan_stays_and_far_values_are_flat(dtype, act):
    from simhand_amd import ops

    big = torch.finfo(dtype).max
    z = torch.tensor([[math.nan, big, -big, 60.0, -200.0]]).to(dtype)
    dz = ops.linear_act_bwd(torch.full_like(z, 2.0).cuda(), z.cuda(), act)[0].cpu().double()
    assert bool(torch.isnan(dz[0, 0])) and torch.equal(dz[0, 1:], torch.tensor([2.0, 0.0, 2.0, 0.0], dtype=torch.float64))
    w = torch.eye(5).to(dtype)
    y = ops.linear_fwd(torch.diag(z[0, 1:].float()).to(dtype).cuda(), w[:, :4].contiguous().cuda(), act=act)  # z on a diagonal through the product
    assert torch.equal(torch.diagonal(y.cpu().double()[:, :4]), torch.tensor([float(z[0, 1]), 0.0, 60.0, 0.0], dtype=torch.float64))
