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


def test_tails_relative_to_their_values():
    """fp32 GELU and SiLU and their slopes over both tails, relative to the 64-bit values.  U = 2^-24.  exp2's argument c z^2 is rounded twice (z^2, the product) and c once (0.23 U), so
    exp(-z^2 / 2) is off by z^2 / 2 times 2.23 U; fit, polynomial, reciprocal and products by 8 U, the two instructions' last bits (2 U each) and the product with z on top:
    (16 + 1.5 z^2) U.  SiLU: exp(-z) by |z| times 1.23 U, the rest by 8 U."""
    from simhand_amd import ops

    U = 2.0 ** -24
    z = torch.cat((torch.linspace(-12.0, 12.0, 60001), torch.linspace(-80.0, 20.0, 60001))).view(-1, 1)
    zd = z.double()
    one = torch.ones(1, 1).cuda()
    for act in ("gelu", "silu"):
        keep = (zd.abs() <= 12).view(-1) if act == "gelu" else torch.ones(len(z), dtype=torch.bool)
        v = zd[keep]
        y = ops.linear_fwd(z[keep].cuda(), one, act=act).cpu().double()  # z times one
        dz = ops.linear_act_bwd(torch.ones_like(z[keep]).cuda(), z[keep].cuda(), act)[0].cpu().double()
        if act == "gelu":
            phi, pdf = torch.erfc(v * -math.sqrt(0.5)) / 2, torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)  # (torch.special.ndtr is (1 + erf) / 2: nothing is left of it at -12)
            want, slope, rel = v * phi, phi + v * pdf, (16 + 1.5 * v * v) * U
            terms = phi + v.abs() * pdf
        else:
            s = torch.sigmoid(v)
            want, slope, rel = v * s, slope_ref(v, act), (10 + 1.5 * v.abs()) * U
            terms = s + s * v.abs() * (torch.sigmoid(-v) + 2 * U)  # 1 - s is off by s's own rounding
        assert bool(((y - want).abs() <= rel * want.abs() + 1e-37).all()), act
        assert bool(((dz - slope).abs() <= 2 * rel * terms + 4 * U * (v.abs() * torch.sigmoid(v) if act == "silu" else 0.0) + 1e-37).all()), act
