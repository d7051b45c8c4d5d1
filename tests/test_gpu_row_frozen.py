"""Frozen arguments of the differentiable linear: the gradients that are left are the full run's, bit for bit, and the other product is not launched."""
import pytest
import torch

from tests.test_gpu_row_ops import dtype, randn  # noqa: F401  (dtype is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n", [(8, 12, 5), (300, 77, 130), (5001, 256, 512)])
@pytest.mark.parametrize("act8", [False, True])
def test_the_other_gradients_stay_as_they_are(dtype, m, k, n, act8, monkeypatch):
    from simhand_amd import ops
    from simhand_amd.host import model_utils as mu

    data = (randn(m, k, dtype=dtype).cuda(), randn(n, k, seed=1, dtype=dtype).cuda(), randn(n, seed=2).cuda())
    dy = randn(m, n, seed=3, dtype=dtype).cuda()

    def run(need):
        t = [v.clone().requires_grad_(bool(f)) for v, f in zip(data, need)]
        y = mu.linear(*t, act="gelu", act8=act8)
        y.backward(dy)
        return y.detach(), [v.grad for v in t]

    y, full = run((1, 1, 1))
    lib = ops._lib_dev()
    launched = []
    for name in ("simhand_linear_dgrad", "simhand_linear_wgrad", "simhand_act8_pack"):
        monkeypatch.setattr(lib, name, (lambda f, name: lambda *a: (launched.append(name), f(*a))[1])(getattr(lib, name), name))
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        launched.clear()
        y1, g = run(need)
        assert torch.equal(y1, y) and [v is not None for v in g] == [bool(f) for f in need]
        assert all(torch.equal(a, b) for a, b in zip(g, full) if a is not None)
        assert sorted(launched) == sorted(["simhand_linear_dgrad"] * need[0] + ["simhand_linear_wgrad"] * need[1] + ["simhand_act8_pack"] * (act8 and need[1]))


def test_linear_bwd_without_its_input():
    from simhand_amd import _lib, ops

    dz, x, w = randn(40, 9).cuda(), randn(40, 7, seed=1).cuda(), randn(9, 7, seed=2).cuda()
    dx, dw = ops.linear_bwd(dz, x, w)
    a = ops.linear_bwd(dz, None, w, need_dw=False)
    assert torch.equal(a[0], dx) and a[1] is None
    assert torch.equal(ops.linear_bwd(dz, x, w, need_dx=False)[1], dw)
    with pytest.raises(_lib.SimhandHipError):
        ops.linear_bwd(dz, None, w)
    with pytest.raises(_lib.SimhandHipError):
        ops.linear_bwd(dz, x[:, :3].contiguous(), w, need_dw=False)
