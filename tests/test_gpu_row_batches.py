"""A row's result does not depend on what else is in the batch: layer norm bit for bit (values, statistics, gate, input gradient), the layer-norm head up to the rounding of its products."""
import pytest
import torch

from tests.test_gpu_row_ops import U, dtype, randn  # noqa: F401  (dtype is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [3, 64, 129, 512, 777, 2049, 5000])
def test_layer_norm_rows_in_any_batch(dtype, cols):
    from simhand_amd import ops

    x, dy = randn(5000 if cols < 1000 else 600, cols, dtype=dtype).cuda(), randn(5000 if cols < 1000 else 600, cols, seed=3, dtype=dtype).cuda()
    gamma, beta = (1 + 0.1 * randn(cols, seed=1)).cuda(), randn(cols, seed=2).cuda()
    full = ops.layer_norm_fwd(x, gamma, beta, relu=True, want_gate=True)
    dx = ops.layer_norm_bwd(dy, x, gamma, beta, full[1], full[2], True)[0]
    c = ops.act8_pack(x)
    dx8 = ops.layer_norm_bwd(dy, c, gamma, beta, full[1], full[2], True, gate=full[3])[0]
    for s in (slice(0, 1), slice(5, 12), slice(100, 163), slice(256, 555)):
        part = ops.layer_norm_fwd(x[s], gamma, beta, relu=True, want_gate=True)
        assert all(torch.equal(a[s], b) for a, b in zip(full, part)), s
        assert torch.equal(dx[s], ops.layer_norm_bwd(dy[s], x[s], gamma, beta, part[1], part[2], True)[0]), s
        assert torch.equal(dx8[s], ops.layer_norm_bwd(dy[s], ops.act8_pack(x[s]), gamma, beta, part[1], part[2], True, gate=part[3])[0]), s


def test_head_rows_in_any_batch():
    """Two products of 512 and a norm between them, each off by its longest sum either way: 2 x 6 x 512 U of the norm, twice (two runs)."""
    from tests.test_gpu_row_paths import _model

    m = _model("18", projection_head_norm="layer")
    enc = randn(3000, 512, seed=3).cuda()
    with torch.no_grad():
        p = m._head(enc)
        for s in (slice(5, 6), slice(0, 24), slice(64, 128), slice(100, 165), slice(1000, 2025)):
            q = m._head(enc[s])
            assert float((q - p[s]).norm()) <= 2 * 2 * 6 * 512 * U * float(p[s].norm()), s
