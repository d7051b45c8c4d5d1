"""Layer norm of rows whose mean is far larger than their spread, and saved activations in 8 bits beside the fp8 configuration."""
import pytest
import torch

from tests.test_gpu_row_ops import U, close, dtype, half_step, ln_ref, randn, tiny  # noqa: F401  (dtype is a fixture)

pytestmark = pytest.mark.gpu
CHAIN = 80  # additions between a value and its row's sum: at most 64 in a lane, 6 + 2 between lanes


@pytest.mark.parametrize("rows,cols", [(33, 512), (9, 777), (3, 4100), (5, 7)])
@pytest.mark.parametrize("shift", [100.0, 10000.0])
@pytest.mark.parametrize("relu", [False, True])
def test_rows_far_from_zero(dtype, rows, cols, shift, relu):
    """Forward: the mean is off by CHAIN U of the row's mean magnitude, so h by that times rstd; the variance is taken about that mean and gains its square only.  Backward, on the
    statistics that the forward pass returned: h = x rstd - mean rstd is off by 2 U of |mean rstd| and of |x rstd|, which the mean's own rounding (U / 2 of it) costs anyway."""
    from simhand_amd import ops

    x = (randn(rows, cols) + shift).to(dtype) if dtype == torch.float32 else ((randn(rows, cols) * 8).round() * (shift / 100) + shift).to(dtype)
    gamma, beta = 1 + 0.1 * randn(cols, seed=1), 0.1 * randn(cols, seed=2)
    dy = randn(rows, cols, seed=3, dtype=dtype)
    y, mean, rstd = ops.layer_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), 1e-5, relu)
    want, m, r, h = ln_ref(x, gamma, beta, 1e-5, relu)
    xd, g = x.double(), gamma.double()
    dm = (CHAIN + 2) * U * xd.abs().mean(dim=1, keepdim=True) * r
    off = dm + (CHAIN / 2 + 8) * U * h.abs() + h.abs() * dm * dm
    close(mean, m[:, 0], (CHAIN + 2) * U * xd.abs().mean(dim=1) + 1e-30, "mean")
    close(y, want, half_step(dtype) * want.abs() + 1.01 * (off * g.abs() + 4 * U * (h * g).abs() + 4 * U * beta.double().abs()) + tiny(dtype), "y")
    m32, r32 = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
    dx, dg, db = ops.layer_norm_bwd(dy.cuda(), x.cuda(), gamma.cuda(), beta.cuda(), mean, rstd, relu)
    hh = (xd - m32) * r32
    u = dy.double()
    if relu:
        u = u * ((((x.float() - mean.cpu()[:, None]) * rstd.cpu()[:, None]) * gamma + beta) > 0)
    gg = u * g
    a, b = gg.mean(dim=1, keepdim=True), (gg * hh).mean(dim=1, keepdim=True)
    exact = r32 * (gg - a - hh * b)
    hb = 4 * U * (xd.abs() + m32.abs()) * r32
    mg, mgh = gg.abs().mean(dim=1, keepdim=True), (gg * hh).abs().mean(dim=1, keepdim=True)
    fp = r32 * (8 * U * gg.abs() + 100 * U * mg + (hh.abs() + hb) * 100 * U * mgh + hb * (b.abs() + mgh) + (hh.abs() + hb) * (gg.abs() * hb).mean(dim=1, keepdim=True))
    close(dx, exact, half_step(dtype) * exact.abs() + 2 * fp + tiny(dtype), "dx")
    close(dg, (u * hh).sum(dim=0), (rows + 8) * U * (u * hh).abs().sum(dim=0) + (u.abs() * hb).sum(dim=0) + 1e-30, "dgamma")
    close(db, u.sum(dim=0), (rows + 8) * U * u.abs().sum(dim=0) + 1e-30, "dbeta")


@pytest.mark.parametrize("size", ["18", "50"])
def test_8_bit_block_inputs_in_the_fp8_configuration(size):
    """Loss and every gradient but the packed layers' are bit for bit those of the fp8 run without them."""
    from oracle import step as orc
    from tests.test_gpu_row_paths import _model

    batch = {k: v.cuda() for k, v in orc.synthetic_batch(4, size=64, seed=5).items()}
    res = []
    for act8 in (False, True):
        m = _model(size, act8=act8)
        m.encoder.set_compute_dtype(torch.bfloat16, fp8=True)
        assert m.encoder.engine.act8 is act8 and m.encoder.engine.fp8
        out = []
        for _ in range(2):  # the second step runs on delayed scales
            m.zero_grad()
            loss = m.training_step(batch, 0)["loss"]
            loss.backward()
            out.append((loss.detach(), {k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None}))
        res.append((out, m))
    (a, m), (b, _) = res
    packed = {f"encoder.features.{li}.{bi}.conv1.weight" for li in (4, 5, 6, 7) for bi, blk in enumerate(m.encoder.features[li]) if blk.downsample is None}
    for (la, ga), (lb, gb) in zip(a, b):
        assert torch.equal(la, lb) and set(ga) == set(gb)
        for k in ga:
            if k in packed:  # (that these are the product with the codes' values is tested without fp8, by the same launch)
                assert bool(torch.isfinite(gb[k]).all()) and not torch.equal(ga[k], gb[k]), k
            else:
                assert torch.equal(ga[k], gb[k]), k
