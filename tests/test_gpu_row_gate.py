"""The ReLU gate behind a layer norm whose input is kept in 8 bits: it is the forward pass's, kept as one bit a value, not the sign that the rounded input gives."""
import pytest
import torch

from tests.test_gpu_row_ops import SHAPES_LN, U, close, dtype, half_step, ln_bound, ln_ref, randn, tiny  # noqa: F401  (dtype is a fixture)

pytestmark = pytest.mark.gpu


def bits_of(gate, cols, dtype):
    """[rows][cols] of the gate's bits, from the layout that the header states: V columns a byte, the last byte of a ragged row over the row's last V columns"""
    v = 4 if dtype == torch.float32 else 8
    gate = gate.cpu().int()
    out = torch.zeros(gate.shape[0], cols, dtype=torch.bool)
    for i in range(gate.shape[1]):
        at = i * v if (i + 1) * v <= cols or cols < v else cols - v
        for e in range(min(v, cols)):
            out[:, at + e] = (gate[:, i] >> e & 1).bool()
    return out


@pytest.mark.parametrize("rows,cols", SHAPES_LN + [(5000, 96), (40, 16384), (1003, 333)])
def test_gate_of_the_forward_pass(dtype, rows, cols):
    """The bits are those of h gamma + beta > 0; nothing else changes."""
    from simhand_amd import ops

    if dtype == torch.float32 and cols > 8192:
        cols = 8192
    x = (randn(rows, cols) + 0.5).to(dtype)
    gamma, beta = 1 + 0.1 * randn(cols, seed=1), 0.1 * randn(cols, seed=2)
    plain = ops.layer_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), 1e-5, True)
    y, mean, rstd, gate = ops.layer_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), 1e-5, True, want_gate=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, (y, mean, rstd)))
    got = bits_of(gate, cols, dtype)
    if dtype == torch.float32:
        assert torch.equal(got, y.cpu() > 0)
    else:
        _, _, r, h = ln_ref(x, gamma, beta, 1e-5, True)
        z = h * gamma.double() + beta.double()
        sure = z.abs() > ln_bound(x, gamma, beta, r)
        assert torch.equal(got[sure], (z > 0)[sure])


@pytest.mark.parametrize("rows,cols", SHAPES_LN + [(5000, 96), (1003, 333)])
@pytest.mark.parametrize("act8", [False, True])
def test_backward_with_the_kept_gate(dtype, rows, cols, act8):
    """dx, dgamma, dbeta of the formula with the forward's gate and h from the saved values; dbeta, which reads no x, is bit for bit the same from the tensor and from its codes."""
    from simhand_amd import ops

    x = (randn(rows, cols) + 2.0).to(dtype)  # a mean that is large against the codes' steps: many gates that the codes would flip
    gamma, beta = 1 + 0.1 * randn(cols, seed=1), 0.1 * randn(cols, seed=2)
    dy = randn(rows, cols, seed=3, dtype=dtype)
    y, mean, rstd, gate = ops.layer_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), 1e-5, True, want_gate=True)
    xs = ops.act8_pack(x.cuda()) if act8 else x.cuda()
    xv = ops.act8_unpack(xs).cpu() if act8 else x
    dx, dg, db = ops.layer_norm_bwd(dy.cuda(), xs, gamma.cuda(), beta.cuda(), mean, rstd, True, gate=gate)
    m64, r64 = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
    h = (xv.double() - m64) * r64
    u = dy.double() * bits_of(gate, cols, dtype)
    g = u * gamma.double()
    a, b = g.mean(dim=1, keepdim=True), (g * h).mean(dim=1, keepdim=True)
    want = r64 * (g - a - h * b)
    mg, mgh = g.abs().mean(dim=1, keepdim=True), (g * h).abs().mean(dim=1, keepdim=True)
    hb = 4 * U * (xv.double().abs() + m64.abs()) * r64  # error of h
    fp = r64 * (8 * U * g.abs() + 100 * U * mg + (h.abs() + hb) * 100 * U * mgh + hb * (b.abs() + mgh) + h.abs() * (g.abs() * hb).mean(dim=1, keepdim=True))
    close(dx, want, half_step(dtype) * want.abs() + 2 * fp + tiny(dtype), "dx")
    n = rows + 8
    close(dg, (u * h).sum(dim=0), n * U * (u * h).abs().sum(dim=0) + (u.abs() * hb).sum(dim=0) + 1e-30, "dgamma")
    close(db, u.sum(dim=0), n * U * u.abs().sum(dim=0) + 1e-30, "dbeta")
    assert torch.equal(db, ops.layer_norm_bwd(dy.cuda(), x.cuda(), gamma.cuda(), beta.cuda(), mean, rstd, True)[2])  # the gate recomputed from the tensor: the same


@pytest.mark.parametrize("shift", [0.5, 2.0, 8.0])
@pytest.mark.parametrize("rows,cols", [(300, 512), (64, 777), (20, 3)])
def test_function_with_relu_and_an_8_bit_input(rows, cols, shift):
    """mu.layer_norm(relu, act8): dbeta is the uncompressed run's, bit for bit; dx and dgamma are the formula's with that run's gate and the codes' values."""
    from simhand_amd import ops
    from simhand_amd.host import model_utils as mu

    x, dy = randn(rows, cols) + shift, randn(rows, cols, seed=3)
    gamma, beta = 1 + 0.1 * randn(cols, seed=1), 0.1 * randn(cols, seed=2)

    def run(act8):
        t = [v.cuda().requires_grad_() for v in (x, gamma, beta)]
        y = mu.layer_norm(*t, relu=True, act8=act8)
        y.backward(dy.cuda())
        return y.detach(), [v.grad for v in t]

    (ya, ga), (yb, gb) = run(False), run(True)
    assert torch.equal(ya, yb) and torch.equal(ga[2], gb[2])
    xv = ops.act8_unpack(ops.act8_pack(x.cuda())).double().cpu()
    _, m, r, _ = ln_ref(x, gamma, beta, 1e-5, True)
    h = (xv - m) * r
    u = dy.double() * (ya.cpu() > 0)
    g = u * gamma.double()
    want = r * (g - g.mean(dim=1, keepdim=True) - h * (g * h).mean(dim=1, keepdim=True))
    # the statistics are off by 100 U of (|x| r)^2 (a mean, a variance), h by as much and its own roundings: every term of dx by that
    off = 200 * U * (1 + (x.double().abs().amax(dim=1, keepdim=True) * r) ** 2)
    mgh = (g * h).abs().mean(dim=1, keepdim=True)
    bound = r * off * (g.abs() + g.abs().mean(dim=1, keepdim=True) + (1 + h.abs()) * (2 * mgh + g.abs().mean(dim=1, keepdim=True)))
    close(gb[0], want, bound + 1e-30, "dx")
    close(gb[1], (u * h).sum(dim=0), (off * u.abs() * (1 + h.abs())).sum(dim=0) + (rows + 8) * U * (u * h).abs().sum(dim=0) + 1e-30, "dgamma")


def test_gate_over_several_launches_and_nothing_beside_it():
    """More rows than one forward launch takes; guard bytes around a gate of odd size stay as they were."""
    from simhand_amd import _lib, ops

    torch.cuda.empty_cache()
    rows, edge, cols = (1 << 27) + 70, 1 << 27, 9  # groups of 16 lanes: 2^27 rows a launch
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_()
    gamma, beta = randn(cols, seed=1).cuda(), randn(cols, seed=2).cuda()
    gate = ops.layer_norm_fwd(x, gamma, beta, relu=True, want_gate=True)[3]
    for s in (slice(0, 70), slice(edge - 70, rows)):
        assert torch.equal(gate[s], ops.layer_norm_fwd(x[s], gamma, beta, relu=True, want_gate=True)[3]), s
    del x, gate
    torch.cuda.empty_cache()
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    for rows, cols in ((131, 45), (3, 5), (7, 2049)):
        x, g = randn(rows, cols).cuda(), torch.ones(cols, device="cuda")
        n = rows * ((cols + 3) // 4)
        buf = torch.full((n + 128,), 7, dtype=torch.uint8, device="cuda")
        y, m, r = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        assert lib.simhand_layer_norm_fwd_ex(x.data_ptr(), g.data_ptr(), g.data_ptr(), 1e-5, 1, y.data_ptr(), buf.data_ptr() + 64, m.data_ptr(), r.data_ptr(), rows, cols, 0, st) == 0
        torch.cuda.synchronize()
        assert bool((buf[:64] == 7).all()) and bool((buf[-64:] == 7).all()) and bool((buf[64:-64] < 16).all())


def test_gate_refusals():
    from simhand_amd import _lib, ops

    x, g = torch.zeros(4, 9, device="cuda"), torch.ones(9, device="cuda")
    y, m, r, gate = ops.layer_norm_fwd(x, g, g, relu=True, want_gate=True)
    assert gate.shape == (4, 3)
    for f in (lambda: ops.layer_norm_fwd(x, g, g, want_gate=True), lambda: ops.layer_norm_bwd(x, x, g, g, m, r, False, gate=gate),
              lambda: ops.layer_norm_bwd(x, x, g, g, m, r, True, gate=gate[:, :2].contiguous()), lambda: ops.layer_norm_bwd(x, x, g, g, m, r, True, gate=gate.int()),
              lambda: ops.layer_norm_bwd(x, x, g, g, m, r, True, gate=gate.cpu())):
        with pytest.raises(_lib.SimhandHipError):
            f()


def test_other_shapes_no_rows_and_two_streams(dtype):
    """Leading dimensions, no rows at all, and the same call on two streams at once."""
    from simhand_amd import ops
    from simhand_amd.host import model_utils as mu

    x, dy = (randn(6, 7, 45) + 1).to(dtype), randn(6, 7, 45, seed=3, dtype=dtype)
    gamma, beta = (1 + 0.1 * randn(45, seed=1)).cuda(), (0.1 * randn(45, seed=2)).cuda()

    def run(shape):
        t = [v.clone().requires_grad_() for v in (x.cuda().view(shape), gamma, beta)]
        y = mu.layer_norm(*t, relu=True, act8=True)
        y.backward(dy.cuda().view(shape))
        return [y.detach().view(-1), t[0].grad.view(-1), t[1].grad, t[2].grad]

    want = run((42, 45))
    assert all(torch.equal(a, b) for a, b in zip(want, run((6, 7, 45))))
    e = torch.empty(0, 45, dtype=dtype, device="cuda")
    y, m, r, gate = ops.layer_norm_fwd(e, gamma, beta, relu=True, want_gate=True)
    assert gate.shape[0] == 0
    dx, dg, db = ops.layer_norm_bwd(e, ops.act8_pack(e), gamma, beta, m, r, True, gate=gate)
    assert dx.shape == (0, 45) and not bool(dg.any()) and not bool(db.any())
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got[i] = run((42, 45))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))
