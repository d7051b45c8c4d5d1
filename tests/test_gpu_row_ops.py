"""Layer norm, linear and 8-bit activations (simhand_amd.ops) against their formulas in 64 bits on the CPU.

Tolerances are counted, not tuned: an output rounded once to a type is off by half a step (finfo.eps / 2, relative); an fp32 sum of n terms by at most
n 2^-24 of the sum of its terms' magnitudes (twice that where the matrix cores add: they need not round to nearest at every step)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(params=["fp32", "bf16", "fp16"])
def dtype(request):
    from simhand_amd import _lib

    _lib.use_half("f16" if request.param == "fp16" else "bf16")
    yield TYPES[request.param]
    _lib.use_half("bf16")


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps  # the smallest subnormal: half of it is lost below the normal range


def close(got, want, tol, what=""):
    err = (got.detach().double().cpu() - want).abs()
    bad = err > tol
    assert not bool(bad.any()) and not bool(torch.isnan(err).any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp(min=1e-300)).max()):.3g} of the tolerance"


def randn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed + 1000 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ------------------------------------------------------------------ layer norm
SHAPES_LN = [(1, 1), (3, 2), (5, 7), (1, 31), (64, 64), (17, 129), (33, 512), (9, 777), (4, 2048), (6, 2049), (3, 4100), (2, 8192), (257, 48)]


def ln_ref(x, gamma, beta, eps, relu):
    x, gamma, beta = x.double(), gamma.double(), beta.double()
    m = x.mean(dim=1, keepdim=True)
    r = 1.0 / torch.sqrt((x - m).square().mean(dim=1, keepdim=True) + eps)
    h = (x - m) * r
    y = h * gamma + beta
    return (y.clamp(min=0) if relu else y), m, r, h


def ln_bound(x, gamma, beta, r):
    """fp32 error of one normalised value: the mean is off by (its longest chain of additions, < 80) U of the row's mean magnitude, everything else by a few U"""
    x = x.double()
    mag = x.abs().mean(dim=1, keepdim=True) + x.abs()
    return 100 * U * (mag * r * (1 + mag * r) * gamma.double().abs() + beta.double().abs()) + 4 * U


@pytest.mark.parametrize("rows,cols", SHAPES_LN)
@pytest.mark.parametrize("relu", [False, True])
def test_layer_norm_forward(dtype, rows, cols, relu):
    from simhand_amd import ops

    x = (randn(rows, cols) + 0.5).to(dtype)
    gamma, beta = 1 + 0.1 * randn(cols, seed=1), 0.1 * randn(cols, seed=2)
    y, mean, rstd = ops.layer_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), 1e-5, relu)
    want, m, r, _ = ln_ref(x, gamma, beta, 1e-5, relu)
    fp = ln_bound(x, gamma, beta, r)
    close(y, want, half_step(dtype) * want.abs() + fp * (1 + half_step(dtype)) + tiny(dtype), "y")
    close(mean, m[:, 0], 100 * U * x.double().abs().mean(dim=1) + 1e-30, "mean")
    var_r = r[:, 0] * 100 * U * (1 + (x.double().abs().amax(dim=1) * r[:, 0]) ** 2)
    close(rstd, r[:, 0], var_r, "rstd")


@pytest.mark.parametrize("rows,cols", SHAPES_LN + [(5000, 96)])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("act8", [False, True])
def test_layer_norm_backward(dtype, rows, cols, relu, act8):
    from simhand_amd import ops

    x = (randn(rows, cols) + 0.5).to(dtype)
    gamma, beta = 1 + 0.1 * randn(cols, seed=1), 0.1 * randn(cols, seed=2)
    dy = randn(rows, cols, seed=3, dtype=dtype)
    xs = ops.act8_pack(x.cuda()) if act8 else x.cuda()
    xv = ops.act8_unpack(xs).cpu() if act8 else x
    _, m, r, _ = ln_ref(xv, gamma, beta, 1e-5, relu)
    m32, r32 = m[:, 0].float(), r[:, 0].float()
    dx, dg, db = ops.layer_norm_bwd(dy.cuda(), xs, gamma.cuda(), beta.cuda(), m32.cuda(), r32.cuda(), relu)
    # the formula on the statistics that were handed in; the gate exactly as documented: h gamma + beta in fp32
    r64 = r32.double()[:, None]
    h = (xv.double() - m32.double()[:, None]) * r64
    u = dy.double()
    if relu:
        z32 = ((xv.float() - m32[:, None]) * r32[:, None]) * gamma + beta
        u = u * (z32 > 0)
    g = u * gamma.double()
    a, b = g.mean(dim=1, keepdim=True), (g * h).mean(dim=1, keepdim=True)
    want = r64 * (g - a - h * b)
    mg, mgh = g.abs().mean(dim=1, keepdim=True), (g * h).abs().mean(dim=1, keepdim=True)
    hb = 4 * U * (xv.double().abs() + m32.double().abs()[:, None]) * r64  # error of h
    fp = r64 * (8 * U * g.abs() + 100 * U * mg + (h.abs() + hb) * 100 * U * mgh + hb * (b.abs() + mgh) + h.abs() * (g.abs() * hb).mean(dim=1, keepdim=True))
    close(dx, want, half_step(dtype) * want.abs() + 2 * fp + tiny(dtype), "dx")
    n = rows + 8
    close(dg, (u * h).sum(dim=0), n * U * (u * h).abs().sum(dim=0) + (u.abs() * hb).sum(dim=0) + 1e-30, "dgamma")
    close(db, u.sum(dim=0), n * U * u.abs().sum(dim=0) + 1e-30, "dbeta")


def test_layer_norm_gradient_against_differences():
    """fp32: the backward pass against central differences of the 64-bit formula along random directions."""
    from simhand_amd import ops

    rows, cols = 6, 37
    x, gamma, beta = randn(rows, cols).double(), 1 + 0.2 * randn(cols, seed=1).double(), randn(cols, seed=2).double()
    dy = randn(rows, cols, seed=3)
    y, mean, rstd = ops.layer_norm_fwd(x.float().cuda(), gamma.float().cuda(), beta.float().cuda())
    dx, dg, db = (t.double().cpu() for t in ops.layer_norm_bwd(dy.cuda(), x.float().cuda(), gamma.float().cuda(), beta.float().cuda(), mean, rstd))
    f = lambda a, b, c: (ln_ref(a, b, c, 1e-5, False)[0] * dy.double()).sum()  # noqa: E731
    for s in range(3):
        ex, eg, eb = randn(rows, cols, seed=10 + s).double(), randn(cols, seed=20 + s).double(), randn(cols, seed=30 + s).double()
        h = 1e-5
        num = (f(x + h * ex, gamma + h * eg, beta + h * eb) - f(x - h * ex, gamma - h * eg, beta - h * eb)) / (2 * h)
        got = (dx * ex).sum() + (dg * eg).sum() + (db * eb).sum()
        # fp32 gradients: each of the 222 + 74 products is off by at most ~100 U; differences: h^2
        assert abs(float(num - got)) < 1e-4 * float((dx * ex).abs().sum() + (dg * eg).abs().sum() + (db * eb).abs().sum())


def test_layer_norm_constant_rows_and_bad_rows():
    """A row of equal values has variance zero (y = beta); NaN and infinite rows stay by themselves."""
    from simhand_amd import ops

    x = randn(6, 40)
    x[1] = 3.0
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    gamma, beta = 1 + 0.1 * randn(40, seed=1), randn(40, seed=2)
    y, mean, rstd = (t.cpu() for t in ops.layer_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda()))
    assert torch.equal(y[1], beta) and abs(float(rstd[1]) - 1e5 ** 0.5) < 1e-3
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    want = ln_ref(x[[0, 4, 5]], gamma, beta, 1e-5, False)[0]
    close(y[[0, 4, 5]], want, torch.full_like(want, 1e-5))


# ---------------------------------------------------------------------- linear
def act_ref(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z)}[act]()


def slope_ref(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


SHAPES_LIN = [(1, 1, 1), (1, 2048, 512), (3, 5, 7), (8, 64, 64), (130, 33, 129), (64, 512, 128), (257, 100, 77), (129, 256, 130), (300, 777, 61), (512, 64, 256), (128, 1024, 384)]


@pytest.mark.parametrize("m,k,n", SHAPES_LIN)
@pytest.mark.parametrize("act,bias,residual,pre", [("none", False, False, False), ("relu", True, True, True), ("gelu", True, False, True),
                                                  ("silu", False, True, False), ("gelu", True, True, False)])
def test_linear_forward(dtype, m, k, n, act, bias, residual, pre):
    from simhand_amd import ops

    x, w = randn(m, k, dtype=dtype), randn(n, k, seed=1, scale=k ** -0.5, dtype=dtype)
    b = randn(n, seed=2) if bias else None
    res = randn(m, n, seed=3, dtype=dtype) if residual else None
    out = ops.linear_fwd(x.cuda(), w.cuda(), b.cuda() if bias else None, act=act, residual=res.cuda() if residual else None, want_pre=pre)
    y, zp = out if pre else (out, None)
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if bias:
        z, mag = z + b.double(), mag + b.double().abs()
    fz = 2 * (k + 2) * U * mag
    want = act_ref(z, act)
    fy = 1.13 * fz + 8 * U * (z.abs() + 1e-30)  # |act'| <= 1.13; erf / exp to a few units
    if residual:
        want = want + res.double()
        fy = fy + U * (want.abs() + z.abs())
    close(y, want, half_step(dtype) * want.abs() + 1.01 * fy + tiny(dtype), "y")
    if pre:
        close(zp, z, half_step(dtype) * z.abs() + 1.01 * fz + tiny(dtype), "pre")


# the kernel for many rows (16 bits, rows of 16-byte chunks, at least 192 tiles of 256 x 256): whole tiles, ragged rows / columns / K, one to five k-steps, the smallest N, several
# tiles per block
SHAPES_MANY = [(49152, 64, 256), (49100, 72, 136), (24600, 128, 520), (6200, 320, 2048), (30011, 8, 384), (131072 + 40, 200, 128), (16640, 136, 1032),
               (16384, 512, 1024), (16389, 384, 1024), (33000, 256, 576), (70001, 120, 320), (66000, 72, 256), (9000, 504, 2048), (524288 + 3, 64, 64),
               (40001, 77, 333), (33333, 333, 520), (20003, 777, 333), (66001, 130, 128), (16400, 1001, 500), (131073, 45, 130), (30000, 513, 300)]


@pytest.mark.parametrize("m,k,n", SHAPES_MANY)
@pytest.mark.parametrize("act,bias,residual,pre", [("none", False, False, False), ("relu", True, True, False), ("gelu", True, True, True), ("silu", False, False, True)])
def test_linear_forward_many_rows(dtype, m, k, n, act, bias, residual, pre):
    from simhand_amd import ops

    if dtype == torch.float32:
        m = m // 16 + 5  # the tile kernel's own sizes are covered above; its 128-wide tiles start at 512 of them
    x, w = randn(m, k, dtype=dtype), randn(n, k, seed=1, scale=k ** -0.5, dtype=dtype)
    b = randn(n, seed=2) if bias else None
    res = randn(m, n, seed=3, dtype=dtype) if residual else None
    out = ops.linear_fwd(x.cuda(), w.cuda(), b.cuda() if bias else None, act=act, residual=res.cuda() if residual else None, want_pre=pre)
    y, zp = out if pre else (out, None)
    xd, wd = x.cuda().double(), w.cuda().double()  # 64-bit products on the GPU (plain torch): too many for the CPU
    z, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias:
        z, mag = z + b.cuda().double(), mag + b.cuda().double().abs()
    fz = 2 * (k + 2) * U * mag
    want = act_ref(z, act)
    fy = 1.13 * fz + 8 * U * (z.abs() + 1e-30)
    if residual:
        want = want + res.cuda().double()
        fy = fy + U * (want.abs() + z.abs())
    assert bool(((y.double() - want).abs() <= half_step(dtype) * want.abs() + 1.01 * fy + tiny(dtype)).all())
    if pre:
        assert bool(((zp.double() - z).abs() <= half_step(dtype) * z.abs() + 1.01 * fz + tiny(dtype)).all())


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 9), (7, 64), (100, 33), (513, 128), (129, 512), (2050, 77), (64, 2048)])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_linear_act_backward(dtype, rows, cols, act):
    from simhand_amd import ops

    dy, z = randn(rows, cols, dtype=dtype), 2 * randn(rows, cols, seed=1)
    z.view(-1)[::7] = 0.0
    z = z.to(dtype)
    dz, db = ops.linear_act_bwd(dy.cuda(), z.cuda() if act != "none" else None, act)
    want = dy.double() * slope_ref(z.double(), act)
    fp = 16 * U * dy.double().abs() * (1 + z.double().abs())
    close(dz, want, half_step(dtype) * want.abs() + fp + tiny(dtype), "dz")
    close(db, want.sum(dim=0), (rows + 4) * U * want.abs().sum(dim=0) + fp.sum(dim=0) + 1e-30, "db")


@pytest.mark.parametrize("m,k,n", SHAPES_LIN + [(33, 1, 1), (39, 3, 1), (65, 1, 9), (36, 2, 3), (8, 1, 1), (7, 500, 300), (6, 1, 3000), (5000, 64, 64), (4097, 40, 72), (1000, 256, 512), (2048, 520, 264), (70, 264, 1032), (5, 128, 136), (8200, 72, 200), (300, 1024, 776), (259, 820, 1024)])
@pytest.mark.parametrize("act8", [False, True])
def test_linear_backward(dtype, m, k, n, act8):
    from simhand_amd import ops

    x, w, dz = randn(m, k, dtype=dtype), randn(n, k, seed=1, dtype=dtype), randn(m, n, seed=2, dtype=dtype)
    xs = ops.act8_pack(x.cuda()) if act8 else x.cuda()
    xv = ops.act8_unpack(xs).cpu() if act8 else x
    dx, dw = ops.linear_bwd(dz.cuda(), xs, w.cuda())
    want = dz.double() @ w.double()
    close(dx, want, half_step(dtype) * want.abs() + 1.01 * 2 * (n + 2) * U * (dz.double().abs() @ w.double().abs()) + tiny(dtype), "dx")
    close(dw, dz.double().t() @ xv.double(), 2 * (m + 40) * U * (dz.double().abs().t() @ xv.double().abs()) + 1e-30, "dw")
    assert ops.linear_bwd(dz.cuda(), xs, w.cuda(), need_dx=False)[0] is None


# the kernels for many rows (weight gradient: at least 4096 rows and 192 columns on both sides; input gradient: 192 tiles): whole and ragged tiles, rows that end inside a step,
# one and several tiles, ranges of rows that leave some blocks with less
@pytest.mark.parametrize("m,k,n", [(4096, 256, 256), (49152, 256, 256), (49157, 200, 328), (8195, 512, 200), (6001, 384, 1024), (20000, 1024, 264), (33333, 640, 192),
                                   (20001, 333, 257), (5003, 777, 131), (30000, 64, 64), (40001, 50, 61), (17000, 100, 30), (100001, 129, 7), (4097, 260, 2047)])
@pytest.mark.parametrize("act8", [False, True])
def test_linear_backward_many_rows(dtype, m, k, n, act8):
    from simhand_amd import ops

    x, w, dz = randn(m, k, dtype=dtype).cuda(), randn(n, k, seed=1, dtype=dtype).cuda(), randn(m, n, seed=2, dtype=dtype).cuda()
    xs = ops.act8_pack(x) if act8 else x
    xv = ops.act8_unpack(xs).double() if act8 else x.double()
    dx, dw = ops.linear_bwd(dz, xs, w)
    zd, wd = dz.double(), w.double()
    want = zd @ wd
    assert bool(((dx.double() - want).abs() <= half_step(dtype) * want.abs() + 1.01 * 2 * (n + 2) * U * (zd.abs() @ wd.abs()) + tiny(dtype)).all())
    assert bool(((dw.double() - zd.t() @ xv).abs() <= 2 * (m + 40) * U * (zd.abs().t() @ xv.abs()) + 1e-30).all())


def test_linear_gradient_against_differences():
    """fp32: dz, db, dx, dw against central differences of the 64-bit formula along random directions."""
    from simhand_amd import ops

    m, k, n = 9, 21, 13
    x, w, b = randn(m, k).double(), randn(n, k, seed=1).double(), randn(n, seed=2).double()
    dy = randn(m, n, seed=3)
    for act in ("gelu", "silu"):
        _, pre = ops.linear_fwd(x.float().cuda(), w.float().cuda(), b.float().cuda(), act=act, want_pre=True)
        dz, db = ops.linear_act_bwd(dy.cuda(), pre, act)
        dx, dw = ops.linear_bwd(dz, x.float().cuda(), w.float().cuda())
        f = lambda p, q, r: (act_ref(p @ q.t() + r, act) * dy.double()).sum()  # noqa: E731
        for s in range(3):
            e = [randn(*t.shape, seed=10 * s + i).double() for i, t in enumerate((x, w, b))]
            h = 1e-5
            num = (f(x + h * e[0], w + h * e[1], b + h * e[2]) - f(x - h * e[0], w - h * e[1], b - h * e[2])) / (2 * h)
            parts = [(g.double().cpu() * t) for g, t in zip((dx, dw, db), e)]
            assert abs(float(num - sum(p.sum() for p in parts))) < 1e-4 * float(sum(p.abs().sum() for p in parts))


def test_linear_many_rows_at_odd_addresses(dtype):
    """Whole rows whose first element is not at a 16-byte address, and one operand of each kind."""
    from simhand_amd import ops

    m, k, n = 40000, 128, 192
    xb, wb = randn(m * k + 5, dtype=dtype).cuda(), randn(n * k + 3, seed=1, dtype=dtype).cuda()
    for ox, ow in ((5, 0), (0, 3), (1, 1), (0, 0)):
        x, w = xb[ox:ox + m * k].view(m, k), wb[ow:ow + n * k].view(n, k)
        y = ops.linear_fwd(x, w)
        want, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
        assert bool(((y.double() - want).abs() <= half_step(dtype) * want.abs() + 2.02 * (k + 2) * U * mag + tiny(dtype)).all()), (ox, ow)
        dz = y[:, :].contiguous()
        dx, dw = ops.linear_bwd(dz, x, w)
        zd = dz.double()
        assert bool(((dx.double() - zd @ w.double()).abs() <= half_step(dtype) * (zd @ w.double()).abs() + 2.02 * (n + 2) * U * (zd.abs() @ w.double().abs()) + tiny(dtype)).all())
        assert bool(((dw.double() - zd.t() @ x.double()).abs() <= 2 * (m + 40) * U * (zd.abs().t() @ x.double().abs())).all())


def test_linear_unaligned_and_inplace_residual(dtype):
    """Operands that start in the middle of a buffer (element alignment only), and a residual that is the output of an earlier call."""
    from simhand_amd import ops

    m, k, n = 70, 45, 53
    buf = randn(m * k + 3, dtype=dtype).cuda()
    x = buf[3:].view(m, k)
    wb = randn(n * k + 1, seed=1, dtype=dtype).cuda()
    w = wb[1:].view(n, k)
    y = ops.linear_fwd(x, w)
    want = x.double().cpu() @ w.double().cpu().t()
    tol = half_step(dtype) * want.abs() + 2.02 * (k + 2) * U * (x.double().abs().cpu() @ w.double().abs().cpu().t()) + tiny(dtype)
    close(y, want, tol)
    assert torch.equal(ops.linear_fwd(x.clone(), w.clone()), y)
    y2 = ops.linear_fwd(x, w, residual=y)
    assert float((y2.double() - 2 * y.double()).abs().max()) <= float((2 * tol + half_step(dtype) * 2 * want.abs() + tol).max())


# ------------------------------------------------------------------------ act8
def act8_ref(x, hold):
    """codes and exponents from the definition, in 64 bits on the CPU: the nearest value of the e4m3 grid, ties to the even code"""
    rows, cols = x.shape
    nb = -(-cols // 32)
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    v = torch.zeros(rows, nb * 32, dtype=torch.float64)
    v[:, :cols] = x.double()
    v = v.view(rows, nb, 32)
    fin = torch.isfinite(v)
    top = torch.where(fin, v.abs(), torch.zeros_like(v)).amax(dim=2)
    e = torch.full(top.shape, -126, dtype=torch.int64)
    for k in range(-126, 128):
        e = torch.where(top > 448.0 * 2.0 ** k, torch.full_like(e, k + 1), e)
    a = torch.where(fin, v.abs(), torch.zeros_like(v)).clamp(max=hold) * torch.pow(torch.tensor(2.0, dtype=torch.float64), -e.double()).unsqueeze(2)
    hi = torch.searchsorted(grid, a.contiguous()).clamp_(max=126)
    lo = (hi - 1).clamp_(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    q = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    codes = q + 128 * torch.signbit(v).long()
    codes = torch.where(fin, codes, torch.full_like(codes, 127))
    val = grid[q] * torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double()).unsqueeze(2) * torch.where(torch.signbit(v), -1.0, 1.0)
    val = torch.where(fin, val, torch.full_like(val, math.nan))
    return codes.view(rows, -1)[:, :cols], e + 127, val.view(rows, -1)[:, :cols]


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 15), (3, 16), (5, 17), (4, 32), (7, 33), (9, 64), (33, 100), (64, 512), (17, 777), (3, 2048)])
def test_act8_codes_and_values(dtype, rows, cols):
    from simhand_amd import ops

    hold = 61440.0 if dtype == torch.float16 else 1.875 * 2.0 ** 127
    x = randn(rows, cols) * torch.pow(10.0, 3 * randn(rows, 1, seed=5).clamp(-2, 1.2))
    x.view(-1)[::5] = 0.0
    x = x.to(dtype)
    c = ops.act8_pack(x.cuda())
    codes, exps, val = act8_ref(x, hold)
    assert torch.equal(c.exps.cpu().long(), exps)
    got = c.codes.cpu().long()
    assert torch.equal(torch.where(got & 127 == 127, torch.full_like(got, 127), got), codes)
    assert torch.equal(ops.act8_unpack(c).cpu(), val.to(dtype))


def test_act8_edges(dtype):
    """All-zero blocks, the type's extremes, subnormals, ties, infinities and NaN, and their neighbours in the same block of 32."""
    from simhand_amd import ops

    f = torch.finfo(dtype)
    hold = 61440.0 if dtype == torch.float16 else 1.875 * 2.0 ** 127
    x = torch.zeros(9, 70)
    x[1] = f.max
    x[2, ::2] = -f.max
    x[3] = f.smallest_normal
    x[4] = f.smallest_normal * f.eps * torch.arange(70)
    x[5] = torch.tensor([math.nan, 1.0, -2.0, math.inf, 3.0, -math.inf, 1e-3] * 10)
    x[6] = (256.0 + 16.0 * torch.arange(70)).clamp(max=448.0) + 8.0  # ties of the grid at scale 1 and 2
    x[7] = torch.linspace(-448.0, 448.0, 70)
    x[8] = torch.linspace(-1.75, 1.76, 70)
    x = x.to(dtype)
    c = ops.act8_pack(x.cuda())
    codes, exps, val = act8_ref(x, hold)
    assert torch.equal(c.exps.cpu().long(), exps)
    got = c.codes.cpu().long()
    assert torch.equal(torch.where(got & 127 == 127, torch.full_like(got, 127), got), codes)
    back = ops.act8_unpack(c).cpu()
    want = val.to(dtype)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(back.double()), torch.nan_to_num(want.double())) and not bool(torch.isinf(back).any())


def test_act8_error_is_the_codes_rounding(dtype):
    """Normal codes are off by at most 2^-4 of the value; below the grid's normal range by half its smallest step."""
    from simhand_amd import ops

    x = randn(50, 96, dtype=dtype)
    c = ops.act8_pack(x.cuda())
    back = ops.act8_unpack(c).double().cpu()
    scale = torch.pow(2.0, c.exps.cpu().double() - 127).repeat_interleave(32, dim=1)
    assert bool(((back - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)).all())


# -------------------------------------------------------- empty, together, graphs, streams
def test_no_rows(dtype):
    from simhand_amd import ops

    z = lambda *s: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
    gamma, beta = torch.ones(24, device="cuda"), torch.zeros(24, device="cuda")
    y, mean, rstd = ops.layer_norm_fwd(z(0, 24), gamma, beta)
    assert y.shape == (0, 24) and mean.shape == (0,) and rstd.shape == (0,)
    dx, dg, db = ops.layer_norm_bwd(z(0, 24), z(0, 24), gamma, beta, mean, rstd)
    assert dx.shape == (0, 24) and not bool(dg.any()) and not bool(db.any())
    w = z(7, 24).fill_(1.0)
    assert ops.linear_fwd(z(0, 24), w).shape == (0, 7)
    dz, b = ops.linear_act_bwd(z(0, 7), z(0, 7), "gelu")
    assert dz.shape == (0, 7) and not bool(b.any())
    dx, dw = ops.linear_bwd(z(0, 7), z(0, 24), w)
    assert dx.shape == (0, 24) and dw.shape == (7, 24) and not bool(dw.any())
    c = ops.act8_pack(z(0, 24))
    assert ops.act8_unpack(c).shape == (0, 24)


def mlp_step(ops, x, p, dy, act8):
    """x + W2 gelu(W1 LN(x) + b1) + b2 and its gradients as a training step would run them, saved activations as they are or in 8 bits"""
    h, mean, rstd = ops.layer_norm_fwd(x, p["gamma"], p["beta"])
    a, pre = ops.linear_fwd(h, p["w1"], p["b1"], act="gelu", want_pre=True)
    y = ops.linear_fwd(a, p["w2"], p["b2"], residual=x)
    sx, sh, sa = (ops.act8_pack(t) for t in (x, h, a)) if act8 else (x, h, a)
    dz2, db2 = ops.linear_act_bwd(dy)
    da, dw2 = ops.linear_bwd(dz2, sa, p["w2"])
    dz1, db1 = ops.linear_act_bwd(da, pre, "gelu")
    dh, dw1 = ops.linear_bwd(dz1, sh, p["w1"])
    dx, dg, db = ops.layer_norm_bwd(dh, sx, p["gamma"], p["beta"], mean, rstd)
    dx = dx + dy  # the residual's gradient
    return {"y": y, "dx": dx, "dgamma": dg, "dbeta": db, "dw1": dw1, "db1": db1, "dw2": dw2, "db2": db2}


def mlp_state(rows, c, hid, dtype):
    p = {"gamma": 1 + 0.1 * randn(c, seed=1), "beta": 0.1 * randn(c, seed=2), "w1": randn(hid, c, seed=3, scale=c ** -0.5, dtype=dtype), "b1": 0.1 * randn(hid, seed=4),
         "w2": randn(c, hid, seed=5, scale=hid ** -0.5, dtype=dtype), "b2": 0.1 * randn(c, seed=6)}
    return randn(rows, c, seed=7, dtype=dtype).cuda(), {k: v.cuda() for k, v in p.items()}, randn(rows, c, seed=8, dtype=dtype).cuda()


@pytest.mark.parametrize("act8", [False, True])
def test_a_block_of_them_together(dtype, act8):
    """The operators in the order a training step runs them, against autograd of the formula in 64 bits.  Norm-wise: every stored tensor between them is rounded once
    (half a step, independent from value to value), the saved activations by 2^-4 at most where they are kept in 8 bits."""
    from simhand_amd import ops

    x, p, dy = mlp_state(200, 136, 264, dtype)
    got = mlp_step(ops, x, p, dy, act8)
    q = {k: v.double().cpu().requires_grad_() for k, v in p.items()}
    xd = x.double().cpu().requires_grad_()
    h = ln_ref_grad(xd, q["gamma"], q["beta"])
    z = h @ q["w1"].t() + q["b1"]
    y = (z * torch.special.ndtr(z)) @ q["w2"].t() + q["b2"] + xd
    y.backward(dy.double().cpu())
    want = {"y": y.detach(), "dx": xd.grad, "dgamma": q["gamma"].grad, "dbeta": q["beta"].grad, "dw1": q["w1"].grad, "db1": q["b1"].grad, "dw2": q["w2"].grad, "db2": q["b2"].grad}
    # at most 8 rounded tensors stand between an input and an output, each at most half a step of its own norm, amplified at most by 4 (|act'| 1.13, unit-scale weights)
    tol = 8 * 4 * half_step(dtype) + 1e-5
    tol8 = tol + 3 * 2.0 ** -4  # up to three saved tensors (x in dx and dgamma, h in dw1, a in dw2) are off by 2^-4
    for k, v in want.items():
        rel = float((got[k].double().cpu() - v).norm() / v.norm())
        assert rel <= (tol8 if act8 and k in ("dx", "dgamma", "dw1", "dw2") else tol), (k, rel)


def ln_ref_grad(x, gamma, beta):
    m = x.mean(dim=1, keepdim=True)
    r = 1.0 / torch.sqrt((x - m).square().mean(dim=1, keepdim=True) + 1e-5)
    return (x - m) * r * gamma + beta


def test_results_do_not_depend_on_the_run(dtype):
    """Fixed orders everywhere: the same call gives the same bits."""
    from simhand_amd import ops

    x, p, dy = mlp_state(3000, 136, 264, dtype)
    a, b = mlp_step(ops, x, p, dy, True), mlp_step(ops, x, p, dy, True)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_captured_and_replayed(dtype):
    """The whole block in a graph, replayed with new inputs between eager work: every replay equals the eager result."""
    from simhand_amd import ops

    x, p, dy = mlp_state(300, 136, 264, dtype)
    mlp_step(ops, x, p, dy, True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp_step(ops, x, p, dy, True)
    for s in range(3):
        x.copy_(randn(*x.shape, seed=50 + s, dtype=dtype))
        eager = mlp_step(ops, x, p, dy, True)
        eager = {k: v.clone() for k, v in eager.items()}
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[k], eager[k]) for k in eager), s


def test_two_streams_at_once(dtype):
    """Calls on two streams do not share anything (workspaces are the caller's)."""
    from simhand_amd import ops

    s1, s2 = mlp_state(2000, 136, 264, dtype), mlp_state(1500, 72, 520, dtype)
    want = [mlp_step(ops, *s, True) for s in (s1, s2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate((s1, s2)):
            with torch.cuda.stream(streams[i]):
                got[i] = mlp_step(ops, *s, True)
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(w[k], g[k]) for k in w)


def test_nothing_is_written_beside_the_outputs(dtype):
    """Guard values around outputs of odd sizes stay as they were (outputs placed in the middle of a larger buffer through the C entry points)."""
    import ctypes as C

    from simhand_amd import _lib, ops

    lib, d = _lib.load(), ops.dt(dtype)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    m, k, n, pad = 131, 45, 77, 64
    x, w, dz = randn(m, k, dtype=dtype).cuda(), randn(n, k, seed=1, dtype=dtype).cuda(), randn(m, n, seed=2, dtype=dtype).cuda()

    def guarded(count, t):
        buf = torch.full((count + 2 * pad,), 7, dtype=t, device="cuda")
        return buf, buf[pad:pad + count]

    def intact(buf):
        return bool((buf[:pad] == 7).all()) and bool((buf[-pad:] == 7).all())

    bufs = []
    y, yv = guarded(m * n, dtype); pre, prev = guarded(m * n, dtype)
    assert lib.simhand_linear_fwd(p(x), p(w), None, 2, None, p(yv), p(prev), m, k, n, d, None, 0, st) == 0
    dx, dxv = guarded(m * k, dtype)
    ws = torch.empty(lib.simhand_linear_dgrad_workspace_bytes(m, k, n, d, 0), dtype=torch.uint8, device="cuda")
    assert lib.simhand_linear_dgrad(p(dz), p(w), p(dxv), m, k, n, d, p(ws), ws.numel(), st) == 0
    dw, dwv = guarded(n * k, torch.float32)
    ws2 = torch.empty(lib.simhand_linear_wgrad_workspace_bytes(m, k, n, d) + 16, dtype=torch.uint8, device="cuda")
    assert lib.simhand_linear_wgrad(p(dz), p(x), None, None, p(dwv), m, k, n, d, p(ws2), ws2.numel(), st) == 0
    codes, cv = guarded(m * k, torch.uint8); exps, ev = guarded(m * 2, torch.uint8)
    assert lib.simhand_act8_pack(p(x), p(cv), p(ev), m, k, d, st) == 0
    back, bv = guarded(m * k, dtype)
    assert lib.simhand_act8_unpack(p(cv), p(ev), p(bv), m, k, d, st) == 0
    gamma, beta = torch.ones(k, device="cuda"), torch.zeros(k, device="cuda")
    ln, lv = guarded(m * k, dtype); mean, mv = guarded(m, torch.float32); rstd, rv = guarded(m, torch.float32)
    assert lib.simhand_layer_norm_fwd(p(x), p(gamma), p(beta), 1e-5, 1, p(lv), p(mv), p(rv), m, k, d, st) == 0
    ldx, ldv = guarded(m * k, dtype); gb, gv = guarded(2 * k, torch.float32)
    ws3 = torch.empty(lib.simhand_layer_norm_bwd_workspace_bytes(m, k, d), dtype=torch.uint8, device="cuda")
    assert lib.simhand_layer_norm_bwd(p(x), p(x), None, None, p(gamma), p(beta), p(mv), p(rv), 1, p(ldv), p(gv), m, k, d, p(ws3), ws3.numel(), st) == 0
    az, azv = guarded(m * n, dtype); db, dbv = guarded(n, torch.float32)
    ws4 = torch.empty(lib.simhand_linear_act_bwd_workspace_bytes(m, n, d), dtype=torch.uint8, device="cuda")
    assert lib.simhand_linear_act_bwd(p(dz), p(prev), 3, p(azv), p(dbv), m, n, d, p(ws4), ws4.numel(), st) == 0
    torch.cuda.synchronize()
    for name, b in dict(y=y, pre=pre, dx=dx, dw=dw, codes=codes, exps=exps, back=back, ln=ln, mean=mean, rstd=rstd, ldx=ldx, gb=gb, az=az, db=db).items():
        assert intact(b), name


def test_refusals_on_the_device():
    from simhand_amd import _lib, ops

    E = _lib.SimhandHipError
    x = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(6, 8, device="cuda")
    g = torch.ones(8, device="cuda")
    bad = [lambda: ops.linear_fwd(x.t(), w.t()), lambda: ops.linear_fwd(x, w[:, :4].contiguous()), lambda: ops.linear_fwd(x, w.bfloat16()), lambda: ops.linear_fwd(x, w, act="tanh"),
           lambda: ops.linear_fwd(x, w, bias=torch.zeros(5, device="cuda")), lambda: ops.linear_fwd(x, w, bias=torch.zeros(6)), lambda: ops.linear_fwd(x, w, residual=x),
           lambda: ops.linear_fwd(x.double(), w.double()), lambda: ops.linear_fwd(x.half(), w.half()), lambda: ops.linear_act_bwd(x, None, "gelu"),
           lambda: ops.linear_act_bwd(x, w, "gelu"), lambda: ops.linear_bwd(x, x, w), lambda: ops.layer_norm_fwd(x, g[:4], g), lambda: ops.layer_norm_fwd(x, g, g.double()),
           lambda: ops.layer_norm_fwd(x, g, g, eps=-1.0), lambda: ops.layer_norm_bwd(x, x, g, g, torch.zeros(3, device="cuda"), torch.zeros(4, device="cuda")),
           lambda: ops.layer_norm_fwd(torch.zeros(1, 20000, device="cuda"), torch.ones(20000, device="cuda"), torch.ones(20000, device="cuda")),
           lambda: ops.act8_pack(torch.zeros(4, 0, device="cuda")), lambda: ops.act8_pack(x.int()), lambda: ops.act8_pack(x.t()),
           lambda: ops.Act8(torch.zeros(4, 40, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), torch.float32),
           lambda: ops.linear_bwd(torch.zeros(4, 6, device="cuda").bfloat16(), ops.act8_pack(x), w.bfloat16())]
    for i, f in enumerate(bad):
        with pytest.raises(E):
            f()
            pytest.fail(f"case {i} was not refused")


# ------------------------------------------------------------------ sizes that 32 bits do not count
def whole_numbers(*shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-2, 3, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype)  # their products sum exactly in fp32


def spots(rows, cols):
    """first, last, and where the element and the byte offset pass 2^31 and 2^32"""
    return [slice(0, 70)] + [slice(max(0, b // cols - 40), min(rows, b // cols + 40)) for b in (1 << 30, 1 << 31) if b // cols < rows] + [slice(rows - 70, rows)]


@pytest.fixture
def huge():
    torch.cuda.empty_cache()
    yield 4300003, 512  # 2.2e9 values
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols", [512, 509])
def test_offsets_past_32_bits_rowwise(dtype, huge, cols):
    from simhand_amd import ops

    rows = huge[0] * huge[1] // cols if dtype != torch.float32 else (1 << 30) // cols + 9999  # (fp32: past 2^32 bytes)
    x = torch.empty(rows, cols, dtype=dtype, device="cuda").normal_()
    dy = torch.empty_like(x).normal_()
    dy[:-300] = 0  # the column sums are the last rows'
    gamma, beta = randn(cols, seed=1).cuda(), randn(cols, seed=2).cuda()
    y, mean, rstd = ops.layer_norm_fwd(x, gamma, beta)
    dx, dg, db = ops.layer_norm_bwd(dy, x, gamma, beta, mean, rstd)
    c = ops.act8_pack(x)
    back = ops.act8_unpack(c)
    dz, dbias = ops.linear_act_bwd(dy, x, "gelu")
    for s in spots(rows, cols):
        ys, ms, rs = ops.layer_norm_fwd(x[s], gamma, beta)
        assert torch.equal(y[s], ys) and torch.equal(mean[s], ms) and torch.equal(rstd[s], rs), s
        assert torch.equal(dx[s], ops.layer_norm_bwd(dy[s].contiguous(), x[s].contiguous(), gamma, beta, ms, rs)[0]), s
        cs = ops.act8_pack(x[s])
        assert torch.equal(c.codes[s], cs.codes) and torch.equal(c.exps[s], cs.exps) and torch.equal(back[s], ops.act8_unpack(cs)), s
        assert torch.equal(dz[s], ops.linear_act_bwd(dy[s], x[s], "gelu")[0]), s
    t = slice(rows - 300, rows)
    h = (x[t].double() - mean[t, None].double()) * rstd[t, None].double()
    d = dy[t].double()
    for got, want, mag in ((dg, (d * h).sum(0), (d * h).abs().sum(0)), (db, d.sum(0), d.abs().sum(0))):
        assert bool(((got.double() - want).abs() <= 320 * U * mag + U * want.abs()).all())  # (terms off by 4 U each, 300 of them added)


@pytest.mark.parametrize("k,n", [(512, 64), (64, 512), (509, 200), (61, 520), (64, 76)])
def test_offsets_past_32_bits_linear(dtype, huge, k, n):
    from simhand_amd import ops

    rows = huge[0] * huge[1] // max(k, n) if dtype != torch.float32 else (1 << 30) // max(k, n) + 9999
    x, w = whole_numbers(rows, k, dtype=dtype), whole_numbers(n, k, dtype=dtype, seed=1)
    res = whole_numbers(rows, n, dtype=dtype, seed=2)
    y, yr = ops.linear_fwd(x, w), ops.linear_fwd(x, w, act="relu", residual=res)
    dx = ops.linear_bwd(res, x[:, :k], w)[0]
    tail = torch.zeros_like(res)
    tail[-300:] = res[-300:]
    dw = ops.linear_wgrad(tail, x)
    assert torch.equal(dw, tail[-300:].float().t().contiguous() @ x[-300:].float())
    for s in spots(rows, max(k, n)):
        z = x[s].float() @ w.float().t().contiguous()
        assert torch.equal(y[s], z.to(dtype)), s
        assert torch.equal(yr[s], (z.clamp(min=0) + res[s].float()).to(dtype)), s
        assert torch.equal(dx[s], (res[s].float() @ w.float()).to(dtype)), s


def test_more_threads_than_32_bits_count():
    """A launch holds fewer than 2^32 threads: calls over more rows go in several."""
    from simhand_amd import ops

    torch.cuda.empty_cache()
    b = torch.bfloat16
    rows, edge = (1 << 26) + 70, 1 << 25
    x = torch.empty(rows, 129, dtype=b, device="cuda").normal_()
    gamma, beta = randn(129, seed=1).cuda(), randn(129, seed=2).cuda()
    y, mean, rstd = ops.layer_norm_fwd(x, gamma, beta)
    for s in (slice(0, 70), slice(edge - 70, edge + 70), slice(2 * edge - 70, rows)):
        ys, ms, rs = ops.layer_norm_fwd(x[s], gamma, beta)
        assert torch.equal(y[s], ys) and torch.equal(mean[s], ms) and torch.equal(rstd[s], rs), s
    del x, y, mean, rstd
    torch.cuda.empty_cache()
    edge = 1 << 29
    rows = edge + 70
    for k, n in ((2, 1), (3, 2), (8, 8)):  # the ragged tiles, and the LDS-DMA ones (both directions)
        x, w = whole_numbers(rows, k, dtype=b), whole_numbers(n, k, dtype=b, seed=1)
        y = ops.linear_fwd(x, w)
        dx = ops.linear_bwd(y, x, w)[0] if n > 1 else None
        for s in (slice(0, 70), slice(edge - 70, rows)):
            assert torch.equal(y[s], (x[s].float() @ w.float().t().contiguous()).to(b)), (k, n, s)
            if dx is not None:
                assert torch.equal(dx[s], (y[s].float() @ w.float()).to(b)), (k, n, s)
        del x, y, dx
        torch.cuda.empty_cache()


@pytest.mark.parametrize("m,k,n", [(40000, 333, 777), (70000, 512, 256), (50000, 256, 512)])
def test_captured_many_rows(dtype, m, k, n):
    """The kernels for many rows in a graph, replayed with new inputs between eager work on the same operands."""
    from simhand_amd import ops

    x, w, r = (randn(*s, seed=i, dtype=dtype).cuda() for i, s in enumerate(((m, k), (n, k), (m, n))))

    def calls():
        y, pre = ops.linear_fwd(x, w, act="gelu", residual=r, want_pre=True)
        dz, db = ops.linear_act_bwd(y, pre, "gelu")
        dx, dw = ops.linear_bwd(dz, ops.act8_pack(x), w)
        return y, pre, dz, db, dx, dw

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for s in range(3):
        x.copy_(randn(m, k, seed=60 + s, dtype=dtype))
        eager = calls()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), s


@pytest.mark.parametrize("m,k,n", [(5, 136, 128), (70, 33, 40), (300, 77, 130), (5001, 1000, 333), (33333, 640, 192), (40001, 333, 777), (66001, 130, 128), (49152, 256, 256),
                                   (20000, 505, 300), (70000, 512, 256)])
def test_linear_bad_values_stay_where_they_belong(dtype, m, k, n):
    """Inf and NaN of one row (column) reach that row (column) of the result and nothing beside it: ragged ends and rows past the end are kept out, not multiplied by zero."""
    from simhand_amd import ops

    x, w, r = (randn(*s, seed=i, scale=0.1, dtype=dtype).cuda() for i, s in enumerate(((m, k), (n, k), (m, n))))
    bad = sorted({1, m // 2, m - 1})
    xb = x.clone()
    xb[bad, k - 1] = torch.tensor([math.inf, math.nan, -math.inf], device="cuda")[:len(bad)].to(dtype)
    xb[bad[0], 0] = math.nan
    for res in (None, r):
        y, yb = ops.linear_fwd(x, w, residual=res), ops.linear_fwd(xb, w, residual=res)
        ok = torch.ones(m, dtype=torch.bool, device="cuda")
        ok[bad] = False
        assert torch.equal(y[ok], yb[ok]) and not bool(torch.isfinite(yb[~ok]).any())
    rb = r.clone()
    rb[bad, n - 1] = math.nan
    dx, dxb = ops.linear_bwd(r, x, w)[0], ops.linear_bwd(rb, x, w)[0]
    assert torch.equal(dx[ok], dxb[ok]) and not bool(torch.isfinite(dxb[~ok]).any())
    for pack in (False, True):
        keep = ops.act8_pack if pack else (lambda t: t)
        dw, dwx, dwz = ops.linear_wgrad(r, keep(x)), ops.linear_wgrad(r, keep(xb)), ops.linear_wgrad(rb, keep(x))
        cols = torch.ones(k, dtype=torch.bool, device="cuda")
        cols[k - 1] = cols[0] = False
        if pack:  # (a block's scale is that of its finite values: the neighbours keep their codes unless the bad value was the largest)
            cols[(k - 1) // 32 * 32:] = False
            cols[:32] = False
        assert torch.equal(dw[:, cols], dwx[:, cols]) and not bool(torch.isfinite(dwx[:, k - 1]).any())
        assert torch.equal(dw[:n - 1], dwz[:n - 1]) and not bool(torch.isfinite(dwz[n - 1]).any())


@pytest.mark.parametrize("m,k,n", [(40001, 333, 777), (66001, 130, 128), (33333, 640, 192), (20001, 505, 300), (9001, 777, 333), (49157, 200, 328), (70001, 512, 256), (7, 33, 5)])
def test_nothing_is_written_beside_outputs_and_workspaces(dtype, m, k, n):
    """As above for the kernels for many rows, with workspaces of exactly the bytes that were asked for."""
    from simhand_amd import _lib, ops

    lib, d, pad = _lib.load(), ops.dt(dtype), 256
    st = torch.cuda.current_stream().cuda_stream
    x, w, dz = randn(m, k, dtype=dtype).cuda(), randn(n, k, seed=1, dtype=dtype).cuda(), randn(m, n, seed=2, dtype=dtype).cuda()
    c = ops.act8_pack(x)
    bufs = []

    def guarded(count, t):
        buf = torch.full((count + 2 * pad,), 7, dtype=t, device="cuda")
        bufs.append(buf)
        return buf[pad:pad + count]

    nf = lib.simhand_linear_fwd_workspace_bytes(m, k, n, d, 1)
    nd, nw = lib.simhand_linear_dgrad_workspace_bytes(m, k, n, d, 1), lib.simhand_linear_wgrad_workspace_bytes(m, k, n, d)
    for res in (0, dz.data_ptr()):
        y, pre, ws = guarded(m * n, dtype), guarded(m * n, dtype), guarded(nf, torch.uint8)
        assert lib.simhand_linear_fwd(x.data_ptr(), w.data_ptr(), 0, 2, res, y.data_ptr(), pre.data_ptr(), m, k, n, d, ws.data_ptr(), nf, st) == 0
    dx, ws = guarded(m * k, dtype), guarded(nd, torch.uint8)
    assert lib.simhand_linear_dgrad(dz.data_ptr(), w.data_ptr(), dx.data_ptr(), m, k, n, d, ws.data_ptr(), nd, st) == 0
    for px, pc, pe in ((x.data_ptr(), 0, 0), (0, c.codes.data_ptr(), c.exps.data_ptr())):
        dw, ws = guarded(n * k, torch.float32), guarded(nw, torch.uint8)
        assert lib.simhand_linear_wgrad(dz.data_ptr(), px, pc, pe, dw.data_ptr(), m, k, n, d, ws.data_ptr(), nw, st) == 0
    torch.cuda.synchronize()
    assert all(bool((b[:pad] == 7).all()) and bool((b[-pad:] == 7).all()) for b in bufs)
