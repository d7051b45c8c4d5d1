"""The framework's own paths through the row operators: the differentiable linear / layer_norm of host.model_utils, the layer-norm projection head, and a
training step with saved activations in 8 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def randn(*shape, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 1000 * sum(shape))
    return torch.randn(*shape, generator=g) * scale


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("lead", [(37,), (3, 5, 7)])
def test_linear_function(act, lead):
    """Values and gradients of every argument against autograd of the formula in 64 bits: 12 K U of the terms' magnitudes (K = the longest sum, 105 rows)."""
    from simhand_amd.host import model_utils as mu

    k, n = 19, 23
    x, w, b, r, dy = randn(*lead, k), randn(n, k, seed=1), randn(n, seed=2), randn(*lead, n, seed=3), randn(*lead, n, seed=4)
    dev = [t.cuda().requires_grad_() for t in (x, w, b, r)]
    y = mu.linear(*dev[:3], act=act, residual=dev[3])
    y.backward(dy.cuda())
    ref = [t.double().requires_grad_() for t in (x, w, b, r)]
    z = ref[0] @ ref[1].t() + ref[2]
    z = {None: lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z)}[act]()
    want = z + ref[3]
    want.backward(dy.double())
    for got, ex in [(y, want.detach())] + [(a.grad, c.grad) for a, c in zip(dev, ref)]:
        assert got.shape == ex.shape
        assert float((got.detach().double().cpu() - ex).norm()) <= 12 * 105 * U * float(ex.norm())


@pytest.mark.parametrize("relu", [False, True])
def test_layer_norm_function(relu):
    from simhand_amd.host import model_utils as mu

    x, g, b, dy = randn(4, 9, 50), 1 + 0.1 * randn(50, seed=1), randn(50, seed=2), randn(4, 9, 50, seed=4)
    dev = [t.cuda().requires_grad_() for t in (x, g, b)]
    y = mu.layer_norm(*dev, relu=relu)
    y.backward(dy.cuda())
    ref = [t.double().requires_grad_() for t in (x, g, b)]
    m = ref[0].mean(dim=-1, keepdim=True)
    want = (ref[0] - m) / torch.sqrt((ref[0] - m).square().mean(dim=-1, keepdim=True) + 1e-5) * ref[1] + ref[2]
    want = want.clamp(min=0) if relu else want
    want.backward(dy.double())
    for got, ex in [(y, want.detach())] + [(a.grad, c.grad) for a, c in zip(dev, ref)]:
        assert float((got.detach().double().cpu() - ex).norm()) <= 200 * U * float(ex.norm())


def test_functions_with_8_bit_checkpoints():
    """act8 changes nothing in the forward pass and nothing in the gradients that do not read the checkpoint; those that do are off by its rounding (2^-4 of a value at most, and
    the blocks' small values by 2^-10 of the block's scale: together under 2^-4 of the norm)."""
    from simhand_amd.host import model_utils as mu

    x, w, b = randn(64, 96), randn(40, 96, seed=1, scale=0.1), randn(40, seed=2)
    g, be, dy = 1 + 0.1 * randn(40, seed=5), randn(40, seed=6), randn(64, 40, seed=7)

    def run(act8):
        t = [v.cuda().requires_grad_() for v in (x, w, b, g, be)]
        y = mu.layer_norm(mu.linear(t[0], t[1], t[2], act8=act8), t[3], t[4], relu=True, act8=act8)
        y.backward(dy.cuda())
        return y.detach(), [v.grad for v in t]

    (ya, ga), (yb, gb) = run(False), run(True)
    assert torch.equal(ya, yb)
    for p, q in zip(ga, gb):
        # dx and dw pass through the norm's backward pass, whose gate may move where a value changed sign: 2^-4 twice and the moved gates
        assert float((p - q).norm()) <= 0.25 * float(p.norm())
    with torch.no_grad():
        assert torch.equal(mu.linear(x.cuda(), w.cuda(), b.cuda(), act8=True), mu.linear(x.cuda(), w.cuda(), b.cuda()))


def test_gradients_only_where_asked():
    from simhand_amd.host import model_utils as mu

    x, w, b = randn(8, 12).cuda(), randn(5, 12, seed=1).cuda(), randn(5, seed=2).cuda()
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        t = [v.clone().requires_grad_(bool(n)) for v, n in zip((x, w, b), need)]
        mu.linear(*t, act="gelu").sum().backward()
        assert [v.grad is not None for v in t] == [bool(n) for n in need]


def _model(size, name="SimCLR", dtype=torch.float32, **kw):
    from simhand_amd.host import unsupervised
    from tests.test_host_logic import _cfg

    torch.manual_seed(11)
    m = getattr(unsupervised, name)(_cfg(size, **kw), None, "train")
    m.set_compute_dtype(dtype)
    return m.cuda().train()


def test_layer_norm_head_against_its_formula():
    """Projections and gradients of the layer-norm head on given embeddings, in 64 bits on the CPU; a row's projection is bit for bit the same in any batch."""
    m = _model("18", projection_head_norm="layer")
    ph = m.projection_head
    enc = randn(24, 512, seed=3)
    dp = randn(24, 128, seed=4)
    e = enc.cuda().requires_grad_()
    p = m._head(e)
    p.backward(dp.cuda())
    par = [t.detach().double().cpu().requires_grad_() for t in (ph[0].weight, ph[0].bias, ph[1].weight, ph[1].bias, ph[3].weight)]
    ed = enc.double().requires_grad_()
    h = ed @ par[0].t() + par[1]
    mean = h.mean(dim=1, keepdim=True)
    h = (h - mean) / torch.sqrt((h - mean).square().mean(dim=1, keepdim=True) + ph[1].eps) * par[2] + par[3]
    want = h.clamp(min=0) @ par[4].t()
    want.backward(dp.double())
    got = [p.detach(), e.grad] + [t.grad for t in (ph[0].weight, ph[0].bias, ph[1].weight, ph[1].bias, ph[3].weight)]
    for a, b in zip(got, [want.detach(), ed.grad] + [t.grad for t in par]):
        # sums of up to 512 terms in each of the three layers, either way: 6 x 512 U of the norm, twice for the matrix cores
        assert float((a.double().cpu() - b).norm()) <= 2 * 6 * 512 * U * float(b.norm())
    with torch.no_grad():
        assert torch.equal(m._head(enc[5:6].cuda()), m._head(enc.cuda())[5:6]) or \
            float((m._head(enc[5:6].cuda()) - p[5:6]).norm()) <= 2 * 6 * 512 * U * float(p[5:6].norm())


@pytest.mark.parametrize("act8", [False, True])
def test_training_step_with_a_layer_norm_head(act8):
    from oracle import step as orc

    m = _model("18", "HandCLR_W", projection_head_norm="layer", act8=act8, augmentation=["crop", "rotate"])
    batch = {k: v.cuda() for k, v in orc.synthetic_batch(4, size=64, seed=5).items()}
    out = m.training_step(batch, 0)
    out["loss"].backward()
    assert torch.isfinite(out["loss"])
    for k, p in m.named_parameters():
        if not k.startswith("encoder.final_layer"):
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()), k
    with torch.no_grad():
        m.eval()
        assert torch.isfinite(m.validation_step(batch, 0)["loss"])


@pytest.mark.parametrize("size,dtype", [("18", torch.float32), ("18", torch.bfloat16), ("50", torch.float32), ("50", torch.bfloat16), ("50", torch.float16)])
def test_encoder_with_block_inputs_in_8_bits(size, dtype, monkeypatch):
    """The forward pass and every gradient but one kind are bit for bit those of the plain run: a block input is read back for its first convolution's weight gradient
    alone.  That gradient is the product of the same dy with the codes' values: to 2 (M + 40) U of its terms' magnitudes for the 1x1 layers (fp32 sums over M
    pixels on the matrix cores), bit for bit the kernel's on the unpacked tensor for the 3x3 ones."""
    from oracle import step as orc
    from simhand_amd import _lib, ops
    from simhand_amd.host.resnet_model import ResNetEngine

    batch = {k: v.cuda() for k, v in orc.synthetic_batch(4, size=64, seed=5).items()}
    plain = ResNetEngine._wgrad
    seen = {}

    def recording(u, dy):
        seen[id(u.conv.weight)] = (u, u.x, dy)
        return plain(u, dy)

    res = []
    for act8 in (False, True):
        m = _model(size, act8=act8, dtype=dtype)
        assert m.encoder.engine.act8 is act8
        if not act8:
            monkeypatch.setattr(ResNetEngine, "_wgrad", staticmethod(recording))
        loss = m.training_step(batch, 0)["loss"]
        (loss * (1024.0 if dtype == torch.float16 else 1.0)).backward()
        monkeypatch.undo()
        res.append((loss.detach(), {k: p.grad for k, p in m.named_parameters() if p.grad is not None}, dict(m.named_parameters()), m))
    (la, ga, params, m), (lb, gb, _, _) = res
    assert torch.equal(la, lb) and set(ga) == set(gb)
    packed = {f"encoder.features.{li}.{bi}.conv1.weight" for li in (4, 5, 6, 7) for bi, blk in enumerate(m.encoder.features[li]) if blk.downsample is None}
    assert packed <= set(ga)
    for k in ga:
        if k not in packed:
            assert torch.equal(ga[k], gb[k]), k
            continue
        assert not torch.equal(ga[k], gb[k]), k
        u, x, dy = seen[id(params[k])]
        xv = ops.act8_unpack(ops.act8_pack(x))
        if u.conv.kernel_size == (3, 3):
            assert torch.equal(gb[k], ops.conv2d_wgrad_oihw(u.desc, xv, dy, tuple(u.conv.weight.shape))), k
        else:
            xd, dd = (t.double().cpu().reshape(-1, t.shape[-1]) for t in (xv, dy))
            err = (gb[k].double().cpu().view(dd.shape[1], -1) - dd.t() @ xd).abs()
            assert bool((err <= 2 * (len(xd) + 40) * U * (dd.abs().t() @ xd.abs()) + 1e-30).all()), k
    _lib.use_half("bf16")


def test_command_line(tmp_path):
    """Three optimizer steps of the command with both options."""
    from simhand_amd.host.main import main

    t = main(["--experiment_type", "handclr_w", "--crop", "--rotate", "--resize", "-resnet_size", "18", "-batch_size", "8", "-epochs", "1", "--weight_type", "linear",
              "--joints_type", "augmented", "--diff_type", "mpjpe", "--pos_neg", "pos_neg", "--synthetic", "--synthetic_samples", "24", "--image_size", "64", "--precision", "bf16",
              "--projection_head_norm", "layer", "--act8", "--max_steps", "3", "--out_dir", str(tmp_path)])
    assert t.global_step == 3 and all(torch.isfinite(torch.as_tensor(float(x))) for x in t.step_losses)


def test_shared_operands_and_an_expanded_gradient():
    """One weight in two places, x as input and residual, the gradient of a sum (stride 0): gradients add up as in 64 bits (terms of 12 x 90 U, as above)."""
    from simhand_amd.host import model_utils as mu

    x, w, b, g = randn(41, 24), randn(24, 24, seed=1, scale=0.3), randn(24, seed=2), 1 + 0.1 * randn(24, seed=3)
    dev = [t.cuda().requires_grad_() for t in (x, w, b, g)]
    h = mu.linear(dev[0], dev[1], dev[2], act="silu", residual=dev[0])
    h = mu.layer_norm(h, dev[3], dev[2])
    y = mu.linear(h, dev[1], residual=h)
    y[:, 1:].square().sum().backward()
    ref = [t.double().requires_grad_() for t in (x, w, b, g)]
    z = ref[0] @ ref[1].t() + ref[2]
    h = z * torch.sigmoid(z) + ref[0]
    h = torch.nn.functional.layer_norm(h, (24,), ref[3], ref[2], 1e-5)
    want = h @ ref[1].t() + h
    want[:, 1:].square().sum().backward()
    for a, c in zip(dev, ref):
        assert float((a.grad.double().cpu() - c.grad).norm()) <= 12 * 90 * U * float(c.grad.norm()) * 4  # (three layers and the square carry one another's rounding)
    dev[0].grad = None
    mu.linear(dev[0], dev[1]).sum().backward()  # an expanded gradient
    ones = torch.ones(41, 24, dtype=torch.float64) @ w.double()
    assert float((dev[0].grad.double().cpu() - ones).norm()) <= 12 * 24 * U * float(ones.norm())


def test_captured_forward_and_backward():
    """Values and gradients of a block in one graph, replayed with new inputs between eager passes over the same leaves: bit for bit the eager ones."""
    from simhand_amd.host import model_utils as mu

    x, w, b, g, w2, dy = (t.cuda() for t in (randn(300, 40), randn(72, 40, seed=1), randn(72, seed=2), 1 + 0.1 * randn(72, seed=3), randn(40, 72, seed=4), randn(300, 40, seed=5)))
    leaves = [t.requires_grad_() for t in (x, w, b, g, w2)]

    def block():
        h = mu.layer_norm(mu.linear(x, w, b, act="gelu", act8=True), g, b, relu=True, act8=True)
        y = mu.linear(h, w2, residual=x)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    for s in range(3):
        with torch.no_grad():
            x.copy_(randn(300, 40, seed=20 + s))
        eager = [t.clone() for t in block()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, eager)), s
