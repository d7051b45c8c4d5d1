"""CPU: the differentiable linear keeps and computes only what the gradients that were asked for read.  The operators are stood in for by their formulas; what is looked at is
which of them are called, and what autograd keeps."""
import pytest
import torch

from simhand_amd import ops


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def fwd(x, w, bias=None, act=None, residual=None, want_pre=False):
        seen.append("pre" if want_pre else "fwd")
        z = x @ w.t() + (0 if bias is None else bias)
        y = (z.clamp(min=0) if act == "relu" else z) + (0 if residual is None else residual)
        return (y, z) if want_pre else y

    def act_bwd(dy, pre=None, act=None):
        seen.append("act")
        dz = dy * (pre > 0) if act == "relu" else dy
        return dz, dz.sum(0)

    def bwd(dz, x, w, need_dx=True, need_dw=True):
        seen.extend(["dx"] * need_dx + ["dw"] * need_dw)
        return dz @ w if need_dx else None, dz.t() @ (x.codes.float() if isinstance(x, ops.Act8) else x) if need_dw else None

    def wgrad(dz, x):
        seen.append("dw")
        return dz.t() @ (x.codes.float() if isinstance(x, ops.Act8) else x)

    def pack(x):
        seen.append("pack")
        return ops.Act8(x.to(torch.uint8), torch.zeros(x.shape[0], (x.shape[1] + 31) // 32, dtype=torch.uint8), x.dtype)

    for name, f in dict(linear_fwd=fwd, linear_act_bwd=act_bwd, linear_bwd=bwd, linear_wgrad=wgrad, act8_pack=pack).items():
        monkeypatch.setattr(ops, name, f)
    return seen


@pytest.mark.parametrize("need", [(1, 1, 1, 1), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 1, 0), (0, 1, 1, 0), (0, 0, 0, 0)])
@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("act8", [False, True])
def test_only_what_is_asked_for(calls, need, act, act8):
    from simhand_amd.host import model_utils as mu

    shapes = ((6, 5), (4, 5), (4,), (6, 4))
    t = [torch.randn(*s, generator=torch.Generator().manual_seed(i)).requires_grad_(bool(n)) for i, (s, n) in enumerate(zip(shapes, need))]
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(tuple(v.shape)) or v, lambda v: v):
        y = mu.linear(*t[:3], act=act, residual=t[3], act8=act8)
    through = any(need[:3])
    assert calls == ["pre" if act and through else "fwd"] + ["pack"] * (act8 and need[1])
    want = ([(6, 5)] + [(6, 1)] * act8) * need[1] + [(4, 5)] * need[0] + [(6, 4)] * bool(act and through)
    assert sorted(kept) == sorted(want)
    if not any(need):
        return
    calls.clear()
    y.sum().backward()
    assert calls == ["act"] * bool(need[2] or (act and through)) + ["dx"] * need[0] + ["dw"] * need[1]
    z = t[0] @ t[1].t() + t[2]
    ref = torch.autograd.grad(((z.clamp(min=0) if act else z) + t[3]).sum(), [v for v, n in zip(t, need) if n])
    for v, n, i in zip(t, need, range(4)):
        assert (v.grad is not None) == bool(n)
        if n and not (act8 and i == 1):
            assert torch.allclose(v.grad, ref[sum(need[:i])], atol=1e-5)


def test_nothing_is_kept_without_gradients(calls):
    from simhand_amd.host import model_utils as mu

    x, w = torch.randn(6, 5, requires_grad=True), torch.randn(4, 5, requires_grad=True)
    with torch.no_grad():
        mu.linear(x, w, act="relu", act8=True)
    assert calls == ["fwd"]
