"""Cases of the layer-norm, linear and 8-bit activation operators of ``simhand_amd.ops``, with their plain forms.

``run`` computes an operator in elementary torch operations in 32 bits where ``own`` is false, and through the library where it is true.
Sizes: the projection head's (512 / 2048 columns; a row per image), the wide 1x1 layers of the encoder with pixels as rows
(2048 images of 7 x 7 = 100 352 rows, of 14 x 14 = 401 408), and ragged ones.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-5


def _case(name, op, rows, cin, cout=0, dtype="bf16", **more):
    c = {"op": op, "rows": rows, "cin": cin, "cout": cout, "dtype": dtype, "act": "none", "bias": False, "residual": False, "pre": False, "relu": False,
         "act8": False, "dx": True}
    c.update(more)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the norm of a projection head that sees one small batch: latency
        _case("ln fwd fp32 256x512 relu", "ln_fwd", 256, 512, dtype="fp32", relu=True),
        # every 7 x 7 pixel of 2048 images, 2048 channels
        _case("ln fwd bf16 100352x2048", "ln_fwd", 100352, 2048),
        # the head's norm at the benchmark's batch (2 x 1024 images)
        _case("ln bwd fp32 2048x512 relu", "ln_bwd", 2048, 512, dtype="fp32", relu=True),
        # a width that no vector divides, from an 8-bit checkpoint
        _case("ln bwd fp16 33001x777 act8", "ln_bwd", 33001, 777, dtype="fp16", act8=True),
        # embedding of a handful of images through the head's first layer: latency
        _case("linear fwd fp32 8x2048-512", "linear_fwd", 8, 2048, 512, "fp32", act="relu", bias=True),
        # expansion of the last stage with the block's residual sum
        _case("linear fwd bf16 100352x512-2048", "linear_fwd", 100352, 512, 2048, act="relu", bias=True, residual=True),
        # training forward, ragged: the pre-activation is kept
        _case("linear fwd fp16 5001x1000-333", "linear_fwd", 5001, 1000, 333, "fp16", act="gelu", bias=True, pre=True),
        # gradient through the activation, with the bias gradient's reduction
        _case("act bwd bf16 100352x2048 gelu", "act_bwd", 100352, 2048, act="gelu"),
        # gradients of the head's first layer at the benchmark's batch
        _case("linear bwd fp32 2048x2048-512", "linear_bwd", 2048, 2048, 512, "fp32"),
        # gradients of the third stage's reduction over all pixels
        _case("linear bwd bf16 401408x1024-256", "linear_bwd", 401408, 1024, 256),
        # the same layer's weight gradient from the 8-bit checkpoint of its input
        _case("linear bwd bf16 401408x1024 act8", "linear_bwd", 401408, 1024, 256, act8=True, dx=False),
        # that checkpoint: written in the forward pass, read back
        _case("act8 bf16 401408x1024", "act8", 401408, 1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    n = _log(rng, lo, hi)
    return max(lo, min(hi, n if rng.random() < 0.5 else (n + 32) // 64 * 64))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "linear_fwd", "linear_fwd", "act_bwd", "linear_bwd", "linear_bwd", "act8"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    cin, cout = _size(rng, 32, 2048), _size(rng, 32, 2048)
    top = 401408
    if op == "linear_bwd":
        top = min(top, 100_000_000_000 // (cin * cout))
    elif op == "linear_fwd":
        top = min(top, 100_000_000_000 // (cin * cout))
    else:
        top = min(top, 200_000_000 // cin)
    rows = _log(rng, 4, max(4, top))
    c = _case("", op, rows, cin, cout if op.startswith("linear") else 0, dtype)
    if op in ("linear_fwd", "act_bwd"):
        c["act"] = rng.choice(["none", "relu", "gelu", "silu"])
    if op == "linear_fwd":
        c["bias"], c["residual"], c["pre"] = rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.5
    if op in ("ln_fwd", "ln_bwd"):
        c["relu"] = rng.random() < 0.5
    if op in ("ln_bwd", "linear_bwd"):
        c["act8"] = rng.random() < 0.4
    if op == "linear_bwd" and c["act8"]:
        c["dx"] = rng.random() < 0.5
    return c


def _pow2(e):
    """2 to the whole power e, -126 <= e <= 127, by its bits: exact."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(x):
    """8-bit checkpoint of x: e4m3 codes and the power of two of every 32 columns."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float32, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, 32)
    m, e = torch.frexp(v.abs().amax(dim=2))  # m in [0.5, 1)
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp_(min=-126)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    v = v * _pow2(-e).unsqueeze(2)
    # round to nearest even at 3 bits behind the leading one, or at the smallest step 2^-9
    _, p = torch.frexp(v)
    p = (p - 4).clamp_(min=-9)
    v = torch.round(v * _pow2(-p)) * _pow2(p)
    codes = v.to(torch.float8_e4m3fn).view(torch.uint8).view(rows, blocks * 32)[:, :cols].contiguous()
    return codes, (e + 127).to(torch.uint8).contiguous()


def _values(codes, exps):
    """What the codes stand for, in 32 bits."""
    cols = codes.shape[1]
    scale = _pow2(exps.to(torch.int32) - 127)
    return codes.view(torch.float8_e4m3fn).to(torch.float32) * scale.repeat_interleave(32, dim=1)[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    t, rows, cin, cout, op = _TYPES[case["dtype"]], case["rows"], case["cin"], case["cout"], case["op"]

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = {"case": dict(case), "type": t}
    if op in ("ln_fwd", "ln_bwd"):
        s["x"] = (randn(rows, cin) + 0.5 * randn(1, cin)).to(t)
        s["gamma"], s["beta"] = 1.0 + 0.1 * randn(cin), 0.1 * randn(cin)
    if op == "ln_bwd":
        s["dy"] = randn(rows, cin, dtype=t)
        if case["act8"]:
            s["codes"], s["exps"] = _codes(s["x"])
            v = _values(s["codes"], s["exps"]).double()
        else:
            v = s["x"].double()
        s["mean"] = v.mean(dim=1)
        s["rstd"] = 1.0 / torch.sqrt((v - s["mean"].unsqueeze(1)).square().mean(dim=1) + _EPS)
        s["mean"], s["rstd"] = s["mean"].float(), s["rstd"].float()
        if case["act8"]:
            del s["x"]
    if op in ("linear_fwd", "linear_bwd"):
        s["x"] = torch.relu(randn(rows, cin)).to(t)  # activations
        s["w"] = randn(cout, cin, scale=math.sqrt(2.0 / cin), dtype=t)
    if op == "linear_fwd":
        s["bias"] = 0.1 * randn(cout) if case["bias"] else None
        s["residual"] = randn(rows, cout, dtype=t) if case["residual"] else None
    if op == "linear_bwd":
        s["dz"] = randn(rows, cout, dtype=t)
        if case["act8"]:
            s["codes"], s["exps"] = _codes(s["x"])
            del s["x"]
    if op == "act_bwd":
        s["dy"] = randn(rows, cin, dtype=t)
        s["pre"] = randn(rows, cin, dtype=t) if case["act"] != "none" else None
    if op == "act8":
        s["x"] = torch.relu(randn(rows, cin)).to(t)
    return s


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return z * 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    sg = 1.0 / (1.0 + torch.exp(-z))
    return sg * (1.0 + z * (1.0 - sg))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    c, t = s["case"], s["type"]
    op = c["op"]
    if op == "ln_fwd":
        x = s["x"].float()
        mean = x.mean(dim=1, keepdim=True)
        x = x - mean
        rstd = 1.0 / torch.sqrt(x.square().mean(dim=1, keepdim=True) + _EPS)
        y = x * rstd * s["gamma"] + s["beta"]
        if c["relu"]:
            y = _act(y, "relu")
        return {"y": y.to(t), "mean": mean.view(-1), "rstd": rstd.view(-1)}
    if op == "ln_bwd":
        x = _values(s["codes"], s["exps"]) if c["act8"] else s["x"].float()
        rstd = s["rstd"].unsqueeze(1)
        h = (x - s["mean"].unsqueeze(1)) * rstd
        u = s["dy"].float()
        if c["relu"]:
            u = u * (h * s["gamma"] + s["beta"] > 0)
        dgamma, dbeta = (u * h).sum(dim=0), u.sum(dim=0)
        u = u * s["gamma"]
        dx = rstd * (u - u.mean(dim=1, keepdim=True) - h * (u * h).mean(dim=1, keepdim=True))
        return {"dx": dx.to(t), "dgamma": dgamma, "dbeta": dbeta}
    if op == "linear_fwd":
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        y = _act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return {"y": y.to(t), "pre": z.to(t)} if c["pre"] else {"y": y.to(t)}
    if op == "act_bwd":
        dz = s["dy"].float()
        if s["pre"] is not None:
            dz = dz * _act_slope(s["pre"].float(), c["act"])
        return {"dz": dz.to(t), "db": dz.sum(dim=0)}
    if op == "linear_bwd":
        dz = s["dz"].float()
        x = _values(s["codes"], s["exps"]) if c["act8"] else s["x"].float()
        out = {"dw": dz.t() @ x}
        if c["dx"]:
            out["dx"] = (dz @ s["w"].float()).to(t)
        return out
    codes, exps = _codes(s["x"])
    return {"x": _values(codes, exps).to(t)}


def _run_own(s):
    from simhand_amd import _lib, ops

    c, t = s["case"], s["type"]
    op = c["op"]
    _lib.use_half("f16" if t is torch.float16 else "bf16")
    x = ops.Act8(s["codes"], s["exps"], t) if c["act8"] else s.get("x")
    if op == "ln_fwd":
        y, mean, rstd = ops.layer_norm_fwd(x, s["gamma"], s["beta"], _EPS, relu=c["relu"])
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "ln_bwd":
        dx, dgamma, dbeta = ops.layer_norm_bwd(s["dy"], x, s["gamma"], s["beta"], s["mean"], s["rstd"], relu=c["relu"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if op == "linear_fwd":
        out = ops.linear_fwd(x, s["w"], s["bias"], act=c["act"], residual=s["residual"], want_pre=c["pre"])
        return {"y": out[0], "pre": out[1]} if c["pre"] else {"y": out}
    if op == "act_bwd":
        dz, db = ops.linear_act_bwd(s["dy"], s["pre"], act=c["act"])
        return {"dz": dz, "db": db}
    if op == "linear_bwd":
        dx, dw = ops.linear_bwd(s["dz"], x, s["w"], need_dx=c["dx"])
        return {"dw": dw, "dx": dx} if c["dx"] else {"dw": dw}
    return {"x": ops.act8_unpack(ops.act8_pack(x))}


def work(case):
    m, k, n, b = case["rows"], case["cin"], case["cout"], _BYTES[case["dtype"]]
    x8 = m * k + m * -(-k // 32)
    x = x8 if case["act8"] else m * k * b
    op = case["op"]
    if op == "ln_fwd":
        return {"bytes": 2 * m * k * b + 8 * m + 8 * k, "flops": 8 * m * k}
    if op == "ln_bwd":
        return {"bytes": 2 * m * k * b + x + 8 * m + 16 * k, "flops": 16 * m * k}
    if op == "linear_fwd":
        outs = 1 + int(case["residual"]) + int(case["pre"])
        return {"bytes": b * (m * k + n * k + outs * m * n) + 4 * n * int(case["bias"]), "flops": 2 * m * n * k}
    if op == "act_bwd":
        return {"bytes": b * m * k * (3 if case["act"] != "none" else 2) + 4 * k, "flops": (20 if case["act"] in ("gelu", "silu") else 2) * m * k}
    if op == "linear_bwd":
        return {"bytes": b * m * n + x + 4 * n * k + (b * (n * k + m * k) if case["dx"] else 0), "flops": (4 if case["dx"] else 2) * m * n * k}
    return {"bytes": 2 * m * k * b + 2 * x8, "flops": 4 * m * k}


def exact(case, seed):
    """From the definitions in 64 bits: normalised rows by their moments, derivatives by the error function and the logistic function, 8-bit values by
    choosing the nearest of all that a block can hold."""
    s = prepare(case, seed)
    op, act = case["op"], case["act"]
    d = torch.float64
    power = torch.tensor([2.0 ** k for k in range(-160, 161)], dtype=d).cuda()  # power[k + 160] = 2^k; torch.pow need not be exact there
    if case["act8"]:
        grid = torch.arange(256, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).to(d)
        scale = power[s["exps"].int() + 33]
        cols = torch.arange(case["cin"], device="cuda") // 32
        x = grid[s["codes"].int()] * scale[:, cols]
    elif "x" in s:
        x = s["x"].to(d)
    if op in ("ln_fwd", "ln_bwd"):
        gamma, beta = s["gamma"].to(d), s["beta"].to(d)
    if op == "ln_fwd":
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        rstd = (var + _EPS).rsqrt()
        y = (x - mean) * rstd * gamma + beta
        return {"y": y.clamp(min=0) if case["relu"] else y, "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if op == "ln_bwd":
        # dx = J^T g of the normalisation with the saved statistics: the row's projections on (1, h) leave g
        rstd = s["rstd"].to(d)[:, None]
        h = (x - s["mean"].to(d)[:, None]) * rstd
        u = s["dy"].to(d)
        if case["relu"]:
            u = torch.where(h * gamma + beta > 0, u, torch.zeros((), dtype=d, device="cuda"))
        g = u * gamma
        n = case["cin"]
        dx = g.sub_(g.sum(dim=1, keepdim=True) / n).sub_(h * ((u * gamma * h).sum(dim=1, keepdim=True) / n)).mul_(rstd)
        return {"dx": dx, "dgamma": (h * u).sum(dim=0), "dbeta": u.sum(dim=0)}
    if op == "linear_fwd":
        z = torch.mm(x, s["w"].to(d).t())
        if s["bias"] is not None:
            z += s["bias"].to(d)
        y = {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z)}[act]()
        if s["residual"] is not None:
            y = y + s["residual"].to(d)
        return {"y": y, "pre": z} if case["pre"] else {"y": y}
    if op == "act_bwd":
        dy = s["dy"].to(d)
        if s["pre"] is None:
            return {"dz": dy, "db": dy.sum(dim=0)}
        z = s["pre"].to(d)
        if act == "relu":
            slope = torch.heaviside(z, torch.zeros((), dtype=d, device="cuda"))
        elif act == "gelu":
            slope = torch.special.ndtr(z) + z * torch.exp(z * z / -2) / math.sqrt(2 * math.pi)
        else:
            slope = torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
        dz = dy * slope
        return {"dz": dz, "db": dz.sum(dim=0)}
    if op == "linear_bwd":
        dz = s["dz"].to(d)
        out = {"dw": torch.mm(dz.t(), x)}
        if case["dx"]:
            out["dx"] = torch.mm(dz, s["w"].to(d))
        return out
    # 8-bit values: for every block the power of two that brings its largest magnitude to (224, 448], then the nearest value of the grid (ties to the even code)
    rows, cols = x.shape
    blocks = -(-cols // 32)
    pad = torch.zeros(rows, blocks * 32, dtype=d, device="cuda")
    pad[:, :cols] = x
    pad = pad.view(rows, blocks, 32)
    top = pad.abs().amax(dim=2, keepdim=True)
    e = torch.searchsorted(448.0 * power[34:], top.contiguous()) - 126  # the least e >= -126 with top <= 448 2^e
    scale = power[e + 160]
    out = torch.empty_like(pad)
    grid = torch.arange(127, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).to(d)  # 0 .. 448, ascending
    for lo in range(0, rows, 65536):  # in parts: the search's indices are eight bytes a value
        v = (pad[lo:lo + 65536] / scale[lo:lo + 65536])
        a = v.abs().contiguous()
        hi = torch.searchsorted(grid, a).clamp_(max=126)
        low = (hi - 1).clamp_(min=0)
        up, down = grid[hi] - a, a - grid[low]
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, low)
        out[lo:lo + 65536] = grid[pick] * torch.sign(v) * scale[lo:lo + 65536]
    return {"x": out.view(rows, blocks * 32)[:, :cols]}
