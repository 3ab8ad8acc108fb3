"""The measured calls of the channels-last operators: group norm with an activation, the gated feed-forward block over
the pixels of a map, and the moves between a convolution layer's NCHW maps and channels-last ones.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, where `own` is true, through
fastconv_b200.  A map of n images with h x w pixels and c channels is [n][h*w][c] when it is channels last."""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_context = None


def _ctx():
    """The program's one context: a stream and an arena for the plans' workspaces."""
    global _context
    if _context is None:
        import fastconv_b200 as fc
        _context = fc.Context(0, arena_bytes=10 << 30)
    return _context


# ---- cases --------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the last stage of a VGG-sized network, one image: nothing but latency
        {"name": "norm_one_14x14x512", "op": "norm", "train": False, "batch": 1, "h": 14, "w": 14, "channels": 512, "groups": 32,
         "wide": 512, "act": "silu", "dtype": "bf16"},
        # a map of odd extent that is a slice of a wider one (joined skip connections), ten channels to a group
        {"name": "norm_skip_37x53x320", "op": "norm", "train": False, "batch": 3, "h": 37, "w": 53, "channels": 320, "groups": 32,
         "wide": 480, "act": "gelu", "dtype": "fp16"},
        # a batch of 64 images between fp32 layers
        {"name": "norm_batch_28x28x512", "op": "norm", "train": False, "batch": 64, "h": 28, "w": 28, "channels": 512, "groups": 32,
         "wide": 512, "act": "relu", "dtype": "fp32"},
        # a training step through the norm at the largest map of the middle stages
        {"name": "norm_train_56x56x256", "op": "norm", "train": True, "batch": 64, "h": 56, "w": 56, "channels": 256, "groups": 32,
         "wide": 256, "act": "silu", "dtype": "bf16"},
        # a block asked for one pixel (one token): the weights are all there is to read
        {"name": "ff_one_1024", "op": "ff", "train": False, "rows": 1, "channels": 1024, "hidden": 4096, "act": "silu", "bias": False,
         "dtype": "bf16"},
        # one 14x14 image
        {"name": "ff_image_1024", "op": "ff", "train": False, "rows": 196, "channels": 1024, "hidden": 4096, "act": "gelu_tanh",
         "bias": True, "dtype": "fp16"},
        # 64 images of 28x28
        {"name": "ff_batch_512", "op": "ff", "train": False, "rows": 50176, "channels": 512, "hidden": 2048, "act": "silu",
         "bias": False, "dtype": "bf16"},
        # a training step on 64 images of 14x14
        {"name": "ff_train_1024", "op": "ff", "train": True, "rows": 12544, "channels": 1024, "hidden": 4096, "act": "silu",
         "bias": False, "dtype": "bf16"},
        # a training step on one 28x28 image, with biases
        {"name": "ff_train_one_256", "op": "ff", "train": True, "rows": 784, "channels": 256, "hidden": 1024, "act": "gelu",
         "bias": True, "dtype": "fp16"},
        # one image of 56x56 and a row more, in the layers' own type
        {"name": "ff_fp32_256", "op": "ff", "train": False, "rows": 3137, "channels": 256, "hidden": 1024, "act": "gelu", "bias": True,
         "dtype": "fp32"},
        # a batch on its way from a convolution layer to the operators above
        {"name": "to_last_56x56x256", "op": "move", "back": False, "batch": 64, "h": 56, "w": 56, "channels": 256, "dtype": "bf16"},
        # and back to a convolution layer, a small map of odd sizes
        {"name": "to_planes_37x53x100", "op": "move", "back": True, "batch": 3, "h": 37, "w": 53, "channels": 100, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "norm", "ff", "ff", "ff", "move"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "ff":
        train = rng.random() < 0.4
        while True:
            rows, channels, hidden = _log(rng, 1, 50176), 8 * _log(rng, 8, 256), 8 * _log(rng, 16, 1024)
            if rng.random() < 0.15:  # channel counts that fit no vector width
                channels, hidden = channels - rng.randint(1, 7), hidden + rng.randint(1, 7)
            flops = (18 if train else 6) * rows * channels * hidden
            if flops <= (5e10 if dtype == "fp32" else 9e11):
                return {"op": "ff", "train": train, "rows": rows, "channels": channels, "hidden": hidden,
                        "act": rng.choice(("silu", "gelu", "gelu_tanh", "sigmoid")), "bias": rng.random() < 0.5, "dtype": dtype}
    while True:
        batch, h = _log(rng, 1, 64), _log(rng, 4, 224)
        w = max(1, h + rng.randint(-3, 3))
        groups = rng.choice((1, 4, 8, 16, 32, 32))
        channels = groups * _log(rng, 1, 64)
        size = batch * h * w * channels * (2 if dtype == "fp32" else 1)
        if 8 <= channels <= 2048 and size <= 64 * 56 * 56 * 256:
            break
    if op == "move":
        return {"op": "move", "back": rng.random() < 0.5, "batch": batch, "h": h, "w": w, "channels": channels, "dtype": dtype}
    train = rng.random() < 0.5
    wide = channels + rng.choice((0, 0, 0, 8, channels, 3))
    return {"op": "norm", "train": train, "batch": batch, "h": h, "w": w, "channels": channels, "groups": groups,
            "wide": min(wide, 2 * channels), "act": rng.choice(("silu", "gelu") if train else ("none", "relu", "silu", "gelu")),
            "dtype": dtype}


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "move":
        n = case["batch"] * case["h"] * case["w"] * case["channels"]
        return {"bytes": n * (4 + size), "flops": 0}
    if case["op"] == "norm":
        n = case["batch"] * case["h"] * case["w"] * case["channels"]
        maps = 5 if case["train"] else 2  # x, y; then dy, x, dx
        return {"bytes": maps * n * size + 8 * case["channels"] * (2 if case["train"] else 1), "flops": n * (30 if case["train"] else 10)}
    r, c, f = case["rows"], case["channels"], case["hidden"]
    weights = 3 * c * f * size
    if case["train"]:
        return {"bytes": 2 * weights + 4 * r * c * size, "flops": 18 * r * c * f}
    return {"bytes": weights + 2 * r * c * size, "flops": 6 * r * c * f}


# ---- inputs -------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """What the case's operator reads, from the seed alone."""
    g = torch.Generator(device=DEVICE).manual_seed(1_000_003 * (seed + 1))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE) * scale

    if case["op"] == "move":
        shape = (case["batch"], case["channels"], case["h"] * case["w"])
        x = normal(*shape) + normal(1, case["channels"], 1)
        return {"x": x.transpose(1, 2).contiguous().to(dt) if case["back"] else x}
    if case["op"] == "norm":
        n, p, c = case["batch"], case["h"] * case["w"], case["channels"]
        # activations of a convolution: every channel with a level and a spread of its own
        level, spread = normal(1, 1, c), 0.5 + torch.rand(1, 1, c, generator=g, device=DEVICE)
        wide = torch.zeros(n, p, case["wide"], dtype=dt, device=DEVICE)
        wide[:, :, :c] = (normal(n, p, c) * spread + level).to(dt)
        s = {"x": wide[:, :, :c], "gamma": 1 + normal(c, scale=0.1), "beta": normal(c, scale=0.1)}
        if case["train"]:
            s["dy"] = normal(n, p, c).to(dt)
        return s
    r, c, f = case["rows"], case["channels"], case["hidden"]
    s = {"x": normal(r, c).to(dt),
         "w_gate": normal(f, c, scale=c ** -0.5).to(dt), "w_up": normal(f, c, scale=c ** -0.5).to(dt),
         "w_down": normal(c, f, scale=f ** -0.5).to(dt)}
    for name, size in (("b_gate", f), ("b_up", f), ("b_down", c)):
        s[name] = normal(size, scale=0.1).to(dt) if case["bias"] else None
    if case["train"]:
        s["dy"] = normal(r, c).to(dt)
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        import fastconv_b200 as fc
        ctx, x = _ctx(), state["x"]
        new = torch.empty_like
        if case["op"] == "move":
            n, p, c = case["batch"], case["h"] * case["w"], case["channels"]
            state["y"] = (torch.empty(n, c, p, device=DEVICE) if case["back"]
                          else torch.empty(n, p, c, device=DEVICE, dtype=DTYPES[case["dtype"]]))
        elif case["op"] == "norm":
            n, p, c = x.shape
            state["plan"] = fc.GroupNorm(n, p, c, case["groups"], eps=1e-5, act=case["act"], dtype=case["dtype"], x_stride=case["wide"],
                                         ctx=ctx)
            state["y"] = torch.empty(n, p, c, device=DEVICE, dtype=x.dtype)
            if case["train"]:
                state["mean"], state["rstd"] = torch.empty(2, n, case["groups"], device=DEVICE)
                # dx is laid out like x: the slice of a map as wide
                state["dx"] = torch.zeros(n, p, case["wide"], device=DEVICE, dtype=x.dtype)[:, :, :c]
                state["dgamma"], state["dbeta"] = new(state["gamma"]), new(state["beta"])
        else:
            state["plan"] = fc.GatedFeedForward(case["rows"], case["channels"], case["hidden"], act=case["act"], dtype=case["dtype"],
                                                train=case["train"], ctx=ctx)
            state["y"] = new(x)
            if case["train"]:
                state["saved"] = torch.empty(2, case["rows"], case["hidden"], device=DEVICE)  # fp32, whatever the type
                for name in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"):
                    state["d" + name] = None if state[name] is None else new(state[name])
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _act(z, kind):
    """act(z) and its derivative"""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if kind == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s, s * (1 - s)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(z * -(0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    a, b = (2 / math.pi) ** 0.5, 0.044715  # gelu_tanh: 0.5 (1 + tanh v) is 1 / (1 + exp(-2 v))
    s = 1 / (1 + torch.exp(-2 * a * (z + b * z * z * z)))
    return z * s, s + z * s * (1 - s) * 2 * a * (1 + 3 * b * z * z)


def _plain_norm(s, case):
    x = s["x"].float()
    n, p, c = x.shape
    g = case["groups"]
    xg = x.reshape(n, p, g, c // g)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    centred = xg - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + 1e-5)
    xhat = (centred * rstd).reshape(n, p, c)
    y, slope = _act(xhat * s["gamma"] + s["beta"], case["act"])
    y = y.to(s["x"].dtype)
    if not case["train"]:
        return {"y": y}
    dz = s["dy"].float() * slope
    dgamma, dbeta = (dz * xhat).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    dxhat = (dz * s["gamma"]).reshape(n, p, g, c // g)
    xhat = xhat.reshape(n, p, g, c // g)
    dx = rstd * (dxhat - dxhat.mean(dim=(1, 3), keepdim=True) - xhat * (dxhat * xhat).mean(dim=(1, 3), keepdim=True))
    return {"y": y, "dx": dx.reshape(n, p, c).to(s["x"].dtype), "dgamma": dgamma, "dbeta": dbeta}


def _plain_ff(s, case):
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    gate, up = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        gate, up = gate + s["b_gate"].float(), up + s["b_up"].float()
    a, slope = _act(gate, case["act"])
    hid = a * up
    y = hid @ wd.t()
    if case["bias"]:
        y = y + s["b_down"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dhid = dy @ wd
        dgate, dup = dhid * up * slope, dhid * a
        out["dx"] = (dgate @ wg + dup @ wu).to(dt)
        out["dw_gate"], out["dw_up"], out["dw_down"] = (dgate.t() @ x).to(dt), (dup.t() @ x).to(dt), (dy.t() @ hid).to(dt)
        if case["bias"]:
            out["db_gate"], out["db_up"], out["db_down"] = dgate.sum(0).to(dt), dup.sum(0).to(dt), dy.sum(0).to(dt)
    return out


def _plain_move(s, case):
    x = s["x"].transpose(1, 2)
    return {"y": (x.float() if case["back"] else x.to(DTYPES[case["dtype"]])).contiguous()}


# ---- one pass -----------------------------------------------------------------------------------------------------

def _at(t):
    return 0 if t is None else t.data_ptr()


def _own(s, case):
    if case["op"] == "move":
        import fastconv_b200 as fc
        move = fc.from_channels_last if case["back"] else fc.to_channels_last
        move(_at(s["x"]), _at(s["y"]), case["batch"], case["channels"], case["h"] * case["w"], dtype=case["dtype"], ctx=_ctx())
        return {"y": s["y"]}
    plan = s["plan"]
    if case["op"] == "norm":
        if not case["train"]:
            plan.forward(_at(s["x"]), _at(s["y"]), gamma=_at(s["gamma"]), beta=_at(s["beta"]))
            return {"y": s["y"]}
        plan.forward(_at(s["x"]), _at(s["y"]), gamma=_at(s["gamma"]), beta=_at(s["beta"]), mean=_at(s["mean"]), rstd=_at(s["rstd"]))
        plan.backward(_at(s["dy"]), _at(s["x"]), _at(s["dx"]), gamma=_at(s["gamma"]), beta=_at(s["beta"]), mean=_at(s["mean"]),
                      rstd=_at(s["rstd"]), dgamma=_at(s["dgamma"]), dbeta=_at(s["dbeta"]))
        return {k: s[k] for k in ("y", "dx", "dgamma", "dbeta")}
    weights = {k: _at(s[k]) for k in ("w_gate", "w_up", "w_down")}
    biases = {k: _at(s[k]) for k in ("b_gate", "b_up", "b_down")}
    if not case["train"]:
        plan.forward(_at(s["x"]), _at(s["y"]), **weights, **biases)
        return {"y": s["y"]}
    plan.forward(_at(s["x"]), _at(s["y"]), **weights, **biases, saved=_at(s["saved"]))
    grads = [k for k in ("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down") if s[k] is not None]
    plan.backward(_at(s["dy"]), _at(s["x"]), **weights, saved=_at(s["saved"]), **{k: _at(s[k]) for k in grads})
    return {"y": s["y"], **{k: s[k] for k in grads}}


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"norm": _plain_norm, "ff": _plain_ff, "move": _plain_move}[case["op"]](state, case)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------

def _act64(z, kind):
    if kind == "none":
        return z
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "sigmoid":
        return torch.sigmoid(z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def exact(case, seed):
    """Outputs of `run` from the definitions in 64 bits; gradients by differentiating the definition."""
    s = {k: v if v is None else v.double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "move":
        return {"y": s["x"].permute(0, 2, 1).contiguous()}
    train = case["train"]
    names = ("x", "gamma", "beta") if case["op"] == "norm" else ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")
    names = [k for k in names if s[k] is not None]
    for k in names:
        s[k] = s[k].contiguous().requires_grad_(train)
    if case["op"] == "norm":
        n, p, c = s["x"].shape
        rows = s["x"].view(n, p, case["groups"], -1).permute(0, 2, 1, 3).reshape(n, case["groups"], -1)
        var, mean = torch.var_mean(rows, dim=2, correction=0, keepdim=True)
        rows = (rows - mean) / (var + 1e-5).sqrt()
        z = rows.view(n, case["groups"], p, -1).permute(0, 2, 1, 3).reshape(n, p, c)
        y = _act64(z * s["gamma"] + s["beta"], case["act"])
    else:
        def project(v, w, b):
            v = torch.einsum("rk,fk->rf", v, s[w])
            return v if s[b] is None else v + s[b]

        y = project(_act64(project(s["x"], "w_gate", "b_gate"), case["act"]) * project(s["x"], "w_up", "b_up"), "w_down", "b_down")
    if not train:
        return {"y": y}
    grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, grads)}}
