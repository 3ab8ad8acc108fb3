"""The channels-last operators on the GPU against their plain forms in 64 bits (tests/_last_ref.py)."""
import pytest
import torch

import fastconv_b200 as fc
from _last_ref import DTYPES, act, check, ff, norm, stored

pytestmark = pytest.mark.gpu

GUARD = 7.0  # what stands between the channels of a strided map, and has to stand there afterwards


@pytest.fixture(scope="module")
def lctx():
    c = fc.Context(0, arena_bytes=2 << 30)
    yield c
    c.close()


def at(t):
    return 0 if t is None else t.data_ptr()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def strided(rows, channels, stride, dtype, values=None, offset=0):
    """A [rows][channels] view on the GPU whose rows are `stride` apart, with guards around it."""
    flat = torch.full((rows * stride + offset + 16,), GUARD, dtype=DTYPES[dtype], device="cuda")
    view = flat[offset:offset + rows * stride].view(rows, stride)[:, :channels]
    if values is not None:
        view.copy_(values)
    return flat, view


def guards_hold(flat, rows, channels, stride, offset=0):
    flat = flat.clone()
    flat[offset:offset + rows * stride].view(rows, stride)[:, :channels] = GUARD
    return bool((flat == GUARD).all())


def done(ctx):
    ctx.synchronize()
    torch.cuda.synchronize()


# ---- moves ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("batch,channels,pixels,stride,offset", [
    (1, 1, 1, 0, 0), (2, 3, 224, 0, 0), (3, 100, 37 * 53, 0, 0), (2, 64, 64, 64, 0), (1, 65, 129, 70, 1), (2, 8, 1000, 24, 8),
    (5, 512, 7, 512, 0), (2, 72, 66, 144, 0), (1, 128, 196, 129, 3)])
def test_moves_are_exact_both_ways(lctx, dtype, batch, channels, pixels, stride, offset):
    step = stride or channels
    x = torch.randn(batch, channels, pixels, generator=gen(1)).cuda()
    flat, last = strided(batch * pixels, channels, step, dtype, offset=offset)
    torch.cuda.synchronize()
    fc.to_channels_last(at(x), at(last), batch, channels, pixels, dtype=dtype, stride=stride, ctx=lctx)
    done(lctx)
    want = x.transpose(1, 2).to(DTYPES[dtype])
    assert torch.equal(last.view(batch, pixels, channels) if step == channels else last.reshape(batch, pixels, channels), want)
    assert guards_hold(flat, batch * pixels, channels, step, offset)
    back = torch.full_like(x, GUARD)
    torch.cuda.synchronize()
    fc.from_channels_last(at(last), at(back), batch, channels, pixels, dtype=dtype, stride=stride, ctx=lctx)
    done(lctx)
    assert torch.equal(back, want.float().transpose(1, 2).contiguous())


def test_a_move_keeps_infinities_and_nans(lctx):
    x = torch.tensor([[[float("inf"), -float("inf"), float("nan"), 1e38]]]).cuda()
    y = torch.empty(1, 4, 1, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    fc.to_channels_last(at(x), at(y), 1, 1, 4, dtype="fp16", ctx=lctx)
    done(lctx)
    assert y.flatten().tolist()[:2] == [float("inf"), -float("inf")]
    assert torch.isnan(y.flatten()[2]) and y.flatten()[3] == float("inf")


# ---- group norm -----------------------------------------------------------------------------------------------------

def run_norm(ctx, n, p, c, groups, kind, dtype, *, params="fp32", xs=0, ys=0, offset=0, affine=True, level=1.0, train=True, eps=1e-5,
             seed=3):
    g = gen(seed)
    xs, ys = xs or c, ys or c
    values = (torch.randn(n * p, c, generator=g) * (0.5 + torch.rand(c, generator=g)) + level * torch.randn(c, generator=g))
    fx, x = strided(n * p, c, xs, dtype, values.cuda(), offset)
    fdy, dy = strided(n * p, c, ys, dtype, torch.randn(n * p, c, generator=g).cuda(), offset)
    fy, y = strided(n * p, c, ys, dtype, offset=offset)
    fdx, dx = strided(n * p, c, xs, dtype, offset=offset)
    pt = DTYPES[params]
    gamma = (1 + 0.2 * torch.randn(c, generator=g)).to(pt).cuda() if affine else None
    beta = (0.3 * torch.randn(c, generator=g)).to(pt).cuda() if affine else None
    mean, rstd = torch.empty(2, n, groups, device="cuda")
    dgamma, dbeta = torch.full((2, c), GUARD, dtype=pt, device="cuda")
    plan = fc.GroupNorm(n, p, c, groups, eps=eps, act=kind, dtype=dtype, param_dtype=params, x_stride=xs, y_stride=ys, ctx=ctx)
    torch.cuda.synchronize()
    plan.forward(at(x), at(y), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd))
    if train:
        plan.backward(at(dy), at(x), at(dx), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd), dgamma=at(dgamma),
                      dbeta=at(dbeta))
    done(ctx)
    wide = lambda t: t.double().cpu().reshape(n, p, c)  # noqa: E731
    flat1 = lambda t, fill: torch.full((c,), fill, dtype=torch.float64) if t is None else t.double().cpu()  # noqa: E731
    want = norm(wide(x), groups, eps, flat1(gamma, 1.0), flat1(beta, 0.0), kind, dtype, wide(dy) if train else None)
    check(y.reshape(n, p, c), *want["y"], dtype, "y")
    check(mean, *want["mean"], "fp32", "mean")
    check(rstd, *want["rstd"], "fp32", "rstd")
    assert guards_hold(fy, n * p, c, ys, offset) and guards_hold(fx, n * p, c, xs, offset)
    if train:
        check(dx.reshape(n, p, c), *want["dx"], dtype, "dx")
        check(dgamma, *want["dgamma"], params, "dgamma")
        check(dbeta, *want["dbeta"], params, "dbeta")
        assert guards_hold(fdx, n * p, c, xs, offset) and guards_hold(fdy, n * p, c, ys, offset)
    plan.release()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,p,c,groups", [
    (1, 1, 1, 1), (1, 1, 32, 32), (2, 1, 64, 8), (1, 5, 8, 2), (3, 49, 24, 3), (2, 196, 512, 32), (1, 3136, 64, 32),
    (4, 100, 320, 32), (1, 37 * 53, 96, 1), (2, 17, 2056, 8), (2, 1000, 4096, 4), (1, 12544, 128, 16), (65, 9, 48, 6),
    (2, 3000, 130, 13), (1, 50176, 64, 4), (1, 777, 33, 3)])
def test_norm_shapes(lctx, dtype, n, p, c, groups):
    run_norm(lctx, n, p, c, groups, "silu", dtype)


@pytest.mark.parametrize("kind", ["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_norm_activations(lctx, dtype, kind):
    run_norm(lctx, 2, 150, 64, 4, kind, dtype)


@pytest.mark.parametrize("dtype,c,xs,ys,offset", [
    ("bf16", 320, 480, 320, 0), ("bf16", 320, 320, 640, 0), ("fp16", 64, 67, 64, 0), ("fp32", 64, 64, 65, 0), ("bf16", 64, 64, 64, 1),
    ("fp32", 40, 44, 48, 4), ("fp32", 40, 40, 40, 1), ("fp16", 36, 36, 36, 0), ("fp16", 72, 80, 88, 8)])
def test_norm_of_slices(lctx, dtype, c, xs, ys, offset):
    run_norm(lctx, 2, 333, c, 4, "gelu", dtype, xs=xs, ys=ys, offset=offset)


@pytest.mark.parametrize("affine,params", [(False, "fp32"), (True, "bf16")])
def test_norm_parameters(lctx, affine, params):
    run_norm(lctx, 3, 64, 64, 8, "silu", "bf16", affine=affine, params=params)


def test_norm_of_a_map_far_from_zero(lctx):
    run_norm(lctx, 2, 3136, 64, 8, "none", "fp32", level=1000.0)
    run_norm(lctx, 1, 900, 64, 64, "none", "fp32", level=1000.0)


def test_norm_of_a_constant_map(lctx):
    """The variance is zero: rstd is 1 / sqrt(eps), and the result beta."""
    n, p, c = 2, 300, 32
    x = torch.full((n, p, c), 3.7, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(n, 4, device="cuda"), torch.empty(n, 4, device="cuda")
    plan = fc.GroupNorm(n, p, c, 4, eps=1e-5, ctx=lctx)
    torch.cuda.synchronize()
    plan.forward(at(x), at(y), mean=at(mean), rstd=at(rstd))
    done(lctx)
    # the mean is within a step of 3.7, which rstd (316) makes of the result
    assert (mean - 3.7).abs().max() <= 4e-7 and y.abs().max() <= 4e-7 * 317
    assert torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-5)


def test_norm_confines_a_nan_to_its_group(lctx):
    n, p, c, groups = 2, 200, 64, 8
    x = torch.randn(n, p, c, generator=gen(5)).cuda().half()
    x[1, 77, 20] = float("nan")
    y = torch.empty_like(x)
    for kind in ("relu", "silu"):
        plan = fc.GroupNorm(n, p, c, groups, act=kind, dtype="fp16", ctx=lctx)
        torch.cuda.synchronize()
        plan.forward(at(x), at(y))
        done(lctx)
        bad = torch.isnan(y)
        assert bool(bad[1, :, 16:24].all()) and int(bad.sum()) == p * 8


def test_norm_gradients_one_by_one_and_of_no_images(lctx):
    n, p, c = 2, 60, 32
    x, dy = torch.randn(2, n, p, c, generator=gen(6)).cuda()
    full, alone = [torch.empty_like(x), torch.empty(c, device="cuda"), torch.empty(c, device="cuda")], None
    alone = [torch.empty_like(t) for t in full]
    y, mean, rstd = torch.empty_like(x), torch.empty(n, 4, device="cuda"), torch.empty(n, 4, device="cuda")
    plan = fc.GroupNorm(n, p, c, 4, act="silu", ctx=lctx)
    none = fc.GroupNorm(0, p, c, 4, act="silu", ctx=lctx)
    torch.cuda.synchronize()
    plan.forward(at(x), at(y), mean=at(mean), rstd=at(rstd))
    plan.backward(at(dy), at(x), at(full[0]), mean=at(mean), rstd=at(rstd), dgamma=at(full[1]), dbeta=at(full[2]))
    plan.backward(at(dy), at(x), at(alone[0]), mean=at(mean), rstd=at(rstd))
    plan.backward(at(dy), at(x), mean=at(mean), rstd=at(rstd), dgamma=at(alone[1]))
    plan.backward(at(dy), at(x), mean=at(mean), rstd=at(rstd), dbeta=at(alone[2]))
    done(lctx)
    assert all(torch.equal(a, b) for a, b in zip(full, alone))
    none.forward(0, 0)
    none.backward(0, 0, mean=0, rstd=0, dgamma=at(full[1]), dbeta=at(full[2]))
    done(lctx)
    assert not full[1].any() and not full[2].any()


def test_norm_gradient_against_differences(lctx):
    """d(sum w y) along a direction: central differences of the forward kernel, fp32.  A step of 2^-6 leaves a cubic term of
    2^-12 / 6 times the third derivative (of order one here, as x, w and the direction are), and the kernel's own rounding,
    about 1e-6 a value over a step of 2^-5: together under 1e-3 of the gradient's and the direction's length."""
    n, p, c, groups = 2, 40, 32, 4
    g = gen(8)
    x, w, v = (torch.randn(n, p, c, generator=g).cuda() for _ in range(3))
    gamma, beta = 1 + 0.2 * torch.randn(c, generator=g).cuda(), 0.3 * torch.randn(c, generator=g).cuda()
    vg, vb = torch.randn(c, generator=g).cuda(), torch.randn(c, generator=g).cuda()
    plan = fc.GroupNorm(n, p, c, groups, act="gelu", ctx=lctx)
    mean, rstd, y = torch.empty(n, groups, device="cuda"), torch.empty(n, groups, device="cuda"), torch.empty_like(x)
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
    torch.cuda.synchronize()
    plan.forward(at(x), at(y), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd))
    plan.backward(at(w), at(x), at(dx), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd), dgamma=at(dgamma),
                  dbeta=at(dbeta))
    done(lctx)

    def along(step, dx_, dg_, db_):
        xs, gs, bs = (x + step * dx_).contiguous(), gamma + step * dg_, beta + step * db_
        torch.cuda.synchronize()
        plan.forward(at(xs), at(y), gamma=at(gs), beta=at(bs))
        done(lctx)
        return (y.double() * w.double()).sum().item()

    step, zx, zc = 2.0 ** -6, torch.zeros_like(x), torch.zeros_like(gamma)
    for grad, direction, args in ((dx, v, (v, zc, zc)), (dgamma, vg, (zx, vg, zc)), (dbeta, vb, (zx, zc, vb))):
        slope = (along(step, *args) - along(-step, *args)) / (2 * step)
        want = (grad.double() * direction.double()).sum().item()
        assert abs(slope - want) <= 2e-3 * grad.double().norm().item() * direction.double().norm().item()


# ---- gated feed-forward block ---------------------------------------------------------------------------------------

def run_ff(ctx, rows, k, f, o, kind, dtype, *, bias=True, xs=0, ys=0, train=True, seed=11, scale=1.0):
    g = gen(seed)
    xs, ys = xs or k, ys or o
    dt = DTYPES[dtype]
    rnd = lambda *s, by=1.0: (torch.randn(*s, generator=g) * by).to(dt).cuda()  # noqa: E731
    fx, x = strided(rows, k, xs, dtype, rnd(rows, k))
    fdy, dy = strided(rows, o, ys, dtype, rnd(rows, o))
    fy, y = strided(rows, o, ys, dtype)
    fdx, dx = strided(rows, k, xs, dtype)
    t = {"x": x, "w_gate": rnd(f, k, by=scale * k ** -0.5), "w_up": rnd(f, k, by=scale * k ** -0.5), "w_down": rnd(o, f, by=f ** -0.5)}
    for name, size in (("b_gate", f), ("b_up", f), ("b_down", o)):
        t[name] = rnd(size, by=0.2) if bias else None
    saved = torch.full((2, rows, f), GUARD, device="cuda") if train else None
    plan = fc.GatedFeedForward(rows, k, f, o, act=kind, dtype=dtype, x_stride=xs, y_stride=ys, train=train, ctx=ctx)
    weights = {n: at(t[n]) for n in ("w_gate", "w_up", "w_down")}
    grads = {"dx": dx}
    for n in ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"):
        if t[n] is not None:
            grads["d" + n] = torch.full_like(t[n], GUARD)
    torch.cuda.synchronize()
    plan.forward(at(x), at(y), **weights, **{n: at(t[n]) for n in ("b_gate", "b_up", "b_down")}, saved=at(saved))
    if train:
        plan.backward(at(dy), at(x), **weights, saved=at(saved), **{n: at(v) for n, v in grads.items()})
    done(ctx)
    wide = lambda v: None if v is None else v.double().cpu()  # noqa: E731
    want = ff({n: wide(v) for n, v in t.items()}, kind, dtype, wide(dy) if train else None)
    check(y, *want["y"], dtype, "y")
    assert guards_hold(fy, rows, o, ys)
    if train:
        for v, n in zip(saved, ("gate", "up")):  # in an order of the library's own: compared as sets
            w, e = (q.flatten() for q in want[n])
            check(v.flatten().sort().values, w.sort().values, e.max().expand_as(w), "fp32", n)
        for n, v in grads.items():
            check(v, *want[n], dtype, n)
        assert guards_hold(fdx, rows, k, xs)
    plan.release()


FF_SHAPES = [(1, 8, 8, 8), (1, 64, 128, 64), (1, 1, 1, 1), (2, 33, 65, 17), (3, 72, 200, 40), (7, 128, 256, 136), (16, 256, 512, 256),
             (17, 96, 320, 64), (64, 200, 328, 104), (100, 64, 1000, 72), (129, 256, 264, 128), (196, 104, 520, 264), (300, 320, 136, 520),
             (515, 64, 128, 64), (1000, 136, 72, 40), (128, 127, 129, 65), (260, 250, 130, 66)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,k,f,o", FF_SHAPES)
def test_ff_shapes(lctx, dtype, rows, k, f, o):
    run_ff(lctx, rows, k, f, o, "silu", dtype)


@pytest.mark.parametrize("kind", ["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 140])
def test_ff_activations(lctx, rows, dtype, kind):
    run_ff(lctx, rows, 64, 136, 72, kind, dtype, scale=3.0)


@pytest.mark.parametrize("dtype,rows,xs,ys", [("bf16", 70, 128, 64), ("bf16", 70, 64, 72), ("fp16", 5, 65, 64), ("fp32", 70, 68, 67),
                                              ("bf16", 1, 80, 80), ("fp16", 300, 96, 71)])
def test_ff_of_slices(lctx, dtype, rows, xs, ys):
    run_ff(lctx, rows, 64, 128, 64, "silu", dtype, xs=xs, ys=ys)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ff_without_biases_and_for_inference(lctx, dtype):
    for rows in (1, 9, 300):
        run_ff(lctx, rows, 64, 128, 64, "silu", dtype, bias=False)
        run_ff(lctx, rows, 64, 128, 64, "gelu", dtype, train=False)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ff_long_reductions(lctx, dtype):
    run_ff(lctx, 5000, 64, 64, 64, "silu", dtype)
    run_ff(lctx, 40, 64, 4096, 64, "silu", dtype)
    run_ff(lctx, 40, 2048, 64, 64, "silu", dtype)
    run_ff(lctx, 1, 4096, 4096, 256, "silu", dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ff_of_no_rows(lctx, dtype):
    k, f, o = 64, 128, 72
    dt = DTYPES[dtype]
    plan = fc.GatedFeedForward(0, k, f, o, dtype=dtype, train=True, ctx=lctx)
    sizes = {"dw_gate": (f, k), "dw_up": (f, k), "dw_down": (o, f), "db_gate": (f,), "db_up": (f,), "db_down": (o,)}
    grads = {n: torch.full(s, GUARD, dtype=dt, device="cuda") for n, s in sizes.items()}
    torch.cuda.synchronize()
    plan.forward(0, 0, w_gate=0, w_up=0, w_down=0)
    plan.backward(0, 0, w_gate=0, w_up=0, w_down=0, saved=0, **{n: at(v) for n, v in grads.items()})
    done(lctx)
    assert not any(v.any() for v in grads.values())


@pytest.mark.parametrize("dtype,rows", [("bf16", 300), ("bf16", 3), ("fp32", 300)])
def test_ff_gradients_one_by_one(lctx, dtype, rows):
    """Each gradient alone is the one that comes with the others, bit for bit, and again on a second run."""
    k, f = 64, 128
    dt = DTYPES[dtype]
    g = gen(21)
    rnd = lambda *s: (0.3 * torch.randn(*s, generator=g)).to(dt).cuda()  # noqa: E731
    x, dy, saved = rnd(rows, k), rnd(rows, k), rnd(2, rows, f).float()
    w = {"w_gate": rnd(f, k), "w_up": rnd(f, k), "w_down": rnd(k, f)}
    sizes = {"dx": (rows, k), "dw_gate": (f, k), "dw_up": (f, k), "dw_down": (k, f), "db_gate": (f,), "db_up": (f,), "db_down": (k,)}
    full = {n: torch.full(s, GUARD, dtype=dt, device="cuda") for n, s in sizes.items()}
    plan = fc.GatedFeedForward(rows, k, f, dtype=dtype, train=True, ctx=lctx)
    call = lambda d: plan.backward(at(dy), at(x), **{n: at(v) for n, v in w.items()}, saved=at(saved),  # noqa: E731
                                   **{n: at(v) for n, v in d.items()})
    torch.cuda.synchronize()
    call(full)
    for n, s in sizes.items():
        one = torch.full(s, GUARD, dtype=dt, device="cuda")
        torch.cuda.synchronize()
        call({n: one})
        done(lctx)
        assert torch.equal(one, full[n]), n


def test_ff_gradient_against_differences(lctx):
    """As for the norm, fp32: the block is smooth and its third derivatives are of order one at these scales."""
    rows, k, f, o = 30, 32, 48, 24
    g = gen(31)
    t = {"x": torch.randn(rows, k, generator=g), "w_gate": torch.randn(f, k, generator=g) * k ** -0.5,
         "w_up": torch.randn(f, k, generator=g) * k ** -0.5, "w_down": torch.randn(o, f, generator=g) * f ** -0.5,
         "b_gate": 0.1 * torch.randn(f, generator=g), "b_up": 0.1 * torch.randn(f, generator=g), "b_down": 0.1 * torch.randn(o, generator=g)}
    t = {n: v.cuda() for n, v in t.items()}
    w = torch.randn(rows, o, generator=g).cuda()
    plan = fc.GatedFeedForward(rows, k, f, o, act="gelu_tanh", dtype="fp32", train=True, ctx=lctx)
    y, saved = torch.empty(rows, o, device="cuda"), torch.empty(2, rows, f, device="cuda")
    grads = {n: torch.empty_like(v) for n, v in t.items()}

    def forward(values, keep=0):
        torch.cuda.synchronize()
        plan.forward(at(values["x"]), at(y), **{n: at(v) for n, v in values.items() if n != "x"}, saved=keep)
        done(lctx)
        return (y.double() * w.double()).sum().item()

    forward(t, at(saved))
    plan.backward(at(w), at(t["x"]), **{n: at(t[n]) for n in ("w_gate", "w_up", "w_down")}, saved=at(saved),
                  **{"d" + n: at(v) for n, v in grads.items()})
    done(lctx)
    for n in t:
        v = torch.randn(t[n].shape, generator=g).cuda()
        v /= v.norm() / 4
        step = 2.0 ** -6
        up, down = dict(t), dict(t)
        up[n], down[n] = t[n] + step * v, t[n] - step * v
        slope = (forward(up) - forward(down)) / (2 * step)
        want = (grads[n].double() * v.double()).sum().item()
        assert abs(slope - want) <= 2e-3 * grads[n].double().norm().item() * v.double().norm().item(), n


# ---- together -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_a_convolution_and_what_follows_it(lctx, dtype):
    """conv -> channels last -> norm and activation -> block -> back to planes -> conv, all on the device, twice: once call
    by call and once replayed from a graph captured on the context's stream.  Each operator is held to its own bound on the
    inputs that it had."""
    n, c, h, w, f, groups = 2, 24, 13, 11, 80, 4
    p = h * w
    dt = DTYPES[dtype]
    x = fc.synth.conv_input(n, c, h, w, 41)
    convs = []
    for seed in (42, 43):
        layer = fc.ConvWinoF63ZCLayer(x, fc.synth.conv_weights(c, c, 3, 3, seed), None, None, c, h, w, c, batch=n, ctx=lctx)
        layer.Init()
        convs.append(layer)
    g = gen(44)
    rnd = lambda *s, by=1.0: (torch.randn(*s, generator=g) * by).to(dt).cuda()  # noqa: E731
    d_in = torch.from_numpy(x).cuda()
    planes, end, out = (torch.zeros(n, c, p, device="cuda") for _ in range(3))
    a, b, d = (torch.zeros(n * p, c, dtype=dt, device="cuda") for _ in range(3))
    gamma, beta = 1 + 0.1 * torch.randn(c, generator=g).cuda(), 0.1 * torch.randn(c, generator=g).cuda()
    t = {"w_gate": rnd(f, c, by=c ** -0.5), "w_up": rnd(f, c, by=c ** -0.5), "w_down": rnd(c, f, by=f ** -0.5)}
    gn = fc.GroupNorm(n, p, c, groups, act="silu", dtype=dtype, ctx=lctx)
    block = fc.GatedFeedForward(n * p, c, f, act="silu", dtype=dtype, ctx=lctx)
    lib = fc.load()

    def chain():
        assert lib.fc_conv_forward_device(convs[0]._conv, at(d_in), at(planes)) == 0
        fc.to_channels_last(at(planes), at(a), n, c, p, dtype=dtype, ctx=lctx)
        gn.forward(at(a), at(b), gamma=at(gamma), beta=at(beta))
        block.forward(at(b), at(d), **{k: at(v) for k, v in t.items()})
        fc.from_channels_last(at(d), at(end), n, c, p, dtype=dtype, ctx=lctx)
        assert lib.fc_conv_forward_device(convs[1]._conv, at(end), at(out)) == 0

    torch.cuda.synchronize()
    chain()
    done(lctx)
    assert torch.equal(a.view(n, p, c), planes.transpose(1, 2).to(dt))
    want = norm(a.double().cpu().view(n, p, c), groups, 1e-5, gamma.double().cpu(), beta.double().cpu(), "silu", dtype)
    check(b.view(n, p, c), *want["y"], dtype, "norm")
    vals = {"x": b.double().cpu(), **{k: v.double().cpu() for k, v in t.items()}, "b_gate": None, "b_up": None, "b_down": None}
    check(d, *ff(vals, "silu", dtype)["y"], dtype, "block")
    assert torch.equal(end, d.float().view(n, p, c).transpose(1, 2).contiguous())
    first = [v.clone() for v in (planes, a, b, d, end, out)]
    assert out.abs().sum() > 0

    stream = torch.cuda.ExternalStream(lctx.stream.value)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        chain()
    for v in (planes, a, b, d, end, out):
        v.fill_(GUARD)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(3):
            graph.replay()
    done(lctx)
    assert all(torch.equal(u, v) for u, v in zip(first, (planes, a, b, d, end, out)))
    del graph
    for layer in convs:
        layer.release()


def test_two_plans_interleave_on_one_stream(lctx):
    """Calls of plans with workspaces of their own do not disturb one another."""
    g = gen(51)
    x = torch.randn(700, 64, generator=g).cuda().bfloat16()
    w = {k: (0.1 * torch.randn(*s, generator=g)).cuda().bfloat16() for k, s in
         (("w_gate", (128, 64)), ("w_up", (128, 64)), ("w_down", (64, 128)))}
    plans = [fc.GatedFeedForward(r, 64, 128, dtype="bf16", ctx=lctx) for r in (700, 3, 700)]
    ys = [[torch.empty(r, 64, dtype=torch.bfloat16, device="cuda") for r in (700, 3, 700)] for _ in range(2)]
    torch.cuda.synchronize()
    for plan, y in zip(plans, ys[0]):
        plan.forward(at(x), at(y), **{k: at(v) for k, v in w.items()})
        lctx.synchronize()
    for _ in range(5):
        for plan, y in zip(plans, ys[1]):
            plan.forward(at(x), at(y), **{k: at(v) for k, v in w.items()})
    done(lctx)
    assert all(torch.equal(a, b) for a, b in zip(*ys)) and torch.equal(ys[0][0], ys[0][2])


# ---- refusals that need a context -----------------------------------------------------------------------------------

def test_calls_that_are_refused(lctx):
    """Nothing is launched: the checks are the host's."""
    lib, bad = fc.load(), -1
    a = torch.full((4096,), GUARD, device="cuda")
    p, q, w, h = a.data_ptr(), a.data_ptr() + 4096, a.data_ptr() + 8192, lctx.handle
    torch.cuda.synchronize()
    assert lib.fc_map_to_channels_last(h, None, q, 1, 4, 4, 0, 0) == bad
    assert lib.fc_map_to_channels_last(h, p + 2, q, 1, 4, 4, 0, 0) == bad
    assert lib.fc_map_from_channels_last(h, p + 1, q, 1, 4, 4, 0, 1) == bad
    assert lib.fc_map_to_channels_last(h, p, q, 1, 4, 4, 3, 0) == bad
    assert lib.fc_map_to_channels_last(h, p, q, 1, 4, 4, 0, 7) == bad
    assert lib.fc_map_to_channels_last(h, p, q, -1, 4, 4, 0, 0) == bad
    assert lib.fc_map_to_channels_last(h, p, q, 1, 1 << 30, 4, 0, 0) == -2
    gn = fc.GroupNorm(1, 16, 8, 2, ctx=lctx)
    d, n = gn._ref, gn.workspace_bytes
    fwd = lib.fc_group_norm_forward
    assert fwd(h, d, p, None, None, None, None, None, w, n) == bad
    assert fwd(h, d, p, None, None, p, None, None, w, n) == bad
    assert fwd(h, d, p + 2, None, None, q, None, None, w, n) == bad
    assert fwd(h, d, p, p + 1, None, q, None, None, w, n) == bad
    assert fwd(h, d, p, None, None, q, None, None, None, n) == bad
    assert fwd(h, d, p, None, None, q, None, None, w + 4, n) == bad
    assert fwd(h, d, p, None, None, q, None, None, w, 16) == bad
    bwd = lib.fc_group_norm_backward
    assert bwd(h, d, p, p + 512, None, None, None, None, q, None, None, w, n) == bad  # no mean and rstd
    assert bwd(h, d, p, q, None, None, p, p, q, None, None, w, n) == bad
    assert bwd(h, d, p, q, None, None, p, p, w, None, None, w, 16) == bad
    ff = fc.GatedFeedForward(4, 8, 16, dtype="fp32", train=True, ctx=lctx)
    d, n = ff._ref, ff.workspace_bytes
    fwd, bwd = lib.fc_gated_ff_forward, lib.fc_gated_ff_backward
    ops = [p, p, p, p, None, None, None, q, None, w, n]
    for i, v in ((0, None), (1, None), (2, None), (3, None), (7, None), (7, p), (0, p + 2), (4, p + 1), (8, p + 2), (9, None), (9, w + 8),
                 (10, 64)):
        assert fwd(h, d, *[v if j == i else o for j, o in enumerate(ops)]) == bad, i
    ops = [p, p, p, p, p, p, q, None, None, None, None, None, None, w, n]
    for i, v in ((0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (6, p), (6, q + 1), (7, q + 2), (5, p + 2), (13, None),
                 (14, 64)):
        assert bwd(h, d, *[v if j == i else o for j, o in enumerate(ops)]) == bad, i
    with pytest.raises(RuntimeError, match="train"):
        fc.GatedFeedForward(4, 8, 16, dtype="fp32", ctx=lctx).backward(p, p, w_gate=p, w_up=p, w_down=p, saved=p)
    gn.release()
    with pytest.raises(RuntimeError, match="released"):
        gn.forward(p, q)
    done(lctx)
    assert bool((a == GUARD).all())


# ---- far offsets, far levels ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("channels", [16, 15])
def test_offsets_past_32_bits(lctx, channels):
    """Rows so far apart that the last ones' offsets pass 2^31 elements."""
    rows, stride = 40000, 1 << 16
    flat = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    view = flat.view(rows, stride)
    x = torch.randn(rows, channels, generator=gen(61)).cuda().bfloat16()
    view[:, :channels] = x
    near = torch.empty_like(x)
    for kind in ("norm", "ff", "move"):
        torch.cuda.synchronize()
        if kind == "norm":
            for xs, ys, src, dst in ((0, 0, x, near), (stride, stride, view, view[:, 64:])):
                fc.GroupNorm(1, rows, channels, 1, act="silu", dtype="bf16", x_stride=xs, y_stride=ys, ctx=lctx).forward(at(src), at(dst))
        elif kind == "ff":
            w = {k: (0.2 * torch.randn(*s, generator=gen(62))).cuda().bfloat16() for k, s in
                 (("w_gate", (24, channels)), ("w_up", (24, channels)), ("w_down", (channels, 24)))}
            torch.cuda.synchronize()
            for xs, ys, src, dst in ((0, 0, x, near), (stride, stride, view, view[:, 64:])):
                fc.GatedFeedForward(rows, channels, 24, dtype="bf16", x_stride=xs, y_stride=ys, ctx=lctx).forward(
                    at(src), at(dst), **{k: at(v) for k, v in w.items()})
        else:
            planes = torch.empty(channels, rows, device="cuda")
            torch.cuda.synchronize()
            fc.from_channels_last(at(view), at(planes), 1, channels, rows, dtype="bf16", stride=stride, ctx=lctx)
            fc.to_channels_last(at(planes), at(view[:, 64:]), 1, channels, rows, dtype="bf16", stride=stride, ctx=lctx)
            near = x
        done(lctx)
        assert torch.equal(view[:, 64:64 + channels], near), kind
    assert torch.equal(view[:, :channels], x)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("p,c,groups", [(196, 64, 8), (5000, 64, 4), (777, 33, 3)])
def test_norm_where_a_groups_first_value_is_far_off(lctx, dtype, p, c, groups):
    """The value that squares are taken around is an outlier of 3000 standard deviations."""
    n = 2
    x = torch.randn(n, p, c, generator=gen(71))
    x[:, 0, ::c // groups] = 3000.0
    x[:, p // 2, 1::c // groups] = -2000.0
    x = x.cuda().to(DTYPES[dtype])
    y, mean, rstd = torch.empty_like(x), torch.empty(n, groups, device="cuda"), torch.empty(n, groups, device="cuda")
    plan = fc.GroupNorm(n, p, c, groups, dtype=dtype, ctx=lctx)
    torch.cuda.synchronize()
    plan.forward(at(x), at(y), mean=at(mean), rstd=at(rstd))
    done(lctx)
    one, zero = torch.ones(c, dtype=torch.float64), torch.zeros(c, dtype=torch.float64)
    want = norm(x.double().cpu(), groups, 1e-5, one, zero, "none", dtype)
    check(y, *want["y"], dtype, "y")
    check(rstd, *want["rstd"], "fp32", "rstd")


def test_ff_of_very_large_and_very_small_fp32(lctx):
    """Operands of 1e20 and 1e-20: each is split by its own size."""
    rows, k, f = 140, 72, 136
    g = gen(81)
    t = {"x": 1e20 * torch.randn(rows, k, generator=g), "w_gate": 1e-20 * torch.randn(f, k, generator=g) * k ** -0.5,
         "w_up": 1e-20 * torch.randn(f, k, generator=g) * k ** -0.5, "w_down": 1e18 * torch.randn(k, f, generator=g) * f ** -0.5}
    t = {n: v.cuda() for n, v in t.items()}
    y = torch.empty(rows, k, device="cuda")
    plan = fc.GatedFeedForward(rows, k, f, dtype="fp32", ctx=lctx)
    torch.cuda.synchronize()
    plan.forward(at(t["x"]), at(y), **{n: at(v) for n, v in t.items() if n != "x"})
    done(lctx)
    want = ff({**{n: v.double().cpu() for n, v in t.items()}, "b_gate": None, "b_up": None, "b_down": None}, "silu", "fp32")
    check(y, *want["y"], "fp32", "y")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("kind", ["silu", "gelu_tanh", "sigmoid"])
def test_ff_activations_of_huge_arguments(lctx, rows, dtype, kind):
    """Gates that are exact powers of two, up to 2^100 of either sign: act(z) goes to 0 or z, act'(z) to 0 or 1.

    up and the down matrix are ones and the identity, so that y is act(z), rounded once, and the first column of the gate's
    gradient is act'(z), rounded once.  Beside the half step: the exponential's argument, up to 87 in size where its result
    is one that counts, is off by some four roundings, 2^-15 of the result at most; the types of 16 bits bound the sigmoid at
    2^-60, 64 times of which is 5.6e-17.  act' has 1 - s, off by two steps of 1 where it is not 0, times up to 8 (|z|) in SiLU
    and less in the others: 2^-19."""
    dt = DTYPES[dtype]
    z = [0.0] + [s * 2.0 ** e for s in (1, -1) for e in (-1, 1, 3, 5, 6, 9, 40, 66, 100)]
    f = 64
    z = (z * 4)[:f]
    w_gate, w_up = torch.zeros(f, f), torch.zeros(f, f)
    w_gate[:, 0], w_up[:, 0] = torch.tensor(z), 1.0
    x, dy = torch.zeros(rows, f), torch.zeros(rows, f)
    x[:, 0], dy[rows - 1] = 1.0, 1.0
    x, dy, w_gate, w_up, w_down = (t.to(dt).cuda() for t in (x, dy, w_gate, w_up, torch.eye(f)))
    y, dw, saved = torch.empty_like(x), torch.empty_like(w_gate), torch.empty(2, rows, f, device="cuda")
    plan = fc.GatedFeedForward(rows, f, f, act=kind, dtype=dtype, train=True, ctx=lctx)
    torch.cuda.synchronize()
    ws = {"w_gate": at(w_gate), "w_up": at(w_up), "w_down": at(w_down)}
    plan.forward(at(x), at(y), **ws, saved=at(saved))
    plan.backward(at(dy), at(x), **ws, saved=at(saved), dw_gate=at(dw))
    done(lctx)
    v, d = act(torch.tensor(z, dtype=torch.float64), kind)
    rel = torch.finfo(dt).eps / 2 + 2.0 ** -15
    for got, want, tiny, what in ((y, v.expand(rows, f), 1e-35 if dtype == "fp32" else 1e-16, "y"), (dw[:, 0], d, 2.0 ** -19, "dw_gate")):
        off = (got.double().cpu() - want).abs()
        assert bool((off <= rel * want.abs() + tiny).all()), (what, off.max())


def test_a_nan_stays_in_its_row(lctx):
    rows, k, f = 300, 64, 128
    for dtype in ("fp32", "bf16"):
        dt = DTYPES[dtype]
        g = gen(91)
        x = torch.randn(rows, k, generator=g).to(dt).cuda()
        x[137, 5] = float("nan")
        x[299, 63] = float("inf")
        w = {n: (0.1 * torch.randn(*s, generator=g)).to(dt).cuda() for n, s in
             (("w_gate", (f, k)), ("w_up", (f, k)), ("w_down", (k, f)))}
        y = torch.empty_like(x)
        plan = fc.GatedFeedForward(rows, k, f, dtype=dtype, ctx=lctx)
        torch.cuda.synchronize()
        plan.forward(at(x), at(y), **{n: at(v) for n, v in w.items()})
        done(lctx)
        bad = ~torch.isfinite(y)
        assert bool(torch.isnan(y[137]).all()) and bool(bad[299].all()) and int(bad.sum()) == 2 * k


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_training_step_replayed_from_a_graph(lctx, dtype):
    """Norm and block, forward and backward, captured once and replayed on other inputs: the bits of the calls."""
    n, p, c, f, groups = 3, 150, 64, 136, 8
    dt = DTYPES[dtype]
    g = gen(101)
    rnd = lambda *s: (0.5 * torch.randn(*s, generator=g)).to(dt).cuda()  # noqa: E731
    x, dy, w = rnd(n * p, c), rnd(n * p, c), {"w_gate": rnd(f, c), "w_up": rnd(f, c), "w_down": rnd(c, f)}
    gamma, beta = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    mean, rstd, saved = torch.empty(n, groups, device="cuda"), torch.empty(n, groups, device="cuda"), torch.empty(2, n * p, f, device="cuda")
    outs = {"mid": torch.empty_like(x), "y": torch.empty_like(x), "dmid": torch.empty_like(x), "dx": torch.empty_like(x),
            "dgamma": torch.empty_like(gamma), "dbeta": torch.empty_like(beta), **{"d" + k: torch.empty_like(v) for k, v in w.items()}}
    gn = fc.GroupNorm(n, p, c, groups, act="gelu", dtype=dtype, ctx=lctx)
    block = fc.GatedFeedForward(n * p, c, f, dtype=dtype, train=True, ctx=lctx)

    def step():
        gn.forward(at(x), at(outs["mid"]), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd))
        block.forward(at(outs["mid"]), at(outs["y"]), **{k: at(v) for k, v in w.items()}, saved=at(saved))
        block.backward(at(dy), at(outs["mid"]), at(outs["dmid"]), **{k: at(v) for k, v in w.items()}, saved=at(saved),
                       **{"d" + k: at(outs["d" + k]) for k in w})
        gn.backward(at(outs["dmid"]), at(x), at(outs["dx"]), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd),
                    dgamma=at(outs["dgamma"]), dbeta=at(outs["dbeta"]))

    stream, graph = torch.cuda.ExternalStream(lctx.stream.value), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(2):
        x.copy_(rnd(n * p, c))
        torch.cuda.synchronize()
        step()
        done(lctx)
        called = {k: v.clone() for k, v in outs.items()}
        for v in outs.values():
            v.fill_(GUARD)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        done(lctx)
        for k, v in outs.items():
            assert torch.equal(v, called[k]), k
    del graph


def test_norm_of_very_many_images(lctx):
    """More images than a launch has rows of blocks."""
    run_norm(lctx, 70000, 4, 8, 2, "silu", "fp32")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("k", [64, 65])
def test_what_lies_between_rows_does_not_matter(lctx, dtype, k):
    """NaN between the channels of the maps: the same bits as from maps without gaps, in the block and in the norm."""
    rows, f, wide = 200, 72, 80
    dt = DTYPES[dtype]
    g = gen(111)
    rnd = lambda *s: (0.5 * torch.randn(*s, generator=g)).to(dt).cuda()  # noqa: E731
    x, dy = rnd(rows, k), rnd(rows, k)
    w = {"w_gate": rnd(f, k), "w_up": rnd(f, k), "w_down": rnd(k, f)}
    gapped = {n: torch.full((rows, wide), float("nan"), dtype=dt, device="cuda") for n in ("x", "dy", "y", "dx", "n", "ndx")}
    gapped["x"][:, :k], gapped["dy"][:, :k] = x, dy
    results = []
    for stride, t in ((0, {"x": x, "dy": dy, **{n: torch.empty_like(x) for n in ("y", "dx", "n", "ndx")}}), (wide, gapped)):
        saved, mean, rstd = torch.empty(2, rows, f, device="cuda"), torch.empty(2, 1, device="cuda"), torch.empty(2, 1, device="cuda")
        grads = {"d" + n: torch.empty_like(v) for n, v in w.items()}
        block = fc.GatedFeedForward(rows, k, f, dtype=dtype, x_stride=stride, y_stride=stride, train=True, ctx=lctx)
        gn = fc.GroupNorm(2, rows // 2, k, 1, act="silu", dtype=dtype, x_stride=stride, y_stride=stride, ctx=lctx)
        dgamma, dbeta = torch.empty(2, k, device="cuda")
        torch.cuda.synchronize()
        block.forward(at(t["x"]), at(t["y"]), **{n: at(v) for n, v in w.items()}, saved=at(saved))
        block.backward(at(t["dy"]), at(t["x"]), at(t["dx"]), **{n: at(v) for n, v in w.items()}, saved=at(saved),
                       **{n: at(v) for n, v in grads.items()})
        gn.forward(at(t["x"]), at(t["n"]), mean=at(mean), rstd=at(rstd))
        gn.backward(at(t["dy"]), at(t["x"]), at(t["ndx"]), mean=at(mean), rstd=at(rstd), dgamma=at(dgamma), dbeta=at(dbeta))
        done(lctx)
        for n in ("y", "dx", "n", "ndx"):
            assert torch.isnan(t[n][:, k:]).all()
        results.append([t[n][:, :k].clone() for n in ("y", "dx")] + list(grads.values()))
        norms = [t["n"][:, :k], t["ndx"][:, :k], dgamma, dbeta, mean, rstd]
        assert all(bool(torch.isfinite(v).all()) for v in norms)
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_two_contexts_at_once(lctx):
    """Calls of two contexts overlap on the GPU; each has its own stream and workspaces, and gets the bits it gets alone."""
    other = fc.Context(0, arena_bytes=512 << 20)
    try:
        g = gen(121)
        jobs = []
        for ctx, (rows, k, f) in ((lctx, (3000, 256, 520)), (other, (2000, 320, 264))):
            t = {"x": torch.randn(rows, k, generator=g).cuda().bfloat16()}
            for n, s in (("w_gate", (f, k)), ("w_up", (f, k)), ("w_down", (k, f))):
                t[n] = (0.05 * torch.randn(*s, generator=g)).cuda().bfloat16()
            jobs.append((fc.GatedFeedForward(rows, k, f, dtype="bf16", ctx=ctx), fc.GroupNorm(4, rows // 4, k, 8, act="silu", dtype="bf16", ctx=ctx),
                         t, torch.empty_like(t["x"]), torch.empty_like(t["x"])))

        def run(job):
            plan, gn, t, mid, y = job
            gn.forward(at(t["x"]), at(mid))
            plan.forward(at(mid), at(y), **{n: at(v) for n, v in t.items() if n != "x"})

        torch.cuda.synchronize()
        alone = []
        for job in jobs:
            run(job)
            lctx.synchronize()
            other.synchronize()
            alone.append(job[4].clone())
            job[4].fill_(GUARD)
        torch.cuda.synchronize()
        for _ in range(20):
            for job in jobs:
                run(job)
        lctx.synchronize()
        other.synchronize()
        assert all(torch.equal(job[4], a) for job, a in zip(jobs, alone))
    finally:
        other.close()
