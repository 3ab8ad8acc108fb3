"""GELU far from zero, held to act(z) itself and not to z: gates and betas that are exact values from -12 to 12.

The bound.  Beside the half step of the stored type: exp(-z^2 / 2) has an argument of up to 104 in powers of two, off by three
roundings of its own size, 72 * 3 * 2^-24 of the result; erfc's scaled argument z / sqrt 2 by two, which z^2 multiplies, 144 * 2^-23;
the exponential, the fit or the library's erfc and the products by less than 2^-18.  Together under 2^-15 of the value, and of
|cdf| + |z density| where the two parts of the slope cancel."""
import math

import pytest
import torch

import fastconv_b200 as fc
from _last_ref import DTYPES

pytestmark = pytest.mark.gpu

REL = 2.0 ** -15


@pytest.fixture(scope="module")
def lctx():
    c = fc.Context(0, arena_bytes=512 << 20)
    yield c
    c.close()


def at(t):
    return t.data_ptr()


def gelu(z):
    """act(z), act'(z), |cdf| + |z density|"""
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    density = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z * cdf, cdf + z * density, cdf + (z * density).abs()


def half_step(value, dtype):
    f = torch.finfo(DTYPES[dtype])
    return torch.maximum(f.eps / 2 * value.abs(), torch.full_like(value, f.smallest_normal * f.eps / 2))


def done(ctx):
    ctx.synchronize()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [1, 200])
def test_block_gelu_of_exact_gates(lctx, dtype, rows):
    """up and the down matrix are ones and the identity: y is act(z) rounded once, the gate's gradient act'(z) rounded once."""
    f, dt = 256, DTYPES[dtype]
    z = torch.linspace(-12, 12, f).to(dt)
    w_gate, w_up = torch.zeros(f, f), torch.zeros(f, f)
    w_gate[:, 0], w_up[:, 0] = z.float(), 1.0
    x, dy = torch.zeros(rows, f), torch.zeros(rows, f)
    x[:, 0], dy[rows - 1] = 1.0, 1.0
    x, dy, w_gate, w_up, w_down = (t.to(dt).cuda() for t in (x, dy, w_gate, w_up, torch.eye(f)))
    y, dw, saved = torch.empty_like(x), torch.empty_like(w_gate), torch.empty(2, rows, f, device="cuda")
    plan = fc.GatedFeedForward(rows, f, f, act="gelu", dtype=dtype, train=True, ctx=lctx)
    torch.cuda.synchronize()
    ws = {"w_gate": at(w_gate), "w_up": at(w_up), "w_down": at(w_down)}
    plan.forward(at(x), at(y), **ws, saved=at(saved))
    plan.backward(at(dy), at(x), **ws, saved=at(saved), dw_gate=at(dw))
    done(lctx)
    a, d, parts = gelu(z.double())
    # fp32 has a smallest normal number too: products below it come out as zero
    tiny = 2.0 ** -120
    off = (y.double().cpu() - a).abs()
    assert (off / (half_step(a, dtype) + REL * a.abs() + tiny)).max().item() <= 1
    off = (dw[:, 0].double().cpu() - d).abs()
    assert (off / (half_step(d, dtype) + REL * parts + tiny)).max().item() <= 1


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("channels,groups", [(64, 8), (64, 16), (36, 3)])  # whole vectors, vectors across groups, single elements
def test_norm_gelu_of_exact_betas(lctx, dtype, channels, groups):
    """gamma is zero: y is act(beta) rounded once; one pixel's dy is one: dbeta is act'(beta) in fp32."""
    n, p, dt = 1, 40, DTYPES[dtype]
    z = torch.linspace(-12, 12, channels)
    x = torch.randn(n, p, channels, generator=torch.Generator().manual_seed(3)).to(dt).cuda()
    dy = torch.zeros_like(x)
    dy[0, 17] = 1.0
    gamma, beta = torch.zeros(channels, device="cuda"), z.cuda()
    y, mean, rstd = torch.empty_like(x), torch.empty(groups, device="cuda"), torch.empty(groups, device="cuda")
    dbeta = torch.empty(channels, device="cuda")
    plan = fc.GroupNorm(n, p, channels, groups, act="gelu", dtype=dtype, ctx=lctx)
    torch.cuda.synchronize()
    plan.forward(at(x), at(y), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd))
    plan.backward(at(dy), at(x), gamma=at(gamma), beta=at(beta), mean=at(mean), rstd=at(rstd), dbeta=at(dbeta))
    done(lctx)
    a, d, parts = gelu(z.double())
    tiny = 2.0 ** -120
    off = (y[0].double().cpu() - a).abs()
    assert (off / (half_step(a, dtype) + REL * a.abs() + tiny)).max().item() <= 1
    off = (dbeta.double().cpu() - d).abs()
    assert (off / (REL * parts + tiny)).max().item() <= 1
