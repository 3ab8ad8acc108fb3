"""Group norm over slices of wider maps gives the bits that it gives over the same map without gaps."""
import pytest
import torch

import fastconv_b200 as fc
from _last_ref import DTYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lctx():
    c = fc.Context(0, arena_bytes=512 << 20)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("batch,pixels,channels,groups", [(2, 100, 64, 1), (2, 100, 65, 1), (3, 333, 80, 5), (1, 20000, 64, 2)])
@pytest.mark.parametrize("gap_x,gap_y", [(16, 0), (0, 16), (8, 24)])
def test_norm_has_the_same_bits_with_and_without_gaps(lctx, dtype, batch, pixels, channels, groups, gap_x, gap_y):
    """The gaps keep every row on its 16-byte boundary or, with 65 channels, off it both times: one width of vectors, so one order
    of sums.  What lies in them is NaN and stays so; neighbouring rows are other values, so a wrong stride shows."""
    rows, dt = batch * pixels, DTYPES[dtype]
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, dy = rnd(rows, channels).to(dt).cuda(), rnd(rows, channels).to(dt).cuda()
    gamma, beta = (1 + 0.1 * rnd(channels)).cuda(), rnd(channels).cuda()
    results = []
    for gx, gy in ((0, 0), (gap_x, gap_y)):
        wide = {n: torch.full((rows, channels + gap), float("nan"), dtype=dt, device="cuda")
                for n, gap in (("x", gx), ("dx", gx), ("dy", gy), ("y", gy))}
        wide["x"][:, :channels], wide["dy"][:, :channels] = x, dy
        mean, rstd = torch.empty(2, batch, groups, device="cuda")
        dgamma, dbeta = torch.empty(2, channels, device="cuda")
        plan = fc.GroupNorm(batch, pixels, channels, groups, act="silu", dtype=dtype, x_stride=channels + gx, y_stride=channels + gy, ctx=lctx)
        torch.cuda.synchronize()
        p = {n: t.data_ptr() for n, t in (*wide.items(), ("gamma", gamma), ("beta", beta), ("mean", mean), ("rstd", rstd))}
        affine = {n: p[n] for n in ("gamma", "beta", "mean", "rstd")}
        plan.forward(p["x"], p["y"], **affine)
        plan.backward(p["dy"], p["x"], p["dx"], **affine, dgamma=dgamma.data_ptr(), dbeta=dbeta.data_ptr())
        lctx.synchronize()
        torch.cuda.synchronize()
        for t in wide.values():
            assert torch.isnan(t[:, channels:]).all()
        results.append([wide["y"][:, :channels], wide["dx"][:, :channels], mean, rstd, dgamma, dbeta])
        plan.release()
    for name, a, b in zip(("y", "dx", "mean", "rstd", "dgamma", "dbeta"), *results):
        assert torch.isfinite(a).all() and torch.equal(a, b), name
