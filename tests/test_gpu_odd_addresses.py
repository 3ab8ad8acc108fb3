"""Operands of the block and the norm that begin one element past a 16-byte boundary, one at a time and all at once."""
import pytest
import torch

import fastconv_b200 as fc
from _last_ref import DTYPES, check, ff, norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lctx():
    c = fc.Context(0, arena_bytes=512 << 20)
    yield c
    c.close()


def place(t, odd):
    """The tensor on the GPU, on a 16-byte boundary or one element past it, with a guard of one element on either side."""
    flat = torch.full((t.numel() + 16,), 7.0, dtype=t.dtype, device="cuda")
    first = 9 if odd else 8
    view = flat[first:first + t.numel()].view(t.shape)
    view.copy_(t)
    return flat, view, first


def guarded(placed):
    return all(bool((flat[:first] == 7).all()) and bool((flat[first + view.numel():] == 7).all()) for flat, view, first in placed)


BLOCK = ("x", "dy", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down", "y", "saved", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up",
         "db_down")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_block_operands_at_odd_addresses(lctx, rows, dtype):
    k, f, o, dt = 64, 136, 72, DTYPES[dtype]
    g = torch.Generator().manual_seed(37)
    rnd = lambda *s, by=1.0: (torch.randn(*s, generator=g) * by).to(dt)  # noqa: E731
    t = {"x": rnd(rows, k), "dy": rnd(rows, o), "w_gate": rnd(f, k, by=k ** -0.5), "w_up": rnd(f, k, by=k ** -0.5),
         "w_down": rnd(o, f, by=f ** -0.5), "b_gate": rnd(f, by=0.2), "b_up": rnd(f, by=0.2), "b_down": rnd(o, by=0.2),
         "y": torch.zeros(rows, o, dtype=dt), "saved": torch.zeros(2, rows, f)}
    for name in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"):
        t["d" + name] = torch.zeros_like(t[name])
    want = ff({n: t[n].double() for n in BLOCK[:1] + BLOCK[2:8]}, "silu", dtype, t["dy"].double())
    plan = fc.GatedFeedForward(rows, k, f, o, dtype=dtype, train=True, ctx=lctx)
    for odd in [(name,) for name in BLOCK] + [BLOCK]:
        placed = {n: place(v, n in odd) for n, v in t.items()}
        at = {n: view.data_ptr() for n, (_, view, _) in placed.items()}
        weights = {n: at[n] for n in ("w_gate", "w_up", "w_down")}
        torch.cuda.synchronize()
        plan.forward(at["x"], at["y"], **weights, **{n: at[n] for n in ("b_gate", "b_up", "b_down")}, saved=at["saved"])
        plan.backward(at["dy"], at["x"], at["dx"], **weights, saved=at["saved"], **{n: at[n] for n in BLOCK[11:]})
        lctx.synchronize()
        torch.cuda.synchronize()
        assert guarded(placed.values()), odd
        for n in ("y", *BLOCK[10:]):
            check(placed[n][1], *want[n], dtype, f"{n} with {odd} at odd addresses")


@pytest.mark.parametrize("dtype,params", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
def test_norm_operands_at_odd_addresses(lctx, dtype, params):
    n, p, c, groups, dt, pt = 2, 100, 64, 8, DTYPES[dtype], DTYPES[params]
    g = torch.Generator().manual_seed(41)
    t = {"x": torch.randn(n, p, c, generator=g).to(dt), "dy": torch.randn(n, p, c, generator=g).to(dt),
         "gamma": (1 + 0.2 * torch.randn(c, generator=g)).to(pt), "beta": (0.3 * torch.randn(c, generator=g)).to(pt),
         "y": torch.zeros(n, p, c, dtype=dt), "dx": torch.zeros(n, p, c, dtype=dt), "mean": torch.zeros(n, groups),
         "rstd": torch.zeros(n, groups), "dgamma": torch.zeros(c, dtype=pt), "dbeta": torch.zeros(c, dtype=pt)}
    want = norm(t["x"].double(), groups, 1e-5, t["gamma"].double(), t["beta"].double(), "gelu", dtype, t["dy"].double())
    plan = fc.GroupNorm(n, p, c, groups, act="gelu", dtype=dtype, param_dtype=params, ctx=lctx)
    for odd in [(name,) for name in t] + [tuple(t)]:
        placed = {k: place(v, k in odd) for k, v in t.items()}
        at = {k: view.data_ptr() for k, (_, view, _) in placed.items()}
        affine = {k: at[k] for k in ("gamma", "beta", "mean", "rstd")}
        torch.cuda.synchronize()
        plan.forward(at["x"], at["y"], **affine)
        plan.backward(at["dy"], at["x"], at["dx"], **affine, dgamma=at["dgamma"], dbeta=at["dbeta"])
        lctx.synchronize()
        torch.cuda.synchronize()
        assert guarded(placed.values()), odd
        for k, kind in (("y", dtype), ("dx", dtype), ("mean", "fp32"), ("rstd", "fp32"), ("dgamma", params), ("dbeta", params)):
            check(placed[k][1], *want[k], kind, f"{k} with {odd} at odd addresses")
