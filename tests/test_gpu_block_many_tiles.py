"""The feed-forward block where a pair of SMs computes several tiles, against the 64-bit reference with its derived bounds (the
reference itself runs on the GPU here: it is elementary operations on doubles)."""
import pytest
import torch

import fastconv_b200 as fc
from fastconv_b200 import _lib
from _last_ref import DTYPES, U, act, act_error, check, ff

pytestmark = pytest.mark.gpu

PAIRS = 74
PRODUCTS = tuple(_lib.FF_PRODUCT_NAMES)
# rows, in, hidden, out; the products with tiles (or shares of them) for more than one round of all pairs, and their widths in the types
# of 16 bits (fp32 has one width, 128)
SHAPES = [((5000, 1032, 4104, 1032), dict.fromkeys(PRODUCTS, 256)),
          ((4999, 1031, 4101, 1029), dict.fromkeys(PRODUCTS, 256)),  # rows that fit no copy: packed operands, results stored by warps
          ((40001, 72, 136, 40), {"gate": 256, "down": 64, "back_gate": 256, "dx": 128}),
          ((40000, 64, 64, 64), {"gate": 128, "down": 64, "back_gate": 128, "dx": 128}),
          ((40003, 40, 24, 72), {"gate": 64, "down": 128, "back_gate": 128, "dx": 128})]


@pytest.fixture(scope="module")
def lctx():
    c = fc.Context(0, arena_bytes=4 << 30)
    yield c
    c.close()


def at(t):
    return 0 if t is None else t.data_ptr()


def by_place(saved, rows, cols):
    """One half of `saved` -> [rows][cols]: blocks of 32 rows ordered [4 columns][row][column], the last block with fewer rows, and
    plain rows where the columns are no multiple of 4."""
    flat = saved.flatten()
    if cols % 4:
        return flat.view(rows, cols)
    out, whole = torch.empty(rows, cols, device=saved.device), rows // 32 * 32
    out[:whole] = flat[:whole * cols].view(-1, cols // 4, 32, 4).permute(0, 2, 1, 3).reshape(whole, cols)
    if rows > whole:
        out[whole:] = flat[whole * cols:].view(cols // 4, rows - whole, 4).permute(1, 0, 2).reshape(rows - whole, cols)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape,widths", SHAPES, ids=["x".join(map(str, s)) for s, _ in SHAPES])
def test_block_of_several_tiles_a_pair(lctx, shape, widths, dtype):
    rows, k, f, o = shape
    dt = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(17)
    rnd = lambda *s, by=1.0: (torch.randn(*s, generator=g, device="cuda") * by).to(dt)  # noqa: E731
    plan = fc.GatedFeedForward(rows, k, f, o, act="silu", dtype=dtype, train=True, ctx=lctx)
    for name, width in widths.items():
        cut = plan.product_plan(name)
        assert cut.tile_columns == (128 if dtype == "fp32" else width), name
        assert cut.tiles * cut.shares > PAIRS, name
    t = {"x": rnd(rows, k), "w_gate": rnd(f, k, by=k ** -0.5), "w_up": rnd(f, k, by=k ** -0.5), "w_down": rnd(o, f, by=f ** -0.5),
         "b_gate": rnd(f, by=0.2), "b_up": rnd(f, by=0.2), "b_down": rnd(o, by=0.2)}
    dy = rnd(rows, o)
    weights = {n: at(t[n]) for n in ("w_gate", "w_up", "w_down")}
    runs = []
    for _ in range(2):
        y, saved = torch.empty_like(dy), torch.full((2, rows, f), 7.0, device="cuda")
        grads = {n: torch.full_like(v, 7.0) for n, v in t.items()}
        torch.cuda.synchronize()
        plan.forward(at(t["x"]), at(y), **weights, **{n: at(t[n]) for n in ("b_gate", "b_up", "b_down")}, saved=at(saved))
        plan.backward(at(dy), at(t["x"]), **weights, saved=at(saved), **{"d" + n: at(v) for n, v in grads.items()})
        lctx.synchronize()
        torch.cuda.synchronize()
        runs.append({"y": y, "gate": by_place(saved[0], rows, f), "up": by_place(saved[1], rows, f),
                     **{"d" + n: v for n, v in grads.items()}})
    plan.release()
    want = ff({n: v.double() for n, v in t.items()}, "silu", dtype, dy.double())
    for name, value in runs[0].items():
        check(value, want[name][0].cpu(), want[name][1].cpu(), "fp32" if name in ("gate", "up") else dtype, name)
        assert torch.equal(value, runs[1][name]), name  # bit for bit again


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,f", [(1, 8), (5, 64), (8, 36), (33, 64), (70, 65), (200, 136)])
def test_saved_values_lie_where_they_should(lctx, rows, f, dtype):
    """Place by place, not as a set: from the kernels of few rows and from the tensor cores'."""
    k, dt = 64, DTYPES[dtype]
    g = torch.Generator().manual_seed(23)
    t = {"x": torch.randn(rows, k, generator=g), "w_gate": torch.randn(f, k, generator=g) / 8, "w_up": torch.randn(f, k, generator=g) / 8,
         "w_down": torch.randn(k, f, generator=g) / 8}
    t = {n: v.to(dt).cuda() for n, v in t.items()}
    y, saved = torch.empty_like(t["x"]), torch.full((2, rows, f), 7.0, device="cuda")
    plan = fc.GatedFeedForward(rows, k, f, dtype=dtype, ctx=lctx)
    torch.cuda.synchronize()
    plan.forward(at(t["x"]), at(y), **{n: at(v) for n, v in t.items() if n != "x"}, saved=at(saved))
    lctx.synchronize()
    want = ff({**{n: v.double().cpu() for n, v in t.items()}, "b_gate": None, "b_up": None, "b_down": None}, "silu", dtype)
    for name, half in zip(("gate", "up"), saved):
        check(by_place(half, rows, f), *want[name], "fp32", name)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,k,f,o", [(1, 8, 16, 256), (2, 16, 64, 64), (4, 64, 64, 40), (8, 32, 40, 128)])
def test_blocks_of_few_rows_round_once(lctx, rows, k, f, o, dtype):
    """Nothing is rounded to 16 bits before the result: the bound is that of the two products' fp32 sums, short ones here so that it is
    small, and one half step."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(29)
    rnd = lambda *s, by=1.0: (torch.randn(*s, generator=g) * by).to(dt)  # noqa: E731
    x, wg, wu, wd = rnd(rows, k), rnd(f, k, by=k ** -0.5), rnd(f, k, by=k ** -0.5), rnd(o, f, by=f ** -0.5)
    on = {n: v.cuda() for n, v in (("x", x), ("w_gate", wg), ("w_up", wu), ("w_down", wd))}
    y = torch.empty(rows, o, dtype=dt, device="cuda")
    plan = fc.GatedFeedForward(rows, k, f, o, dtype=dtype, ctx=lctx)
    torch.cuda.synchronize()
    plan.forward(at(on["x"]), at(y), **{n: at(v) for n, v in on.items() if n != "x"})
    lctx.synchronize()
    x, wg, wu, wd = (v.double() for v in (x, wg, wu, wd))
    gate, up = x @ wg.t(), x @ wu.t()
    e_gate, e_up = ((k + 4) * U * (x.abs() @ w.t().abs()) for w in (wg, wu))
    a, e_a = act(gate, "silu")[0], act_error(gate, e_gate, "silu")[0]
    h = a * up
    e_h = 1.05 * (e_a * up.abs() + a.abs() * e_up + e_a * e_up) + U * h.abs()
    check(y, h @ wd.t(), e_h @ wd.t().abs() + (f + 4) * U * (h.abs() @ wd.t().abs()), dtype, "y")
