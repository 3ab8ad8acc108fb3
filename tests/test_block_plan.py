"""What the feed-forward block's products are cut into: asked on the host."""
import ctypes as C

import pytest

import fastconv_b200 as fc
from fastconv_b200 import _lib
from fastconv_b200._lib import FfProductPlan, GatedFfDesc


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("product", list(_lib.FF_PRODUCT_NAMES))
def test_plans_cover_their_products(dtype, product):
    lib, plan = fc.load(), FfProductPlan()
    for rows, k, f, o in ((1, 8, 8, 8), (196, 1024, 4096, 1024), (5000, 1032, 4104, 1031), (50176, 512, 2048, 512)):
        d = GatedFfDesc(rows, k, f, o, dtype, 2, 0, 0)
        assert lib.fc_gated_ff_plan(C.byref(d), _lib.FF_PRODUCT_NAMES[product], C.byref(plan)) == 0
        assert plan.tile_columns in ((128,) if dtype == 0 else (64, 128, 256)) and 1 <= plan.shares <= 16
        m, n, reduction = {"gate": (rows, 2 * f, k), "down": (rows, o, f), "back_gate": (rows, f, o), "dx": (rows, k, 2 * f),
                           "dw_in": (2 * f, k, rows), "dw_down": (o, f, rows)}[product]
        assert plan.tiles * 256 * plan.tile_columns >= m * n
        assert plan.shares == 1 or (plan.shares <= (reduction + 63) // 64 and product not in ("gate", "back_gate"))


def test_plans_that_are_refused():
    lib, plan, d = fc.load(), FfProductPlan(), GatedFfDesc(4, 8, 16, 8, 0, 2, 0, 0)
    invalid = _lib.FC_ERR_INVALID_ARG
    assert lib.fc_gated_ff_plan(C.byref(d), 0, C.byref(plan)) == 0
    for product in (-1, 6):
        assert lib.fc_gated_ff_plan(C.byref(d), product, C.byref(plan)) == invalid
    assert lib.fc_gated_ff_plan(C.byref(d), 0, None) == invalid
    assert lib.fc_gated_ff_plan(None, 0, C.byref(plan)) == invalid
    assert lib.fc_gated_ff_plan(C.byref(GatedFfDesc(0, 8, 16, 8, 0, 2, 0, 0)), 0, C.byref(plan)) == invalid
