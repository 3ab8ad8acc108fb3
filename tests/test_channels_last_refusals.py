"""What the channels-last operators refuse, and the sizes they report: checked on the host, before anything is launched."""
import ctypes as C

import pytest

import fastconv_b200 as fc
from fastconv_b200 import _lib
from fastconv_b200._lib import GatedFfDesc, GroupNormDesc

INVALID = _lib.FC_ERR_INVALID_ARG


def gn(**kw):
    base = dict(batch=2, pixels=10, channels=8, groups=2, type=0, param_type=0, act=0, eps=1e-5, x_stride=0, y_stride=0)
    base.update(kw)
    return GroupNormDesc(**base)


def ffd(**kw):
    base = dict(rows=4, in_channels=8, hidden=16, out_channels=8, type=0, act=2, x_stride=0, y_stride=0)
    base.update(kw)
    return GatedFfDesc(**base)


@pytest.mark.parametrize("bad", [dict(batch=-1), dict(pixels=0), dict(channels=0), dict(groups=0), dict(groups=3), dict(type=3), dict(type=-1),
                                 dict(param_type=1), dict(act=6), dict(act=-1), dict(eps=-1e-5), dict(eps=float("nan")),
                                 dict(x_stride=7), dict(y_stride=7), dict(x_stride=-8)])
def test_norm_descriptors_that_are_refused(bad):
    f, b = C.c_size_t(), C.c_size_t()
    lib = fc.load()
    assert lib.fc_group_norm_workspace(C.byref(gn()), C.byref(f), C.byref(b)) == 0 and f.value > 0 and b.value > 0
    assert lib.fc_group_norm_workspace(C.byref(gn(**bad)), C.byref(f), C.byref(b)) == INVALID
    assert lib.fc_last_error() != b""


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(in_channels=0), dict(hidden=0), dict(out_channels=-2), dict(type=5), dict(act=9),
                                 dict(x_stride=7), dict(y_stride=-1)])
def test_block_descriptors_that_are_refused(bad):
    f, b = C.c_size_t(), C.c_size_t()
    lib = fc.load()
    assert lib.fc_gated_ff_workspace(C.byref(ffd()), C.byref(f), C.byref(b)) == 0 and 0 < f.value < b.value
    assert lib.fc_gated_ff_workspace(C.byref(ffd(**bad)), C.byref(f), C.byref(b)) == INVALID


def test_null_contexts_and_descriptors_are_refused():
    lib = fc.load()
    assert lib.fc_map_to_channels_last(None, 16, 16, 1, 1, 1, 0, 0) == INVALID
    assert lib.fc_map_from_channels_last(None, 16, 16, 1, 1, 1, 0, 0) == INVALID
    assert lib.fc_group_norm_workspace(None, None, None) == INVALID
    assert lib.fc_gated_ff_workspace(None, None, None) == INVALID
    assert lib.fc_group_norm_forward(None, C.byref(gn()), *[16] * 7, 0) == INVALID
    assert lib.fc_group_norm_backward(None, C.byref(gn()), *[16] * 10, 0) == INVALID
    assert lib.fc_gated_ff_forward(None, C.byref(ffd()), *[16] * 10, 0) == INVALID
    assert lib.fc_gated_ff_backward(None, C.byref(ffd()), *[16] * 14, 0) == INVALID
    assert lib.fc_gated_ff_workspace(C.byref(ffd(hidden=1 << 30)), None, None) == _lib.FC_ERR_UNSUPPORTED


def test_sizes_that_indices_do_not_hold_are_refused():
    lib, unsupported = fc.load(), _lib.FC_ERR_UNSUPPORTED
    assert lib.fc_group_norm_workspace(C.byref(gn(pixels=1 << 30)), None, None) == unsupported
    assert lib.fc_group_norm_workspace(C.byref(gn(channels=1 << 21)), None, None) == unsupported
    assert lib.fc_group_norm_workspace(C.byref(gn(batch=1 << 30, groups=4)), None, None) == unsupported
    for name in ("in_channels", "hidden", "out_channels"):
        assert lib.fc_gated_ff_workspace(C.byref(ffd(**{name: 1 << 30})), None, None) == unsupported


def test_names_are_checked():
    with pytest.raises(ValueError, match="act"):
        fc.GroupNorm(1, 1, 8, 2, act="swish", ctx=object())
    with pytest.raises(ValueError, match="dtype"):
        fc.GatedFeedForward(1, 8, 8, dtype="int8", ctx=object())


def test_sizes_past_32_bits_are_counted():
    f, b = C.c_size_t(), C.c_size_t()
    lib = fc.load()
    assert lib.fc_gated_ff_workspace(C.byref(ffd(rows=1 << 21, hidden=1 << 13, type=1)), C.byref(f), C.byref(b)) == 0
    assert f.value >= (1 << 35) and b.value >= 3 << 35


@pytest.mark.parametrize("batch", [0, 2])
def test_addresses_that_are_no_multiple_of_the_element_are_refused(batch):
    """Before the context is looked at (here bytes of zero): parameters' gradients of no images are written too."""
    lib, ctx = fc.load(), C.create_string_buffer(1 << 16)
    d, p, n = C.byref(gn(batch=batch)), 4096, 1 << 40
    ops = [p, p, p, p, p, p, 2 * p, p, p, p, n]  # dy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta, workspace, bytes
    for i in (2, 3, 4, 5, 7, 8):
        assert lib.fc_group_norm_backward(ctx, d, *[v + 2 if j == i else v for j, v in enumerate(ops)]) == INVALID, i
        assert b"multiple" in lib.fc_last_error(), i
    ops = [p, p, p, 2 * p, p, p, p, n]  # x, gamma, beta, y, mean, rstd, workspace, bytes
    for i in (1, 2, 4, 5) if batch else ():
        assert lib.fc_group_norm_forward(ctx, d, *[v + 2 if j == i else v for j, v in enumerate(ops)]) == INVALID, i
        assert b"multiple" in lib.fc_last_error(), i
    ops = [p, p, p, p, p, p, 2 * p, p, p, p, p, p, p, p, n]  # dy, x, three weights, saved, dx, six gradients, workspace, bytes
    d = C.byref(ffd(rows=2 * batch))
    for i in (5, 7, 8, 9, 10, 11, 12):
        assert lib.fc_gated_ff_backward(ctx, d, *[v + 2 if j == i else v for j, v in enumerate(ops)]) == INVALID, i
        assert b"multiple" in lib.fc_last_error(), i
