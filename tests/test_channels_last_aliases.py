"""An output of a channels-last operator that is one of its inputs, another output or the workspace is refused on the host."""
import ctypes as C

import pytest

import fastconv_b200 as fc
from fastconv_b200 import _lib
from fastconv_b200._lib import GatedFfDesc, GroupNormDesc

NORM = GroupNormDesc(2, 10, 8, 2, 0, 0, 0, 1e-5, 0, 0)
BLOCK = GatedFfDesc(4, 8, 16, 8, 0, 2, 0, 0)
# name, descriptor, inputs by place, outputs by place (the workspace's last)
CALLS = [("fc_group_norm_forward", NORM, (0, 1, 2), (3, 4, 5, 6)),
         ("fc_group_norm_backward", NORM, (0, 1, 2, 3, 4, 5), (6, 7, 8, 9)),
         ("fc_gated_ff_forward", BLOCK, (0, 1, 2, 3, 4, 5, 6), (7, 8, 9)),
         ("fc_gated_ff_backward", BLOCK, (0, 1, 2, 3, 4, 5), (6, 7, 8, 9, 10, 11, 12, 13))]


@pytest.mark.parametrize("name,desc,inputs,outputs", CALLS, ids=[c[0] for c in CALLS])
def test_an_output_that_is_another_operand_is_refused(name, desc, inputs, outputs):
    """Before the context is looked at (here bytes of zero).  Addresses are never read, and a workspace of no bytes ends the call
    where all of them differ."""
    call, ctx = getattr(fc.load(), name), C.create_string_buffer(1 << 16)
    ops = [4096 * (i + 1) for i in range(len(inputs) + len(outputs))]
    assert call(ctx, C.byref(desc), *ops, 0) == _lib.FC_ERR_INVALID_ARG
    assert b"workspace" in fc.load().fc_last_error()
    for o in outputs:
        for other in inputs + tuple(p for p in outputs if p != o):
            same = list(ops)
            same[o] = ops[other]
            assert call(ctx, C.byref(desc), *same, 0) == _lib.FC_ERR_INVALID_ARG
            assert fc.load().fc_last_error() in (b"an output is an input", b"two outputs are one"), (o, other)


@pytest.mark.parametrize("name", ["fc_map_to_channels_last", "fc_map_from_channels_last"])
def test_a_move_onto_itself_is_refused(name):
    ctx = C.create_string_buffer(1 << 16)
    assert getattr(fc.load(), name)(ctx, 4096, 4096, 1, 4, 4, 0, 0) == _lib.FC_ERR_INVALID_ARG
    assert fc.load().fc_last_error() == b"an output is an input"
