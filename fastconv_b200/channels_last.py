"""Channels-last operators over the C ABI: group norm with an activation, the gated feed-forward block, and the moves
between a convolution layer's NCHW maps and channels-last ones.

Addresses are device pointers as integers (`Context.alloc`, or any allocation on the context's GPU); 0 stands for an
operand that is absent.  Calls run asynchronously on the context's stream, in the order in which they are made; work of
other streams that makes or reads the maps has to be ordered with that stream by the caller.  A plan (`GroupNorm`,
`GatedFeedForward`) fixes the shape and holds the workspace, so one plan's calls must not overlap: that is so by itself
on the one stream, and has to be seen to when graphs captured from it are replayed on several.

The reference has no operator of this kind; `act`, `dtype` and the layouts are those of include/fastconv_b200.h.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib
from ._lib import FfProductPlan, GatedFfDesc, GroupNormDesc, check
from .layers import Context, default_context


def _named(names: dict, what: str, value):
    if value not in names:
        raise ValueError(f"{what} {value!r}: one of {', '.join(names)}")
    return names[value]


def to_channels_last(src: int, dst: int, batch: int, channels: int, pixels: int, *, dtype: str = "fp32", stride: int = 0,
                     ctx: Optional[Context] = None) -> None:
    """fp32 [batch][channels][pixels] at `src` -> [batch][pixels][channels] in `dtype` at `dst`; `stride`: elements from one
    pixel of `dst` to the next (0 = channels)."""
    ctx = ctx or default_context()
    check(ctx._lib.fc_map_to_channels_last(ctx.handle, src, dst, batch, channels, pixels, stride,
                                           _named(_lib.DTYPE_NAMES, "dtype", dtype)), "fc_map_to_channels_last")


def from_channels_last(src: int, dst: int, batch: int, channels: int, pixels: int, *, dtype: str = "fp32", stride: int = 0,
                       ctx: Optional[Context] = None) -> None:
    """The way back: [batch][pixels][channels] in `dtype` at `src` -> fp32 [batch][channels][pixels] at `dst`."""
    ctx = ctx or default_context()
    check(ctx._lib.fc_map_from_channels_last(ctx.handle, src, dst, batch, channels, pixels, stride,
                                             _named(_lib.DTYPE_NAMES, "dtype", dtype)), "fc_map_from_channels_last")


class _Plan:
    """A shape, the context it runs on, and its workspace in the context's arena."""

    def _take(self, ctx: Optional[Context], size_of, desc, backward: bool) -> None:
        self.ctx = ctx or default_context()
        self._lib = self.ctx._lib
        self.desc = desc
        self._ref = C.byref(desc)
        sizes = C.c_size_t(), C.c_size_t()
        check(size_of(self._ref, C.byref(sizes[0]), C.byref(sizes[1])), size_of.__name__)
        self.workspace_bytes = max(sizes[0].value, sizes[1].value if backward else 0)
        self._workspace = self.ctx.alloc(self.workspace_bytes) if self.workspace_bytes else 0
        self.ctx.adopt(self)

    def release(self) -> None:
        """Gives the workspace back.  Work already enqueued is safe: later users of the arena follow it on the stream.  A graph
        that has captured a call writes to that workspace whenever it is replayed, so the plan has to outlive it."""
        if getattr(self, "_workspace", 0):
            self.ctx.free(self._workspace)
        self._workspace = 0
        self._lib = None

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    def _ready(self):
        if self._lib is None:
            raise RuntimeError("the plan is released")
        return self._lib


class GroupNorm(_Plan):
    """y = act(gamma (x - mean) / sqrt(var + eps) + beta) over channels-last maps [batch][pixels][channels]."""

    def __init__(self, batch: int, pixels: int, channels: int, groups: int, *, eps: float = 1e-5, act: str = "none",
                 dtype: str = "fp32", param_dtype: str = "fp32", x_stride: int = 0, y_stride: int = 0, ctx: Optional[Context] = None):
        self._workspace, self._lib = 0, None
        desc = GroupNormDesc(batch, pixels, channels, groups, _named(_lib.DTYPE_NAMES, "dtype", dtype),
                             _named(_lib.DTYPE_NAMES, "param_dtype", param_dtype), _named(_lib.ACT_NAMES, "act", act), eps, x_stride,
                             y_stride)
        self._take(ctx, _lib.load().fc_group_norm_workspace, desc, True)

    def forward(self, x: int, y: int, *, gamma: int = 0, beta: int = 0, mean: int = 0, rstd: int = 0) -> None:
        """`mean`, `rstd`: fp32 [batch][groups] that the backward pass will need (0 = not wanted)."""
        check(self._ready().fc_group_norm_forward(self.ctx.handle, self._ref, x, gamma, beta, y, mean, rstd, self._workspace,
                                                  self.workspace_bytes), "fc_group_norm_forward")

    def backward(self, dy: int, x: int, dx: int = 0, *, mean: int, rstd: int, gamma: int = 0, beta: int = 0, dgamma: int = 0,
                 dbeta: int = 0) -> None:
        check(self._ready().fc_group_norm_backward(self.ctx.handle, self._ref, dy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta,
                                                   self._workspace, self.workspace_bytes), "fc_group_norm_backward")


class GatedFeedForward(_Plan):
    """y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd over the rows of a channels-last map.

    Weights are those of 1x1 convolutions: w_gate, w_up [hidden][in_channels], w_down [out_channels][hidden].  `train`
    takes the backward pass's workspace too."""

    def __init__(self, rows: int, in_channels: int, hidden: int, out_channels: Optional[int] = None, *, act: str = "silu",
                 dtype: str = "bf16", x_stride: int = 0, y_stride: int = 0, train: bool = False, ctx: Optional[Context] = None):
        self._workspace, self._lib = 0, None
        self.train = train
        desc = GatedFfDesc(rows, in_channels, hidden, in_channels if out_channels is None else out_channels,
                           _named(_lib.DTYPE_NAMES, "dtype", dtype), _named(_lib.ACT_NAMES, "act", act), x_stride, y_stride)
        self._take(ctx, _lib.load().fc_gated_ff_workspace, desc, train)

    def product_plan(self, product: str):
        """What "gate", "down", "back_gate", "dx", "dw_in" or "dw_down" is cut into on the tensor cores: `tile_columns`, `shares` of
        the reduction and `tiles`."""
        plan = FfProductPlan()
        check(self._ready().fc_gated_ff_plan(self._ref, _named(_lib.FF_PRODUCT_NAMES, "product", product), C.byref(plan)),
              "fc_gated_ff_plan")
        return plan

    def forward(self, x: int, y: int, *, w_gate: int, w_up: int, w_down: int, b_gate: int = 0, b_up: int = 0, b_down: int = 0,
                saved: int = 0) -> None:
        """`saved`: 2 * rows * hidden floats, whatever the type, that the backward pass will need (0 = not wanted)."""
        check(self._ready().fc_gated_ff_forward(self.ctx.handle, self._ref, x, w_gate, w_up, w_down, b_gate, b_up, b_down, y,
                                                saved, self._workspace, self.workspace_bytes), "fc_gated_ff_forward")

    def backward(self, dy: int, x: int, dx: int = 0, *, w_gate: int, w_up: int, w_down: int, saved: int, dw_gate: int = 0,
                 dw_up: int = 0, dw_down: int = 0, db_gate: int = 0, db_up: int = 0, db_down: int = 0) -> None:
        if not self.train:
            raise RuntimeError("the plan was made without train=True: it has no workspace for the backward pass")
        check(self._ready().fc_gated_ff_backward(self.ctx.handle, self._ref, dy, x, w_gate, w_up, w_down, saved, dx, dw_gate,
                                                 dw_up, dw_down, db_gate, db_up, db_down, self._workspace,
                                                 self.workspace_bytes), "fc_gated_ff_backward")
