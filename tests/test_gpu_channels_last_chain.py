"""Channels-last operators and convolution layers behind one another on a context's stream, without a wait between them."""
import pytest
import torch

import fastconv_b200 as fc
from fastconv_b200._lib import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lctx():
    c = fc.Context(0, arena_bytes=2 << 30)
    yield c
    c.close()


def at(t):
    return t.data_ptr()


def done(ctx):
    ctx.synchronize()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("hw,batch", [(5, 6000), (1, 30000)])
def test_layers_of_few_pixels_wait_for_the_operators_around_them(lctx, dtype, hw, batch):
    """1x1 layers of 24 channels (the kernel of the smallest layers) that read planes which a move has just written, and that
    write planes which a move has just read: the bits of the same calls with a wait after each."""
    c, p = 24, hw * hw
    dt = torch.float32 if dtype == "fp32" else torch.bfloat16
    g = torch.Generator().manual_seed(7)
    x = torch.randn(batch, c, p, generator=g)
    w = (torch.randn(c, c, generator=g) * c ** -0.5).numpy().reshape(c, c, 1, 1)
    layer = fc.ConvIm2colLayer(x.numpy().reshape(batch, c, hw, hw), w, None, None, c, hw, hw, c, 1, 1, 1, 1, 0, 0, 0, 0, 1, False, 1, 1,
                               batch=batch, ctx=lctx)
    layer.Init()
    lib = fc.load()
    rnd = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dt).cuda()  # noqa: E731
    weights = {"w_gate": rnd(40, c), "w_up": rnd(40, c), "w_down": rnd(c, 40)}
    d_in, d_other = x.cuda(), torch.randn(batch, c, p, generator=g).cuda()
    planes, end, out = (torch.zeros(batch, c, p, device="cuda") for _ in range(3))
    a, b, again = (torch.zeros(batch * p, c, dtype=dt, device="cuda") for _ in range(3))
    block = fc.GatedFeedForward(batch * p, c, 40, dtype=dtype, ctx=lctx)
    run = lambda src, dst: check(lib.fc_conv_forward_device(layer._conv, at(src), at(dst)), "layer")  # noqa: E731

    def chain(after=lambda: None):
        for call in (lambda: run(d_in, planes),
                     lambda: fc.to_channels_last(at(planes), at(a), batch, c, p, dtype=dtype, ctx=lctx),
                     lambda: block.forward(at(a), at(b), **{k: at(v) for k, v in weights.items()}),
                     lambda: fc.from_channels_last(at(b), at(end), batch, c, p, dtype=dtype, ctx=lctx),
                     lambda: run(end, out),  # reads what the move writes
                     lambda: fc.to_channels_last(at(out), at(again), batch, c, p, dtype=dtype, ctx=lctx),
                     lambda: run(d_other, out)):  # writes what the move reads
            call()
            after()

    everything = (planes, a, b, end, again, out)
    torch.cuda.synchronize()
    chain(lambda: done(lctx))
    want = [v.clone() for v in everything]
    flat = torch.from_numpy(w.reshape(c, c)).cuda().double()
    exact = torch.einsum("oc,ncp->nop", flat, d_other.double())
    # 24 rounded products and sums in order
    assert bool(((out.double() - exact).abs() <= 48 * 2.0 ** -24 * torch.einsum("oc,ncp->nop", flat.abs(), d_other.double().abs())).all())

    stream, graph = torch.cuda.ExternalStream(lctx.stream.value), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        chain()
    for how in (chain, graph.replay):
        for _ in range(5):
            for v in everything:
                v.fill_(7.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                how()
            done(lctx)
            assert all(torch.equal(u, v) for u, v in zip(everything, want))
    del graph
    layer.release()
