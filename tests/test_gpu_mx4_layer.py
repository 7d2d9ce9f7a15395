"""The example layer (examples/long_conv_layer.py) on the GPU: the calls together, as a model
uses them.

Bounds.  Step form against FFT convolution of the same cache: both in fp32, 2e-6 for
the transforms (this library's fp32 bar) and for the sum, 5e-6 together.  Against the same layer
in 64 bits with unrounded weights and activations: a 4-bit value is off by at most 1/4 of
itself or 1/24 of its block's largest value, in the mean square by less than 0.15 of
the block's for these Gaussian values, so a product of two such factors is within 0.15 sqrt(2)
+ 0.15^2 = 0.24 of its root mean square, and four in a row (input projection with x and Wi,
the cache, the output projection with y and Wo) add in squares to less than 0.5."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "long_conv_layer.py"
    spec = importlib.util.spec_from_file_location("long_conv_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def exact(torch, x, wi, wo, taps):
    """The layer in 64 bits: (out, v, c, g) for x (texts, length, width)."""
    v, g = (x @ wi.t()).split(wi.shape[0] // 2, dim=2)
    n = 2 * x.shape[1]
    f = torch.fft.rfft(v, n=n, dim=1) * torch.fft.rfft(taps[:x.shape[1]], n=n, dim=0)
    c = torch.fft.irfft(f, n=n, dim=1)[:, :x.shape[1]]
    return (c * g) @ wo.t()


def test_layer(dev, example):
    import torch
    torch.manual_seed(5)
    weights = []
    plain = example.Projection.__init__

    def keep(self, w):
        weights.append(w.double())
        plain(self, w)

    example.Projection.__init__ = keep
    try:
        layer = example.LongConvLayer(width=200, channels=96, longest=300, page=16)
    finally:
        example.Projection.__init__ = plain
    wi, wo = weights
    x = torch.randn(2, 257, 200, device=dev)
    out = layer.prompt(x)
    rel = (layer.last() - layer.convolved[:, -1]).norm() / layer.convolved[:, -1].norm()
    assert float(rel) <= 5e-6
    x64 = x.double().requires_grad_()
    wi.requires_grad_(), wo.requires_grad_()
    want = exact(torch, x64, wi, wo, layer.taps.double())
    plain_want = want.detach()
    assert float((out - plain_want).norm() / plain_want.norm()) <= 0.5
    # one more token: the layer on the longer text
    more = torch.randn(2, 200, device=dev)
    token = layer.step(more)
    with torch.no_grad():
        longer = exact(torch, torch.cat((x.double(), more[:, None].double()), dim=1), wi, wo, layer.taps.double())[:, -1]
    assert layer.lens.tolist() == [258, 258]
    assert float((token - longer).norm() / longer.norm()) <= 0.5
    # gradients of sum(dout * out) against autograd in 64 bits: two more products behind each
    dout = torch.randn_like(out)
    grads = layer.gradients(x, dout)
    for got, ref in zip(grads, torch.autograd.grad((want * dout.double()).sum(), (x64, wi, wo))):
        assert float((got - ref).norm() / ref.norm()) <= 0.6


def test_example_runs(dev, example, capsys):
    example.main()
    assert "gradients" in capsys.readouterr().out
