"""GPU tests of the example layer (examples/long_conv_layer.py) in two parts, each with a bound
that a subtle fault does not pass: the layer around the 4-bit calls, with projections that do not
round, against the same layer in 64 bits; and every 4-bit call that it makes, on the very
arguments that it makes it with."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest

import mx4_reference as R
from test_gpu_mx4_layer import exact

pytestmark = pytest.mark.gpu


@pytest.fixture()
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "long_conv_layer.py"
    spec = importlib.util.spec_from_file_location("long_conv_layer_parts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_layer_around_the_calls(dev, example, monkeypatch):
    """Projections in 64 bits; x and Wi are whole numbers, so that v is exact and the cache rounds the
    same v here and there.  What is left is the fp32 transforms (2e-6 each, two in a row at most) and
    roundings to fp32 between: within 1e-5 in norm."""
    import torch
    torch.manual_seed(7)
    weights = []

    class Plain:
        def __init__(self, w):
            self.w = torch.randint(-2, 3, w.shape, device=dev).double() if not weights else w.double()
            self.n, self.k = w.shape
            weights.append(self.w)

        def __call__(self, x):
            return (x.double() @ self.w.t().contiguous()).float()

        tokens = __call__

        def gradients(self, x, dy):
            return (dy.double() @ self.w).float(), (dy.double().t().contiguous() @ x.double()).float()

    monkeypatch.setattr(example, "Projection", Plain)
    layer = example.LongConvLayer(width=200, channels=96, longest=300, page=16)
    wi, wo = weights
    x = torch.randint(-3, 4, (2, 257, 200), device=dev).float()
    more = torch.randint(-3, 4, (2, 200), device=dev).float()

    def rounded(x_):
        """The layer on what the cache holds of v."""
        v, g = (x_.double() @ wi.t()).split(96, dim=2)
        flat = v.reshape(-1, 96).cpu().numpy()
        v = torch.from_numpy(R.values(*R.quantize(flat), 96)).to(dev).view_as(v)
        n = 2 * x_.shape[1]
        taps = layer.taps.double()[:x_.shape[1]]
        c = torch.fft.irfft(torch.fft.rfft(v, n=n, dim=1) * torch.fft.rfft(taps, n=n, dim=0), n=n, dim=1)[:, :x_.shape[1]]
        return (c * g) @ wo.t()

    want = rounded(x)
    assert float((layer.prompt(x) - want).norm() / want.norm()) <= 1e-5
    token, last = layer.step(more), rounded(torch.cat((x, more[:, None]), dim=1))[:, -1]
    assert float((token - last).norm() / last.norm()) <= 1e-5
    # the gradients take v as it is
    x64 = x.double().requires_grad_()
    wi.requires_grad_(), wo.requires_grad_()
    dout = torch.randn(2, 257, 200, device=dev)
    refs = torch.autograd.grad((exact(torch, x64, wi, wo, layer.taps.double()) * dout.double()).sum(), (x64, wi, wo))
    wi.requires_grad_(False), wo.requires_grad_(False)
    for got, ref in zip(layer.gradients(x, dout), refs):
        assert float((got - ref).norm() / ref.norm()) <= 1e-5


def host(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def test_calls_of_the_layer(dev, example, monkeypatch):
    """Each call's outputs from its own inputs: codes, scales and what is read back for equality,
    sums within the bound of fp32 summation."""
    import torch
    ff = example.ff
    seen = {}

    def checked(name, check):
        call = getattr(ff, name)

        def wrapped(*a, **kw):
            before = [t.clone() if isinstance(t, torch.Tensor) else t for t in a]
            call(*a, **kw)
            torch.cuda.synchronize()
            check(before, a, kw)
            seen[name] = seen.get(name, 0) + 1
        monkeypatch.setattr(ff, name, wrapped)

    def quantize(before, a, kw):
        x = host(a[0])
        rand = kw.get("rand")
        rand = None if rand is None else host(rand)
        pairs = list(a[1:]) + [None] * (5 - len(a))
        for codes, scales, v, r in ((pairs[0], pairs[1], x, rand), (pairs[2], pairs[3], x.T, None if rand is None else rand.T)):
            if codes is not None:
                want = R.quantize(v, "fit", r)
                assert np.array_equal(host(codes), want[0]) and np.array_equal(host(scales), want[1])

    def product(x, w, out):
        assert R.within(out, x @ w.T, np.abs(x) @ np.abs(w).T, 3 * x.shape[1] + 1, out.dtype)

    def matmul(before, a, kw):
        product(R.values(host(a[0]), host(a[1]), a[5]), R.values(host(a[2]), host(a[3]), a[5]), a[4])

    def linear(before, a, kw):
        x = host(a[0])
        product(x, R.values(host(a[1]), host(a[2]), x.shape[1]), a[3])

    def write(before, a, kw):
        codes, scales = host(before[2]).copy(), host(before[3]).copy()
        want = R.quantize(host(a[0]))
        slots = host(a[1])
        codes.reshape(-1, codes.shape[2])[slots], scales.reshape(-1, scales.shape[2])[slots] = want
        assert np.array_equal(host(a[2]), codes) and np.array_equal(host(a[3]), scales)

    def read(before, a, kw):
        codes, scales, table, lens, out = (host(t) for t in a)
        assert kw == {"order": "channels"}
        for b in range(len(lens)):
            want = np.zeros(out.shape[1:])
            h = R.history(codes, scales, table[b], lens[b], out.shape[1])
            want[:, :len(h)] = h.T
            assert np.array_equal(out[b], want)

    def conv(before, a, kw):
        codes, scales, table, lens, taps = (host(t) for t in a[:5])
        for b in range(len(lens)):
            want, mag = R.conv_step(R.history(codes, scales, table[b], lens[b], taps.shape[1]), taps)
            assert R.within(a[5][b], want, mag, len(taps) + 64, a[5].dtype)

    for name, check in (("quantize", quantize), ("matmul", matmul), ("linear", linear), ("cache_write", write),
                        ("cache_read", read), ("cache_conv", conv)):
        checked("mx4_" + name, check)
    torch.manual_seed(9)
    layer = example.LongConvLayer(width=136, channels=72, longest=150, page=16)
    x = torch.randn(2, 131, 136, device=dev)
    out = layer.prompt(x)
    for _ in range(3):
        layer.step(torch.randn(2, 136, device=dev))
    layer.gradients(x, torch.randn_like(out))
    assert seen == {"mx4_quantize": 2 + 2 + 1 + 4, "mx4_matmul": 2 + 1 + 4, "mx4_linear": 6, "mx4_cache_write": 4,
                    "mx4_cache_read": 1, "mx4_cache_conv": 3}
