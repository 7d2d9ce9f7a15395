"""GPU test: the 4-bit calls without the native binding reach the same kernels, bit for bit."""
import pytest

pytestmark = pytest.mark.gpu


def every_call(torch, ff, dev):
    torch.manual_seed(3)
    m, n, k, page = 20, 40, 300, 4
    x, w = torch.randn(m, k, device=dev), torch.randn(n, k, device=dev).bfloat16()
    bias, rand = torch.randn(n, device=dev), torch.randint(0, 256, (m, k), dtype=torch.uint8, device=dev)
    qx, qt, qw = ff.mx4_empty(m, k), ff.mx4_empty(k, m), ff.mx4_empty(n, k)
    back, y, lin = (torch.empty(*s, device=dev) for s in ((m, k), (m, n), (m, n)))
    ff.mx4_quantize(x, *qx, *qt, rand=rand, rule="floor")
    ff.mx4_quantize(w, *qw)
    ff.mx4_dequantize(*qx, back)
    ff.mx4_matmul(*qx, *qw, y, k, bias=bias)
    ff.mx4_linear(x, *qw, lin, bias=bias)
    c, s = (t.zero_().view(6, page, -1) for t in ff.mx4_empty(6 * page, k))
    ff.mx4_cache_write(x, torch.arange(m, device=dev), c, s)
    table = torch.tensor([[4, 1], [0, 2]], dtype=torch.int32, device=dev)
    lens = torch.tensor([7, 4], dtype=torch.int32, device=dev)
    out, conv = torch.empty(2, k, 8, device=dev), torch.empty(2, k, device=dev).half()
    ff.mx4_cache_read(c, s, table, lens, out, order="channels")
    ff.mx4_cache_conv(c, s, table, lens, torch.randn(8, k, device=dev), conv, work=torch.empty(3, 2, k, device=dev))
    torch.cuda.synchronize()
    kept = [t[:, :k // 2] for t in (qx[0], qw[0])]
    return [back, y, lin, c, s, out, conv, *qt, *kept]


def test_same_without_the_binding(dev, monkeypatch):
    import torch
    import fufft_amd as ff
    assert ff._binding is not None
    want = every_call(torch, ff, dev)
    monkeypatch.setattr(ff, "_binding", None)
    for got, ref in zip(every_call(torch, ff, dev), want):
        assert torch.equal(got, ref)


def test_any_integer_as_k(dev, monkeypatch):
    """numpy's and a 0-dimensional array's too, with the binding and without; a number that is none is refused."""
    import numpy as np
    import torch
    import fufft_amd as ff
    q, out = ff.mx4_empty(4, 200), torch.empty(4, 4, device=dev)
    ff.mx4_quantize(torch.randn(4, 200, device=dev), *q)
    ff.mx4_matmul(*q, *q, out, 200)
    for binding in (ff._binding, None):
        monkeypatch.setattr(ff, "_binding", binding)
        for k in (np.int64(200), np.array(200)):
            got = torch.empty(4, 4, device=dev)
            ff.mx4_matmul(*q, *q, got, k)
            torch.cuda.synchronize()
            assert torch.equal(got, out)
        for k in (200.0, "200", None):
            with pytest.raises(TypeError):
                ff.mx4_matmul(*q, *q, out, k)
