"""GPU tests of the microscaled 4-bit calls on arrays beyond 4 GiB or 2^32 elements: what lies
behind the 32-bit offsets is read and written in its place."""
import numpy as np
import pytest

import mx4_reference as R

pytestmark = pytest.mark.gpu


def test_cache_beyond_4gib(dev, rng):
    """A cache of 4.5 GiB of codes: tokens written to its last pages, read back and convolved."""
    import torch
    import fufft_amd as ff
    channels, page = 4096, 64
    pages = 36000                                       # 36000 * 64 tokens * 2 KiB
    codes = torch.zeros(pages, page, channels // 2, dtype=torch.uint8, device=dev)
    scales = torch.full((pages, page, channels // 32), 127, dtype=torch.uint8, device=dev)
    assert codes.nbytes > 1 << 32
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=dev)
    lens = torch.tensor([150], dtype=torch.int32, device=dev)
    x = torch.randn(150, channels, device=dev)
    t = torch.arange(150, device=dev)
    ff.mx4_cache_write(x, table[0].long()[t // page] * page + t % page, codes, scales)
    back = torch.empty(1, 150, channels, device=dev)
    ff.mx4_cache_read(codes, scales, table, lens, back)
    turned = torch.empty(1, channels, 150, device=dev)
    ff.mx4_cache_read(codes, scales, table, lens, turned, order="channels")
    taps = torch.randn(150, channels, device=dev)
    out = torch.empty(1, channels, device=dev)
    ff.mx4_cache_conv(codes, scales, table, lens, taps, out)
    torch.cuda.synchronize()
    want = R.values(*R.quantize(x.double().cpu().numpy()), channels)
    assert np.array_equal(back[0].double().cpu().numpy(), want)
    assert np.array_equal(turned[0].double().cpu().numpy(), want.T)
    y, mag = R.conv_step(want, taps.double().cpu().numpy())
    assert R.within(out[0], y, mag, 150 + 64, out.dtype)


def test_quantize_beyond_32_bit_elements(dev):
    """2^32 elements and more, both ways with random bytes: the last rows and columns, and the values
    read back there."""
    import torch
    import fufft_amd as ff
    rows, k = 65600, 65536
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=dev)
    assert x.numel() > 1 << 32
    x[-40:] = torch.randn(40, k, device=dev)
    x[:, -40:] = torch.randn(rows, 40, device=dev)
    rand = torch.randint(0, 256, (rows, k), dtype=torch.uint8, device=dev)
    q, t = ff.mx4_empty(rows, k), ff.mx4_empty(k, rows)
    ff.mx4_quantize(x, *q, *t, rand=rand)
    tail = torch.empty(rows, k, dtype=torch.bfloat16, device=dev)
    ff.mx4_dequantize(*q, tail)
    torch.cuda.synchronize()
    want = R.quantize(x[-40:].double().cpu().numpy(), "fit", rand[-40:].cpu().numpy())
    assert np.array_equal(q[0][-40:].cpu().numpy(), want[0]) and np.array_equal(q[1][-40:].cpu().numpy(), want[1])
    assert np.array_equal(tail[-40:].double().cpu().numpy(), R.values(*want, k))
    want = R.quantize(x[:, -40:].t().double().cpu().numpy(), "fit", rand[:, -40:].t().cpu().numpy())
    assert np.array_equal(t[0][-40:].cpu().numpy(), want[0]) and np.array_equal(t[1][-40:].cpu().numpy(), want[1])


@pytest.mark.parametrize("m", [3, 70, 300])
def test_products_beyond_4gib(dev, m):
    """A weight of 4.3 GiB of codes: the results of its last rows, in both products."""
    import torch
    import fufft_amd as ff
    n, k = 70144, 131072
    codes = torch.zeros(n, k // 2, dtype=torch.uint8, device=dev)
    assert codes.nbytes > 1 << 32
    codes[-50:] = torch.randint(0, 256, (50, k // 2), dtype=torch.uint8, device=dev)
    scales = torch.full((n, k // 32), 120, dtype=torch.uint8, device=dev)
    x = torch.randn(m, k, device=dev).bfloat16()
    q = ff.mx4_empty(m, k)
    ff.mx4_quantize(x, *q)
    out, lin = torch.empty(m, n, device=dev), torch.empty(m, n, device=dev)
    ff.mx4_matmul(*q, codes, scales, out, k)
    ff.mx4_linear(x, codes, scales, lin)
    torch.cuda.synchronize()
    w = R.values(codes[-50:].cpu().numpy(), scales[-50:].cpu().numpy(), k)
    for got, a in ((out, R.values(q[0].cpu().numpy(), q[1].cpu().numpy(), k)), (lin, x.double().cpu().numpy())):
        assert bool((got[:, :-50] == 0).all())
        assert R.within(got[:, -50:].contiguous(), a @ w.T, np.abs(a) @ np.abs(w).T, k, got.dtype)
