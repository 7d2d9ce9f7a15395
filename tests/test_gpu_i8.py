"""GPU tests of the 8-bit rows and their products (fufft_i8_quantize, _dequantize, _matmul).  Codes,
scales and integer sums are compared for equality with the 64-bit form of
tests/layer_reference.py; results within the four fp32 roundings behind them."""
import numpy as np
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu


def signal(rng, rows, k):
    x = rng.standard_normal((rows, k)) * 10.0 ** rng.uniform(-30, 30, (rows, 1))
    return np.where(rng.random((rows, k)) < 1 / 16, 0.0, x)


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 31), (5, 127), (7, 128), (2, 129), (130, 33), (4, 1000), (3, 2049), (3, 5001),
                                    (2, 16385), (2, 40000), (2, 65537), (2, 131071)])
@pytest.mark.parametrize("kind", R.TYPES)
def test_quantize(dev, rng, rows, k, kind):
    import torch
    import fufft_amd as ff
    print(f"case i8_quantize {rows}x{k} {kind}", flush=True)
    x = signal(rng, rows, k)
    if kind == "f16":
        x = np.clip(x, -6e4, 6e4)
    # halves of the largest magnitude are half-way between two codes
    x[:, ::5] = np.sign(x[:, ::5]) * np.abs(x).max(1, keepdims=True) / 2
    x, x64 = R.typed(x, kind, dev)
    want, want_s = R.quantize(x64)
    for view in (x, R.with_stride(x)):
        codes, scales = ff.i8_empty(rows, k)
        codes.fill_(99)
        ff.i8_quantize(view, codes, scales)
        assert np.array_equal(codes.cpu().numpy(), want)
        assert np.array_equal(scales.cpu().numpy(), want_s)
    for to in R.TYPES:
        out = torch.full((rows, k + 3), 7.0, dtype=R.torch_type(to), device=dev)
        ff.i8_dequantize(codes, scales, out[:, :k])
        v = codes[:, :k].double() * scales[:, None].double()
        assert R.inside(out[:, :k], v.cpu().numpy(), R.EPS24 * v.abs().cpu().numpy())
        assert bool((out[:, k:] == 7).all())


def test_every_bf16_near_half_way(dev):
    """All fp32 neighbours of every half-way point of some rows, both signs."""
    import torch
    import fufft_amd as ff
    for top in (1.0, 127.0, 3.1415927, 2.0 ** -140, 1.7e38, 0.99999994):
        top = np.float32(top)
        mid = ((np.arange(127) + 0.5) * np.float64(top) / 127).astype(np.float32)
        near = np.concatenate([[top], mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(np.inf))])
        x = np.concatenate([near, -near]).astype(np.float32)[None]
        x = x[:, np.abs(x[0]) <= top]
        codes, scales = ff.i8_empty(1, x.shape[1])
        ff.i8_quantize(torch.from_numpy(x).to(dev), codes, scales)
        want, want_s = R.quantize(x)
        assert np.array_equal(codes.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), want_s)


def test_quantize_special(dev):
    import torch
    import fufft_amd as ff
    for k in (5, 600, 3000, 9000, 70000):
        x = torch.ones(5, k)
        x[1, k - 1] = float("nan")
        x[2, 0] = float("-inf")
        x[3] = 0
        codes, scales = ff.i8_empty(5, k)
        ff.i8_quantize(x.to(dev), codes, scales)
        out = torch.empty(5, k, device=dev)
        ff.i8_dequantize(codes, scales, out)
        assert scales[1].isnan() and scales[2].isnan() and scales[3] == 0 and not codes[1:4].any()
        assert out[1].isnan().all() and out[2].isnan().all() and not out[3].any()
        assert bool((codes[[0, 4], :k] == 127).all())


def operands(rng, dev, rows, k, full=False):
    import torch
    c = np.zeros((rows, R.padded(k)), dtype=np.int8)
    c[:, :k] = rng.integers(-128 if full else -127, 128, (rows, k))
    s = (rng.uniform(0.5, 2, rows) * 10.0 ** rng.uniform(-3, 3, rows)).astype(np.float32)
    return c, s, torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev)


# every kernel and its edges: few rows (16 rows and 32 columns a workgroup, K split), 64, 128 and 256 tiles
SIZES = [(1, 1, 1), (1, 130, 64), (3, 17, 200), (16, 4100, 129), (1, 8192, 8192), (13, 5000, 2056), (17, 33, 64), (31, 100, 4000),
         (64, 512, 4096), (200, 300, 1024), (129, 257, 65), (333, 777, 513), (1001, 2000, 1504), (2048, 2100, 320),
         (4100, 4000, 130), (4096, 8200, 256), (5, 64, 0), (70, 64, 0)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("kind", R.TYPES)
def test_matmul(dev, rng, m, n, k, kind):
    import torch
    import fufft_amd as ff
    print(f"case i8_matmul {m}x{n}x{k} {kind}", flush=True)
    a, sa, da, dsa = operands(rng, dev, m, k, full=True)
    b, sb, db, dsb = operands(rng, dev, n, k, full=True)
    for with_bias in (False, True):
        bias = rng.standard_normal(n).astype(np.float32) * 1000 if with_bias else None
        dbias = torch.from_numpy(bias).to(dev) if with_bias else None
        big = m * n > 1 << 21
        if big:                                     # the integer sum in fp64 on the GPU: exact below 2^53
            s = (da[:, :k].double() @ db[:, :k].double().t().contiguous()).cpu().numpy()
            v = s * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
            want = v if bias is None else v + bias
            err = R.EPS24 * (3.001 * np.abs(v) + 1.001 * np.abs(want))
        else:
            want, err = R.matmul(a, sa, b, sb, bias, k)
        wide = torch.full((m, n + 5), 3.0, dtype=R.torch_type(kind), device=dev)
        if kind == "f16":
            want, err, = want * 2.0 ** -20, err * 2.0 ** -20
            ff.i8_matmul(da, dsa * 2.0 ** -20, db, dsb, wide[:, 2:n + 2], k, bias=None if dbias is None else dbias * 2.0 ** -20)
            ok = np.abs(want) < 60000
            got = torch.where(torch.from_numpy(ok).to(dev), wide[:, 2:n + 2], torch.zeros_like(wide[:, 2:n + 2]))
            # fp16's own subnormals are multiples of 2^-24: rounding keeps the order there too
            assert R.inside(got, np.where(ok, want, 0), np.where(ok, err, 0))
        else:
            ff.i8_matmul(da, dsa, db, dsb, wide[:, 2:n + 2], k, bias=dbias)
            assert R.inside(wide[:, 2:n + 2], want, err)
        assert bool((wide[:, :2] == 3).all()) and bool((wide[:, n + 2:] == 3).all())


@pytest.mark.parametrize("m", [1, 40, 300])
def test_longest_sum(dev, m):
    """The largest sum there is stays exact: 131071 products of -128 and -128."""
    import torch
    import fufft_amd as ff
    k, n = 131071, 50
    a, b = torch.zeros(m, ff.i8_padded(k), dtype=torch.int8, device=dev), torch.zeros(n, ff.i8_padded(k), dtype=torch.int8, device=dev)
    a[:, :k] = -128
    b[:, :k] = -128
    one = torch.ones(max(m, n), device=dev)
    out = torch.empty(m, n, device=dev)
    ff.i8_matmul(a, one[:m], b, one[:n], out, k)
    assert bool((out == float(np.float32(131071 * 128 * 128))).all())


def test_special_scales(dev, rng):
    """A row's NaN scale (a row that held NaN) fills its results alone."""
    import torch
    import fufft_amd as ff
    for m in (4, 300):
        _, _, a, sa = operands(rng, dev, m, 200)
        _, _, b, sb = operands(rng, dev, 150, 200)
        sa[2] = float("nan")
        out = torch.empty(m, 150, device=dev)
        ff.i8_matmul(a, sa, b, sb, out, 200)
        assert out[2].isnan().all() and not out[:2].isnan().any() and not out[3:].isnan().any()
