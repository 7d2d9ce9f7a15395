"""GPU tests of the microscaled 4-bit blocks and their products (fufft_mx4_quantize,
_dequantize, _matmul, _linear) against the 64-bit form of tests/mx4_reference.py.

Codes and scale bytes are compared for equality.  Products are sums of terms that fp32
holds exactly (mx4 x mx4) or that the parts of x make up exactly (linear), so their
bound is the one of fp32 summation, mx4_reference.within.
"""
import numpy as np
import pytest

import mx4_reference as R

pytestmark = pytest.mark.gpu

TYPES = ("f32", "bf16", "f16")


def torch_type(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def typed(x, name, dev):
    """x rounded to the type: the tensor on the GPU, and its values in 64 bits."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).to(torch_type(name))
    return t.to(dev), t.double().numpy()


def with_stride(t, extra, offset):
    """The same matrix as rows of a wider one, its first element `offset` elements in."""
    import torch
    rows, k = t.shape
    wide = torch.full((rows * (k + extra) + offset,), float("nan"), dtype=t.dtype, device=t.device)
    v = wide[offset:].view(rows, k + extra)[:, :k]
    v.copy_(t)
    return v


def signal(rng, rows, k):
    """Values over a few decades, one in 16 of them zero."""
    x = rng.standard_normal((rows, k)) * 10.0 ** rng.uniform(-2, 2, (rows, 1))
    return np.where(rng.random((rows, k)) < 1 / 16, 0.0, x)


def blocks(dev, rows, k):
    import torch
    kp = R.padded(k)
    return (torch.full((rows, kp // 2), 0xEE, dtype=torch.uint8, device=dev),
            torch.full((rows, kp // 32), 0xEE, dtype=torch.uint8, device=dev))


def to_dev(dev, *arrays):
    import torch
    return [torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in arrays]


SIZES = [(1, 1), (1, 32), (3, 31), (5, 127), (2, 128), (7, 129), (128, 130), (33, 1000), (130, 33), (1, 5001),
         (257, 2048), (300, 7)]


@pytest.mark.parametrize("rows,k", SIZES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rule", ["fit", "floor"])
@pytest.mark.parametrize("random", [False, True])
def test_quantize(dev, rng, rows, k, kind, rule, random):
    import torch
    import fufft_amd as ff
    print(f"case quantize {rows}x{k} {kind} {rule} random={random}", flush=True)
    x, x64 = typed(signal(rng, rows, k), kind, dev)
    rand = rng.integers(0, 256, (rows, k)).astype(np.uint8) if random else None
    drand = None if rand is None else to_dev(dev, rand)[0]
    want, want_t = R.quantize(x64, rule, rand), R.quantize(x64.T, rule, None if rand is None else rand.T)
    for view in (x, with_stride(x, 5, 3)):
        for along, across in ((True, False), (False, True), (True, True)):
            q = blocks(dev, rows, k) if along else (None, None)
            t = blocks(dev, k, rows) if across else (None, None)
            ff.mx4_quantize(view, *q, *t, rand=drand, rule=rule)
            torch.cuda.synchronize()
            for got, ref in ((q, want), (t, want_t)):
                if got[0] is not None:
                    assert np.array_equal(got[1].cpu().numpy(), ref[1])
                    assert np.array_equal(got[0].cpu().numpy(), ref[0])


@pytest.mark.parametrize("rule", ["fit", "floor"])
@pytest.mark.parametrize("random", [False, True])
def test_quantize_special_values(dev, rng, rule, random):
    """Zeros, ties, subnormals, the ends of the range, infinities and NaN, in fp32."""
    import torch
    import fufft_amd as ff
    tiny, top = np.float32(2.0 ** -149), np.finfo(np.float32).max
    ties = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.5, 0.249999, 0.250001, 4.999999, 5.000001, 1])
    ties = np.concatenate([ties, -ties])
    rows = [np.zeros(32), -np.zeros(32), ties, ties * 2.0 ** 100, ties * 2.0 ** -126, ties * 2.0 ** -140,
            np.full(32, tiny), np.full(32, top), np.r_[top, np.full(31, 1.0)], np.r_[1.0, np.full(31, 2.0 ** -127)],
            np.r_[np.inf, np.ones(31)], np.r_[np.ones(31), -np.inf], np.r_[np.nan, np.ones(31)], np.full(32, np.nan),
            np.r_[6.0, ties[1:]], np.r_[np.nextafter(np.float32(6), np.float32(7)), ties[1:]],
            np.r_[8.0, ties[1:]], np.r_[np.nextafter(np.float32(8), np.float32(0)), ties[1:]], 2.0 ** -126 * ties,
            2.0 ** -127 * np.ones(32), 1.5 * 2.0 ** -125 * np.ones(32)]
    x = np.stack(rows).astype(np.float32)
    x = np.concatenate([x, np.roll(x, 1, axis=0)], axis=1)       # blocks with different neighbours
    rand = rng.integers(0, 256, x.shape).astype(np.uint8) if random else None
    q, t = blocks(dev, *x.shape), blocks(dev, *x.shape[::-1])
    drand = None if rand is None else to_dev(dev, rand)[0]
    ff.mx4_quantize(to_dev(dev, x)[0], *q, rand=drand, rule=rule)
    torch.cuda.synchronize()
    want = R.quantize(x, rule, rand)
    assert np.array_equal(q[1].cpu().numpy(), want[1])
    assert np.array_equal(q[0].cpu().numpy(), want[0])
    # the same blocks along columns
    ff.mx4_quantize(to_dev(dev, x.T)[0], None, None, *q, rand=None if rand is None else to_dev(dev, rand.T)[0], rule=rule)
    torch.cuda.synchronize()
    assert np.array_equal(q[1].cpu().numpy(), want[1])
    assert np.array_equal(q[0].cpu().numpy(), want[0])


def test_every_random_byte_at_every_share(dev):
    """Values at 1/256 and half of that between grid neighbours, under every byte."""
    import torch
    import fufft_amd as ff
    share = np.arange(512) / 512
    lo, hi = R.GRID[:7, None], R.GRID[1:, None]
    mag = (lo + (hi - lo) * share).reshape(-1)                    # 3584 magnitudes, exact in fp32
    x = np.zeros((256, -(-len(mag) // 31) * 32), dtype=np.float32)
    body = np.zeros(x.shape[1] // 32 * 31)
    body[:len(mag)] = mag
    x.reshape(256, -1, 32)[:, :, 1:] = body.reshape(-1, 31)
    x.reshape(256, -1, 32)[:, :, 0] = 6                           # the block's power is 1
    rand = np.repeat(np.arange(256, dtype=np.uint8)[:, None], x.shape[1], axis=1)
    q = blocks(dev, *x.shape)
    ff.mx4_quantize(to_dev(dev, x)[0], *q, rand=to_dev(dev, rand)[0])
    torch.cuda.synchronize()
    codes, scales = R.quantize(x, "fit", rand)
    assert np.array_equal(q[1].cpu().numpy(), scales) and np.array_equal(q[0].cpu().numpy(), codes)
    # the mean over the bytes is the value to within half a 256th of a step
    back = R.values(codes, scales, x.shape[1]).mean(0)
    step = np.where(x[0] >= 4, 2, np.where(x[0] >= 2, 1, 0.5))
    assert np.all(np.abs(back - x[0]) <= step / 512 + 1e-12)


@pytest.mark.parametrize("kind", TYPES)
def test_dequantize_every_code_and_scale(dev, kind):
    import torch
    import fufft_amd as ff
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(1, 256), (256, 1))      # 512 values: 16 blocks
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, axis=1)
    scales = (scales + np.arange(16, dtype=np.uint8)[None]).astype(np.uint8)
    want = torch.from_numpy(R.values(codes, scales, 512)).to(torch_type(kind))
    c, s = to_dev(dev, codes, scales)
    for k in (512, 500, 487):
        out = torch.full((256, k + 9), 7.0, dtype=torch_type(kind), device=dev)
        ff.mx4_dequantize(*[t[:, :n].contiguous() for t, n in ((c, R.padded(k) // 2), (s, R.padded(k) // 32))],
                          out[:, 1:k + 1])
        torch.cuda.synchronize()
        got = out[:, 1:k + 1].cpu()
        ok = (got == want[:, :k]) | (got.isnan() & want[:, :k].isnan())
        assert bool(ok.all())
        assert bool((out[:, 0] == 7).all()) and bool((out[:, k + 1:] == 7).all())


def random_blocks(rng, rows, k, spread=6):
    """Blocks of every code, scales over 2^+-spread, zero codes in the padding."""
    kp = R.padded(k)
    q = rng.integers(0, 16, (rows, kp)).astype(np.uint8)
    q[:, k:] = 0
    scales = rng.integers(127 - spread, 128 + spread, (rows, kp // 32)).astype(np.uint8)
    return q[:, 0::2] + 16 * q[:, 1::2], scales


MATMULS = [(1, 1, 1), (1, 17, 32), (2, 5, 127), (16, 16, 128), (17, 33, 129), (33, 40, 384), (64, 64, 256),
           (65, 100, 1000), (5, 1000, 4096), (130, 257, 520), (128, 128, 2048), (256, 256, 512), (300, 513, 2176),
           (129, 640, 1100), (513, 300, 96), (1000, 999, 200), (1, 4096, 640), (2048, 2048, 256),
           # each kernel and tile, with K ending in half a slab and beyond the scales of one fetch
           (7, 5000, 300), (20, 1000, 4200), (32, 4090, 2176), (64, 4090, 2100), (700, 1000, 2500), (2048, 2000, 4700),
           (4096, 4096, 300), (4090, 3900, 2176)]


@pytest.mark.parametrize("m,n,k", MATMULS)
@pytest.mark.parametrize("out", TYPES)
def test_matmul(dev, rng, m, n, k, out):
    import torch
    import fufft_amd as ff
    print(f"case matmul {m}x{n}x{k} {out}", flush=True)
    a, b = random_blocks(rng, m, k), random_blocks(rng, n, k)
    bias = rng.standard_normal(n).astype(np.float32)
    av, bv = R.values(*a, k), R.values(*b, k)
    y, mag = av @ bv.T, np.abs(av) @ np.abs(bv).T
    da, db, (dbias,) = to_dev(dev, *a), to_dev(dev, *b), to_dev(dev, bias)
    for with_bias, extra in ((False, 0), (True, 3)):
        o = torch.full((m + 2, n + extra), 7.0, dtype=torch_type(out), device=dev)
        ff.mx4_matmul(*da, *db, o[1:m + 1, :n], k, bias=dbias if with_bias else None)
        torch.cuda.synchronize()
        want = y + bias if with_bias else y
        assert R.within(o[1:m + 1, :n], want, mag + np.abs(bias) * with_bias, k + 1, o.dtype)
        assert bool((o[0] == 7).all()) and bool((o[m + 1] == 7).all()) and bool((o[:, n:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(16, 32, 300), (300, 400, 640)])
def test_matmul_nan_and_range(dev, rng, m, n, k):
    """A NaN block makes its row or column NaN and no other; the scales' ends keep their
    product; sums of no values are the bias."""
    import torch
    import fufft_amd as ff
    a, b = random_blocks(rng, m, k), random_blocks(rng, n, k)
    a[1][3, 1] = 255
    b[1][5, 0] = 255
    o = torch.empty(m, n, device=dev)
    ff.mx4_matmul(*to_dev(dev, *a), *to_dev(dev, *b), o, k)
    torch.cuda.synchronize()
    nan = np.zeros((m, n), dtype=bool)
    nan[3], nan[:, 5] = True, True
    assert np.array_equal(o.isnan().cpu().numpy(), nan)
    # 2^120 times 2^-120, and 2^-127 times 2^126
    for sa, sb in ((247, 7), (0, 253)):
        a[1][:], b[1][:] = sa, sb
        av, bv = R.values(*a, k), R.values(*b, k)
        ff.mx4_matmul(*to_dev(dev, *a), *to_dev(dev, *b), o, k)
        torch.cuda.synchronize()
        want, mag = av @ bv.T, np.abs(av) @ np.abs(bv).T
        assert R.within(o, want, mag, k, o.dtype)
    e = [t[:, :0].contiguous() for t in to_dev(dev, *a) + to_dev(dev, *b)]
    bias = torch.randn(n, device=dev)
    ff.mx4_matmul(*e, o, 0, bias=bias)
    torch.cuda.synchronize()
    assert torch.equal(o, bias.expand(m, n))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 5, 7), (130, 70, 200), (64, 256, 129)])
def test_layer_gradients(dev, rng, kind, m, n, k):
    """Forward, dx and dw of a layer from the calls against the formulas in 64 bits, and
    against differences: on values that 4 bits hold exactly, sum(dy * y) is linear in x
    and in w, so its difference over a step is the gradient's product with that step."""
    import torch
    import fufft_amd as ff
    print(f"case gradients {m}x{n}x{k} {kind}", flush=True)
    pick = lambda r, c: rng.choice(np.r_[R.GRID, -R.GRID], (r, c))  # noqa: E731
    grid = [pick(m, k), pick(n, k), pick(m, n)]
    free = [signal(rng, *s.shape) for s in grid]
    for exact in (True, False):
        vals = grid if exact else free
        if exact:
            for v in vals:                            # every block holds a 6, along rows and along columns
                v[::32, ::32] = 6
                v[0, :] = 6
                v[:, 0] = 6
                v[::32, :] = 6
                v[:, ::32] = 6
        (x, x64), (w, w64), (dy, dy64) = [typed(v, kind, dev) for v in vals]
        q = {}
        for name, t, t64 in (("x", x, x64), ("w", w, w64), ("dy", dy, dy64)):
            r, c = t.shape
            q[name], q[name + "_t"] = blocks(dev, r, c), blocks(dev, c, r)
            ff.mx4_quantize(t, *q[name], *q[name + "_t"])
        y, dx, dw = (torch.empty(s, device=dev) for s in ((m, n), (m, k), (n, k)))
        ff.mx4_matmul(*q["x"], *q["w"], y, k)
        ff.mx4_matmul(*q["dy"], *q["w_t"], dx, n)
        ff.mx4_matmul(*q["dy_t"], *q["x_t"], dw, m)
        torch.cuda.synchronize()
        rows = lambda t: R.values(*R.quantize(t), t.shape[1])  # noqa: E731
        for got, a, b in ((y, rows(x64), rows(w64)), (dx, rows(dy64), rows(w64.T)), (dw, rows(dy64.T), rows(x64.T))):
            want, mag = a @ b.T, np.abs(a) @ np.abs(b).T
            assert R.within(got, want, mag, a.shape[1], got.dtype)
        if exact:
            f = lambda x_, w_: float(np.sum(dy64 * (x_ @ w_.T)))  # noqa: E731
            hx, hw = rng.standard_normal((m, k)), rng.standard_normal((n, k))
            for got, diff, h in ((dx, f(x64 + hx, w64) - f(x64, w64), hx), (dw, f(x64, w64 + hw) - f(x64, w64), hw)):
                g = got.double().cpu().numpy()
                # f's own rounding, in 64 bits, and the fp32 gradient's (its sums are exact here)
                slack = 2.0 ** -40 * np.sum(np.abs(dy64) * (np.abs(x64) @ np.abs(w64).T + np.abs(hx) @ np.abs(w64).T
                                                            + np.abs(x64) @ np.abs(hw).T))
                assert abs(np.sum(g * h) - diff) <= slack


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 300, 1000), (2, 64, 128), (7, 33, 4100), (15, 16, 129), (16, 100, 256),
                                   (17, 129, 640), (33, 50, 96), (64, 64, 1024), (65, 70, 300), (200, 48, 257),
                                   (1, 4200, 700), (20, 4200, 300), (40, 4200, 1100)])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_linear(dev, rng, m, n, k, kind, out):
    import torch
    import fufft_amd as ff
    print(f"case linear {m}x{n}x{k} {kind} -> {out}", flush=True)
    x, x64 = typed(rng.standard_normal((m, k)), kind, dev)
    w = random_blocks(rng, n, k)
    wv = R.values(*w, k)
    bias = rng.standard_normal(n).astype(np.float32)
    dw, (dbias,) = to_dev(dev, *w), to_dev(dev, bias)
    y, mag = x64 @ wv.T, np.abs(x64) @ np.abs(wv).T
    parts = {"f32": 3, "bf16": 1, "f16": 2}[kind]
    for view, with_bias in ((x, False), (with_stride(x, 3, 1), True)):
        o = torch.full((m, n + 5), 7.0, dtype=torch_type(out), device=dev)
        ff.mx4_linear(view, *dw, o[:, 2:n + 2], bias=dbias if with_bias else None)
        torch.cuda.synchronize()
        want = y + bias if with_bias else y
        assert R.within(o[:, 2:n + 2], want, mag + np.abs(bias) * with_bias, parts * k + 1, o.dtype)
        assert bool((o[:, :2] == 7).all()) and bool((o[:, n + 2:] == 7).all())


@pytest.mark.parametrize("kind", TYPES)
def test_linear_infinities_nan_and_range(dev, kind):
    """An infinity or NaN in a row of x stays in that row; the type's largest value times 1/2
    is right; a NaN of any payload is a NaN."""
    import torch
    import fufft_amd as ff
    t = torch_type(kind)
    k, n = 200, 20
    x = torch.ones(6, k, dtype=t)
    x[1, 7], x[2, 150], x[3, 0] = float("inf"), float("nan"), -float("inf")
    x[4] = 0
    x[4, 3] = torch.finfo(t).max
    w = np.full((n, 256 // 2), 0x11, dtype=np.uint8)           # every value 1/2 (the padding too: x ends before it)
    w[:, k // 2:] = 0
    s = np.full((n, 8), 127, dtype=np.uint8)
    if kind == "f32":
        x[5] = torch.from_numpy(np.full(k, 0x7f800001, dtype=np.uint32).view(np.float32))
    else:
        x[5] = float("nan")
    o = torch.empty(6, n, device=dev)
    ff.mx4_linear(x.to(dev), *to_dev(dev, w, s), o)
    torch.cuda.synchronize()
    o = o.cpu()
    assert bool((o[0] == k / 2).all())
    assert bool((o[1] == float("inf")).all()) and bool((o[3] == -float("inf")).all())
    assert bool(o[2].isnan().all()) and bool(o[5].isnan().all())
    assert bool((o[4] == torch.finfo(t).max / 2).all())


def test_calls_on_another_stream_and_captured(dev, rng):
    """On a side stream, ordered by it; captured into a graph and replayed over new inputs."""
    import torch
    import fufft_amd as ff
    m, n, k = 40, 300, 520
    x = torch.randn(m, k, device=dev)
    w = to_dev(dev, *random_blocks(rng, n, k))
    q, out, lin = blocks(dev, m, k), torch.empty(m, n, device=dev), torch.empty(m, n, device=dev)

    def layer(stream=None):
        ff.mx4_quantize(x, *q, stream=stream)
        ff.mx4_matmul(*q, *w, out, k, stream=stream)
        ff.mx4_linear(x, *w, lin, stream=stream)

    layer()
    torch.cuda.synchronize()
    want = out.clone(), lin.clone()
    side = torch.cuda.Stream()
    out.zero_(), lin.zero_()
    side.wait_stream(torch.cuda.current_stream())
    layer(side)
    side.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lin, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for i in range(4):
        x.copy_(torch.randn(m, k, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lin.clone()
        layer()
        torch.cuda.synchronize()
        assert torch.equal(out, got[0]) and torch.equal(lin, got[1])
        torch.randn(1000, device=dev).sum().item()


def test_refusals_on_the_gpu(dev):
    """What the native binding does not take, the checks in Python name: a short array, another
    type, rows that overlap, a tensor of the host; a tensor subclass and a parameter pass."""
    import torch
    import fufft_amd as ff
    x, (c, s) = torch.randn(6, 300, device=dev), ff.mx4_empty(6, 300)
    out = torch.empty(6, 6, device=dev)
    cache, lens = (torch.zeros(4, 16, 192, dtype=torch.uint8, device=dev), torch.zeros(4, 16, 12, dtype=torch.uint8, device=dev)), \
        torch.zeros(2, dtype=torch.int32, device=dev)
    table = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    for call, message in (
            (lambda: ff.mx4_quantize(x, c[:5].contiguous(), s), "codes: holds"),
            (lambda: ff.mx4_quantize(x, c, s, rand=torch.zeros(6, 299, dtype=torch.uint8, device=dev)), "rand: holds"),
            (lambda: ff.mx4_quantize(x.double(), c, s), "x: dtype"),
            (lambda: ff.mx4_quantize(x[:1].expand(6, 300), c, s), "rows overlap"),
            (lambda: ff.mx4_quantize(x, c.cpu(), s), "codes: tensor is on cpu"),
            (lambda: ff.mx4_quantize(x), "neither"),
            (lambda: ff.mx4_dequantize(c, s[:, :8].contiguous(), x), "codes_scales: holds"),
            (lambda: ff.mx4_matmul(c, s, c, s, torch.empty(6, 7, device=dev), 300), "b: holds"),
            (lambda: ff.mx4_matmul(c, s, c, s, out, 300, bias=torch.zeros(6, device=dev).half()), "bias: dtype"),
            (lambda: ff.mx4_linear(x, c, s, out[:5]), "out: 5 rows"),
            (lambda: ff.mx4_cache_write(x, torch.zeros(6, dtype=torch.int32, device=dev), *cache), "slots: dtype"),
            (lambda: ff.mx4_cache_read(*cache, table.long(), lens, torch.empty(2, 9, 300, device=dev)), "pages: dtype"),
            (lambda: ff.mx4_cache_conv(*cache, table, lens, x, torch.empty(2, 300, device=dev).half()), "workspace"),
            (lambda: ff.mx4_cache_conv(*cache, table, lens, x, torch.empty(3, 300, device=dev)), "3 sequences")):
        with pytest.raises(ValueError, match=message):
            call()
    for bad in (c.view(torch.int8), s):                       # refused by the library itself: x's own bytes as codes
        with pytest.raises((ff.FufftError, ValueError)):
            ff.mx4_quantize(x, x.view(torch.uint8).view(-1), s) if bad is s else ff.mx4_quantize(x, bad, s)
    ff.mx4_quantize(x, c, s)
    want = c.clone()

    class Sub(torch.Tensor):
        pass

    for t in (torch.nn.Parameter(x), x.as_subclass(Sub)):
        c.zero_()
        ff.mx4_quantize(t, c, s)
        torch.cuda.synchronize()
        assert torch.equal(c, want)
