"""GPU tests of the 4-bit calls on long texts, many rows and many sequences: more tiles than one
dimension of a grid takes.  And of the largest tiles called first in a graph."""
import numpy as np
import pytest

import mx4_reference as R
from test_gpu_mx4 import signal, to_dev, torch_type

pytestmark = pytest.mark.gpu


def small_cache(rng, dev, pages, page, channels):
    """A cache of few pages on the GPU, and the values of its slots."""
    c, s = R.quantize(signal(rng, pages * page, channels))
    values = R.values(c, s, channels)
    dc, ds = to_dev(dev, c.reshape(pages, page, -1), s.reshape(pages, page, -1))
    return dc, ds, values


# tokens order: 4 tokens a workgroup above 1024 channels, 64 below 129, so 65535 workgroups are 262140 and
# 4194240 tokens; channels order: 64 always
@pytest.mark.parametrize("order,channels,length,kind", [("tokens", 2048, 300001, "bf16"), ("tokens", 1030, 262141, "f16"),
                                                        ("tokens", 5, 4194300, "f32"), ("channels", 3, 4194305, "f32"),
                                                        ("channels", 130, 4194300, "bf16")])
def test_read_long_texts(dev, rng, order, channels, length, kind):
    """Every token of a long text, a short one and one that ends beyond the last whole round, each a row of
    one of the few pages that the page tables repeat."""
    import torch
    import fufft_amd as ff
    print(f"case cache read {length} x {channels} {kind}, {order}", flush=True)
    page, pages = 64, 11
    codes, scales, values = small_cache(rng, dev, pages, page, channels)
    rows = torch.from_numpy(values).to(torch_type(kind)).to(dev)
    width = -(-length // page)
    table = torch.from_numpy(rng.integers(0, pages, (3, width)).astype(np.int32)).to(dev)
    lens = torch.tensor([length, 70, length - 3], dtype=torch.int32, device=dev)
    shape = (length, channels) if order == "tokens" else (channels, length)
    out = torch.full((3, *shape), 7.0, dtype=torch_type(kind), device=dev)
    ff.mx4_cache_read(codes, scales, table, lens, out, order=order)
    torch.cuda.synchronize()
    t = torch.arange(length, device=dev)
    for b in range(3):
        want = rows[table[b].long()[t // page] * page + t % page]
        want[int(lens[b]):] = 0
        assert torch.equal(out[b] if order == "tokens" else out[b].t(), want)


@pytest.mark.parametrize("n,k,kind,out", [(3, 40, "bf16", "f32"), (5, 130, "f32", "bf16")])
def test_linear_many_rows(dev, rng, n, k, kind, out):
    """More rows than 65535 tiles of 32 hold, in rows apart: each the product of its own x.  Integers and
    halves, whose sums are exact; the last rows are other rows' values, so they differ from the first."""
    import torch
    import fufft_amd as ff
    m = 65535 * 32 + 77
    print(f"case linear {m}x{n}x{k} {kind} -> {out}", flush=True)
    x = torch.randint(-3, 4, (m, k + 3), device=dev).to(torch_type(kind))[:, :k]
    q = rng.integers(0, 4, (n, R.padded(k))).astype(np.uint8)                # 0, .5, 1, 1.5
    q[:, k:] = 0
    codes, scales = q[:, 0::2] + 16 * q[:, 1::2], np.full((n, R.padded(k) // 32), 127, np.uint8)
    w = torch.from_numpy(R.values(codes, scales, k)).float().to(dev)
    o = torch.full((m + 1, n + 1), 7.0, dtype=torch_type(out), device=dev)
    ff.mx4_linear(x, *to_dev(dev, codes, scales), o[:m, :n])
    torch.cuda.synchronize()
    want = (x.double() @ w.double().t().contiguous()).float()
    assert torch.equal(o[:m, :n], want.to(o.dtype))
    assert bool((o[m] == 7).all()) and bool((o[:, n] == 7).all())


# workgroups of 1024 lanes, 8 for a sequence, up to 7 channels; of 512, 2 for a sequence, above; the join
# has 8 lanes a result: each beyond 2^32 lanes in one launch
@pytest.mark.parametrize("batch,channels,kind", [(524300, 3, "f32"), (4194310, 9, "bf16"), (131100, 4100, "bf16")])
def test_conv_many_sequences(dev, rng, batch, channels, kind):
    """Sequences of 0 to 2 tokens; values and taps whose sums are exact in the results' type."""
    import torch
    import fufft_amd as ff
    print(f"case cache conv {batch} x {channels} -> {kind}", flush=True)
    page, pages = 2, 5
    q = rng.integers(0, 16, (pages * page, R.padded(channels))).astype(np.uint8)
    q[:, channels:] = 0
    codes, scales = q[:, 0::2] + 16 * q[:, 1::2], np.full((pages * page, R.padded(channels) // 32), 127, np.uint8)
    values = torch.from_numpy(R.values(codes, scales, channels)).float().to(dev)
    dc, ds = to_dev(dev, codes.reshape(pages, page, -1), scales.reshape(pages, page, -1))
    table = torch.randint(0, pages, (batch, 1), device=dev, dtype=torch.int32)
    lens = torch.randint(0, 3, (batch,), device=dev, dtype=torch.int32)
    taps = torch.randint(-2, 3, (2, channels), device=dev).float()
    out = torch.full((batch + 1, channels), 7.0, dtype=torch_type(kind), device=dev)
    work = None if kind == "f32" else torch.empty(1, batch, channels, device=dev)
    ff.mx4_cache_conv(dc, ds, table, lens, taps, out[:batch], work=work)
    torch.cuda.synchronize()
    # every (page, length) has one result
    first, second = values[0::2], values[1::2]
    each = torch.stack((torch.zeros_like(first), taps[0] * first, taps[0] * second + taps[1] * first)).to(out.dtype)
    for i in torch.arange(batch, device=dev).split(1 << 16):
        assert torch.equal(out[i], each[lens[i].long(), table[i, 0].long()] + 0.0)
    assert bool((out[batch] == 7).all())


@pytest.mark.parametrize("order", ["tokens", "channels"])
def test_read_many_sequences(dev, rng, order):
    """More sequences than a grid's z dimension."""
    import torch
    import fufft_amd as ff
    page, pages, channels, batch, length = 4, 9, 20, 65535 + 1000, 6
    codes, scales, values = small_cache(rng, dev, pages, page, channels)
    rows = torch.from_numpy(values).to(dev)
    table = torch.from_numpy(rng.integers(0, pages, (batch, 2)).astype(np.int32)).to(dev)
    lens = torch.from_numpy(rng.integers(0, 9, batch).astype(np.int32)).to(dev)
    shape = (length, channels) if order == "tokens" else (channels, length)
    out = torch.full((batch, *shape), 7.0, device=dev)
    ff.mx4_cache_read(codes, scales, table, lens, out, order=order)
    torch.cuda.synchronize()
    t = torch.arange(length, device=dev)
    want = rows[table.long()[:, t // page] * page + t % page] * (t < lens[:, None])[..., None]
    assert torch.equal((out if order == "tokens" else out.transpose(1, 2)).double(), want)


@pytest.mark.parametrize("rows,k,kind", [(262140 + 999, 1030, "bf16"), (65535 * 64 + 3, 40, "f32")])
def test_codec_many_rows(dev, rng, rows, k, kind):
    """More tiles of rows than a grid's y dimension, along rows: each row one of a few, read back and
    written into a cache's slots."""
    import torch
    import fufft_amd as ff
    print(f"case codec {rows}x{k} {kind}", flush=True)
    few = torch.from_numpy(signal(rng, 37, k)).to(torch_type(kind))
    which = torch.from_numpy(rng.integers(0, 37, rows)).to(dev)
    want = [torch.from_numpy(a).to(dev) for a in R.quantize(few.double().numpy())]
    values = torch.from_numpy(R.values(*(a.cpu().numpy() for a in want), k)).to(few.dtype).to(dev)
    x = few.to(dev)[which]
    q, back = ff.mx4_empty(rows, k), torch.empty_like(x)
    ff.mx4_quantize(x, *q)
    ff.mx4_dequantize(*q, back)
    torch.cuda.synchronize()
    for got, ref in zip(q, want):
        assert torch.equal(got, ref[which])
    assert torch.equal(back, values[which])
    slots = torch.randperm(rows, device=dev)
    c, s = (t.fill_(0xEE).view(rows, 1, -1) for t in q)
    ff.mx4_cache_write(x, slots, c, s)
    torch.cuda.synchronize()
    for got, ref in zip((c, s), want):
        assert torch.equal(got[slots, 0], ref[which])


@pytest.mark.parametrize("random", [False, True])
def test_columns_of_many_rows(dev, rng, random):
    """More than 65535 tiles of 128 rows, along columns: the blocks of the first rows, of those around the
    65535th tile's end and of the last."""
    import torch
    import fufft_amd as ff
    rows, k = 65535 * 128 + 300, 5
    x = torch.randn(rows, k, device=dev).bfloat16()
    rand = torch.randint(0, 256, (rows, k), dtype=torch.uint8, device=dev) if random else None
    q, t = ff.mx4_empty(rows, k), ff.mx4_empty(k, rows)
    ff.mx4_quantize(x, *q, *t, rand=rand)
    torch.cuda.synchronize()
    for first, last in ((0, 256), (65535 * 128 - 256, 65535 * 128 + 128), (65535 * 128 + 128, rows)):
        x64 = x[first:last].double().cpu().numpy()
        r = None if rand is None else rand[first:last].cpu().numpy()
        want, want_t = R.quantize(x64, "fit", r), R.quantize(x64.T, "fit", None if r is None else r.T)
        end = R.padded(last)
        for got, ref in ((q[0][first:last], want[0]), (q[1][first:last], want[1]), (t[0][:, first // 2:end // 2], want_t[0]),
                         (t[1][:, first // 32:end // 32], want_t[1])):
            assert np.array_equal(got.cpu().numpy(), ref)


def test_first_call_in_a_graph(dev, rng):
    """The largest tiles, whose kernel is given its LDS at its first call, called first while a graph is
    captured, in a process of its own."""
    import subprocess
    import sys
    code = """
import torch, fufft_amd as ff
m, n, k = 4096, 4096, 512
a, b, out = torch.randn(m, k, device="cuda"), torch.randn(n, k, device="cuda"), torch.zeros(m, n, device="cuda").half()
qa, qb = ff.mx4_empty(m, k), ff.mx4_empty(n, k)
ff.mx4_quantize(b, *qb)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ff.mx4_quantize(a, *qa)
    ff.mx4_matmul(*qa, *qb, out, k)
for i in range(3):
    a.normal_()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    ff.mx4_quantize(a, *qa)
    ff.mx4_matmul(*qa, *qb, out, k)
    torch.cuda.synchronize()
    assert torch.equal(got, out) and float(out.abs().sum()) > 0
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=__file__.rsplit("/tests/", 1)[0], capture_output=True, text=True,
                       timeout=100)
    assert r.returncode == 0, r.stderr
