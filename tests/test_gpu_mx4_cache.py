"""GPU tests of the paged cache of signals in microscaled 4-bit blocks
(fufft_mx4_cache_write, _read, _conv) against the 64-bit form of
tests/mx4_reference.py: what is written and read back for equality, the
convolution within the bound of fp32 summation."""
import numpy as np
import pytest

import mx4_reference as R
from test_gpu_mx4 import TYPES, signal, to_dev, torch_type, typed, with_stride

pytestmark = pytest.mark.gpu


def make_cache(rng, pages, page, channels):
    """Codes and scales of a whole cache of values, on the host."""
    c, s = R.quantize(signal(rng, pages * page, channels))
    return c.reshape(pages, page, -1), s.reshape(pages, page, -1)


@pytest.mark.parametrize("channels,page", [(1, 1), (32, 16), (40, 16), (200, 8), (256, 64), (2050, 4)])
@pytest.mark.parametrize("kind", TYPES)
def test_write(dev, rng, channels, page, kind):
    """Rows reach their slots; skipped, negative and too large slots, and every other slot, stay."""
    import torch
    import fufft_amd as ff
    print(f"case cache write {channels} channels, pages of {page}, {kind}", flush=True)
    pages, rows = 7, 5
    codes, scales = make_cache(rng, pages, page, channels)
    slots = rng.permutation(pages * page)[:rows].astype(np.int64)
    slots[1], slots[3] = -1, pages * page
    x, x64 = typed(signal(rng, rows, channels), kind, dev)
    want_c, want_s = codes.copy().reshape(pages * page, -1), scales.copy().reshape(pages * page, -1)
    qc, qs = R.quantize(x64)
    for r in (0, 2, 4):
        want_c[slots[r]], want_s[slots[r]] = qc[r], qs[r]
    for view in (x, with_stride(x, 7, 1)):
        dc, ds, dl = to_dev(dev, codes, scales, slots)
        ff.mx4_cache_write(view, dl, dc, ds)
        torch.cuda.synchronize()
        assert np.array_equal(dc.cpu().numpy().reshape(want_c.shape), want_c)
        assert np.array_equal(ds.cpu().numpy().reshape(want_s.shape), want_s)


@pytest.mark.parametrize("channels,page,length", [(1, 1, 3), (40, 16, 50), (200, 8, 65), (256, 64, 64), (130, 4, 131)])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("order", ["tokens", "channels"])
def test_read(dev, rng, channels, page, length, kind, order):
    """Lengths of zero, one, a page's end and one beside it, and the whole; a page that is none of
    the cache's; lengths outside what the page table holds."""
    import torch
    import fufft_amd as ff
    print(f"case cache read {channels} channels, pages of {page}, {length} tokens, {kind}, {order}", flush=True)
    width = -(-length // page)
    lens = np.array([0, 1, min(page, length), min(page + 1, length), length, length, 2 * width * page, -5], dtype=np.int32)
    batch, pages = len(lens), len(lens) * width + 3
    codes, scales = make_cache(rng, pages, page, channels)
    scales[2, 0, 0] = 255
    table = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)
    table[5, 0], table[4, -1] = -1, pages
    shape = (batch, length, channels) if order == "tokens" else (batch, channels, length)
    out = torch.full((int(np.prod(shape)) + 8,), 7.0, dtype=torch_type(kind), device=dev)
    view = out[4:-4].view(shape)
    ff.mx4_cache_read(*to_dev(dev, codes, scales, table, lens), view, order=order)
    torch.cuda.synchronize()
    want = np.zeros((batch, length, channels))
    for b in range(batch):
        h = R.history(codes, scales, table[b], lens[b], channels)[:length]
        want[b, :len(h)] = h
    want = torch.from_numpy(want if order == "tokens" else want.transpose(0, 2, 1).copy()).to(torch_type(kind))
    got = view.cpu()
    assert bool(((got == want) | (got.isnan() & want.isnan())).all())
    assert bool((out[:4] == 7).all()) and bool((out[-4:] == 7).all())


@pytest.mark.parametrize("channels,page,length,taps", [(1, 1, 3, 3), (40, 16, 50, 70), (200, 8, 300, 33), (513, 64, 64, 1),
                                                       (1030, 4, 131, 131), (96, 16, 2500, 2500), (2048, 16, 40, 40)])
@pytest.mark.parametrize("kind", TYPES)
def test_conv(dev, rng, channels, page, length, taps, kind):
    import torch
    import fufft_amd as ff
    print(f"case cache conv {channels} channels, pages of {page}, {length} tokens, {taps} taps, {kind}", flush=True)
    width = -(-length // page)
    for lens in ([length], [0], [0, 1, length, max(1, length - 1), min(page, length), min(page + 1, length), -3]):
        lens = np.array(lens, dtype=np.int32)
        batch, pages = len(lens), len(lens) * width + 2
        codes, scales = make_cache(rng, pages, page, channels)
        table = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)
        if batch > 2:
            table[3, 0] = -1
        h, h64 = typed(rng.standard_normal((taps, channels)), kind, dev)
        args = to_dev(dev, codes, scales, table, lens)
        want, mag = np.zeros((batch, channels)), np.zeros((batch, channels))
        for b in range(batch):
            want[b], mag[b] = R.conv_step(R.history(codes, scales, table[b], lens[b], channels), h64)
        for out_kind, splits in (("f32", 0), ("f32", 1), (kind, 64), ("bf16", 3)):
            out = torch.full((batch + 1, channels), 7.0, dtype=torch_type(out_kind), device=dev)
            work = None if splits == 0 else torch.full((splits, batch, channels), float("nan"), device=dev)
            ff.mx4_cache_conv(*args, h, out[:batch], work=work)
            torch.cuda.synchronize()
            assert R.within(out[:batch], want, mag, min(length, taps) + 64, out.dtype)
            assert bool((out[batch] == 7).all())


def test_conv_ignores_what_no_token_meets(dev, rng):
    """Taps beyond a sequence's length may be infinite or NaN, as may slots beyond it: the
    result is that of the tokens it has; a NaN that is met stays in its channel."""
    import torch
    import fufft_amd as ff
    channels, page, width = 70, 16, 4
    codes, scales = make_cache(rng, 2 * width, page, channels)
    lens = np.array([19, 3], dtype=np.int32)
    table = np.arange(2 * width, dtype=np.int32).reshape(2, width)
    flat = scales.reshape(2, width * page, -1)
    flat[0, 19:], flat[1, 3:] = 255, 255
    taps = rng.standard_normal((40, channels)).astype(np.float32)
    taps[19:] = np.nan
    taps[3, 5] = np.inf
    taps[1, 9] = np.nan
    out = torch.empty(2, channels, device=dev)
    ff.mx4_cache_conv(*to_dev(dev, codes, scales, table, lens, taps), out)
    torch.cuda.synchronize()
    got = out.cpu()
    for b in range(2):
        hist = R.history(codes, scales, table[b], lens[b], channels)
        clean = np.where(np.isfinite(taps), taps, 0)
        want, mag = R.conv_step(hist, clean)
        fine = np.ones(channels, dtype=bool)
        fine[9] = False
        assert bool(got[b, 9].isnan())
        if b == 0:
            fine[5] = False
            assert not bool(got[0, 5].isfinite())
        assert R.within(got[b][fine], want[fine], mag[fine], 104, got.dtype)


def test_conv_step_equals_the_fft_convolution(dev, rng):
    """Write, read back as padded signals, convolve them with the FFT calls: the value at each
    sequence's last token is the step form's.  Bound: the fp32 transforms' 2e-6 of the
    signal's norm times the filter's, and the sums'."""
    import torch
    import fufft_amd as ff
    channels, page, n = 6, 16, 2048
    lens = np.array([1000, 517, 1], dtype=np.int32)
    width = 1024 // page
    codes, scales = make_cache(rng, 3 * width, page, channels)
    table = rng.permutation(3 * width).reshape(3, width).astype(np.int32)
    taps = rng.standard_normal((1024, channels)).astype(np.float32)
    args = to_dev(dev, codes, scales, table, lens)
    step = torch.empty(3, channels, device=dev)
    ff.mx4_cache_conv(*args, to_dev(dev, taps)[0], step)
    signals = torch.empty(3, channels, n, device=dev)
    ff.mx4_cache_read(*args, signals, order="channels")
    u, v = torch.empty(3, n, device=dev), torch.empty(3, n, device=dev)
    for c in range(channels):
        padded = np.zeros(n, dtype=np.complex64)
        padded[:1024] = taps[:, c]
        filt = to_dev(dev, ff.plan_filter(padded, n, kind=ff.FILTER_TAPS))[0]
        x = signals[:, c].contiguous()
        ff.conv_r2(x, x.clone(), filt, u, v, n, 3)
        torch.cuda.synchronize()
        for b in range(3):
            norm = float(x[b].norm()) * float(np.linalg.norm(taps[:, c]))
            assert abs(float(u[b, lens[b] - 1]) - float(step[b, c])) <= 4e-6 * norm


def test_cache_calls_captured(dev, rng):
    """One step of generation, write and convolve, in a graph that is replayed as the lengths grow."""
    import torch
    import fufft_amd as ff
    channels, page, width, batch = 300, 16, 8, 3
    codes, scales = make_cache(rng, batch * width, page, channels)
    table = np.arange(batch * width, dtype=np.int32).reshape(batch, width)
    dc, ds, dt = to_dev(dev, codes, scales, table)
    lens = torch.tensor([5, 0, 31], dtype=torch.int32, device=dev)
    x = torch.randn(batch, channels, device=dev)
    slots = torch.zeros(batch, dtype=torch.int64, device=dev)
    taps = torch.randn(128, channels, device=dev)
    out, work = torch.empty(batch, channels, device=dev), torch.empty(8, batch, channels, device=dev)
    first = torch.arange(batch, device=dev) * width * page

    def step():
        slots.copy_(first + lens)
        lens.add_(1)
        ff.mx4_cache_write(x, slots, dc, ds)
        ff.mx4_cache_conv(dc, ds, dt, lens, taps, out, work=work)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    torch.cuda.synchronize()
    for _ in range(4):
        x.copy_(torch.randn(batch, channels, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        lens.sub_(1)
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        hist = [R.history(dc.cpu().numpy(), ds.cpu().numpy(), table[b], int(lens[b]), channels) for b in range(batch)]
        for b in range(batch):
            want, mag = R.conv_step(hist[b], taps.double().cpu().numpy())
            assert R.within(out[b], want, mag, 192, out.dtype)
