"""GPU tests that name each way a 4-bit call can go: every kernel shape and loop, on values whose
sums are exact, so that a lost part of any sum, or one value read from another place, is
seen whatever the sum's length."""
import numpy as np
import pytest

import mx4_reference as R
from test_gpu_mx4 import TYPES, to_dev, torch_type, typed
from test_gpu_mx4_cache import make_cache

pytestmark = pytest.mark.gpu


def grid_blocks(rng, rows, k, dev):
    """Random codes under scale 127 (the grid's own values, zeros in the padding) and their
    values, doubled, as integers."""
    import torch
    kp = R.padded(k)
    q = rng.integers(0, 16, (rows, kp)).astype(np.uint8)
    q[:, k:] = 0
    codes, scales = q[:, 0::2] + 16 * q[:, 1::2], np.full((rows, kp // 32), 127, np.uint8)
    twice = torch.from_numpy(2 * R.values(codes, scales, k)).to(dev)
    return to_dev(dev, codes, scales), twice


# a wavefront's K loop goes round again beyond 8192 values of K (8 wavefronts, two runs of four
# groups each, up to 4 x 2 tiles) or 4096 (one run ahead); the last round whole, cut, or of one wavefront
PRODUCTS = [(5, 300, 8192 + 40), (16, 300, 20000), (9, 4200, 9000), (16, 4200, 16384 + 512),      # up to 16 rows
            (40, 90, 8192 + 513), (40, 90, 16900),                                              # 16 x 16 tiles
            (90, 600, 9001), (120, 1000, 8192 + 128),                                           # 32 x 16
            (300, 600, 9000), (250, 1000, 17000),                                               # 32 x 32
            (600, 600, 8700), (1000, 2000, 8256), (1100, 4000, 4160), (4096, 4000, 2112)]         # staged tiles


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_every_way(dev, rng, m, n, k):
    """Sums of at most 36 * 20000, in quarters: exact in fp32 in any order."""
    import torch
    import fufft_amd as ff
    print(f"case matmul {m}x{n}x{k}", flush=True)
    (a, sa), at = grid_blocks(rng, m, k, dev)
    (b, sb), bt = grid_blocks(rng, n, k, dev)
    out = torch.empty(m, n, device=dev)
    ff.mx4_matmul(a, sa, b, sb, out, k)
    torch.cuda.synchronize()
    assert torch.equal(4 * out.double(), at @ bt.t().contiguous())


@pytest.mark.parametrize("m,n,k", [(1, 200, 8192 + 40), (16, 300, 16900), (11, 120, 8164), (3, 4200, 9001), (16, 4200, 17000),
                                   (20, 100, 4096 + 24), (64, 4000, 9003), (17, 4200, 4700), (33, 4200, 8968)])
@pytest.mark.parametrize("kind", TYPES)
def test_linear_every_way(dev, rng, m, n, k, kind):
    """x of whole numbers up to 8: sums of at most 48 * 17000, in halves."""
    import torch
    import fufft_amd as ff
    print(f"case linear {m}x{n}x{k} {kind}", flush=True)
    (w, s), wt = grid_blocks(rng, n, k, dev)
    x = torch.randint(-8, 9, (m, k), device=dev).to(torch_type(kind))
    out = torch.empty(m, n, device=dev)
    ff.mx4_linear(x, w, s, out)
    torch.cuda.synchronize()
    assert torch.equal(2 * out.double(), x.double() @ wt.t().contiguous())


@pytest.mark.parametrize("m,n,k", [(1, 40, 100), (3, 40, 4096), (16, 50, 8300), (5, 4130, 515), (16, 4100, 8704), (17, 40, 129),
                                   (32, 60, 5000), (40, 4130, 640), (50, 4097, 4361)])
@pytest.mark.parametrize("kind", TYPES)
def test_linear_every_bit_of_x(dev, rng, m, n, k, kind):
    """Row j of w is one value in a column of its own, a power of two: the results are that
    column of x with all its bits, over the type's whole normal range."""
    import torch
    import fufft_amd as ff
    print(f"case linear one column {m}x{n}x{k} {kind}", flush=True)
    t = torch_type(kind)
    lo, hi = (-14, 15) if kind == "f16" else (-100, 100)
    x64 = rng.uniform(1, 2, (m, k)) * 2.0 ** rng.integers(lo, hi, (m, k)) * rng.choice([-1, 1], (m, k))
    x = torch.from_numpy(x64).to(t).to(dev)
    # the first and last columns, the ends of groups, runs and rounds, and any
    ends = [c for g in (8, 32, 128, 512, 4096, 8192) for c in (g - 1, g) if c < k]
    cols = np.r_[0, k - 1, ends, rng.integers(0, k, n)][:n]
    cols = np.r_[cols, rng.integers(0, k, n - len(cols))].astype(int)
    kp = R.padded(k)
    codes, scales = np.zeros((n, kp // 2), np.uint8), np.full((n, kp // 32), 100, np.uint8)
    power = rng.integers(125, 130, n)
    for j, c in enumerate(cols):
        codes[j, c // 2] = 2 << (4 * (c % 2))                   # 1.0
        scales[j, c // 32] = power[j]
    out = torch.empty(m, n, device=dev)
    ff.mx4_linear(x, *to_dev(dev, codes, scales), out)
    torch.cuda.synchronize()
    want = x.double().cpu().numpy()[:, cols] * 2.0 ** (power - 127.0)
    assert np.array_equal(out.double().cpu().numpy(), want)


def test_linear_subnormal_parts(dev):
    """Weights whose values are subnormal in bf16 (scale bytes near 0), and rows of x that are, or
    whose lower parts are: each by one large power of two, so that the results are normal.  All of
    x's bits from 2^-133 on count."""
    import torch
    import fufft_amd as ff
    k, n = 160, 12
    # weights: row j has code j % 7 + 1 in column 5 under scale byte j // 2
    codes, scales = np.zeros((n, 128), np.uint8), np.zeros((n, 8), np.uint8)
    for j in range(n):
        codes[j, 2], scales[j] = (j % 7 + 1) << 4, j // 2
    for t in (torch.float32, torch.bfloat16):
        x = torch.zeros(3, k, dtype=t)
        x[:, 5] = torch.tensor([2.0 ** 100, -1.5 * 2.0 ** 90, 2.0 ** 127])
        out = torch.empty(3, n, device=dev)
        ff.mx4_linear(x.to(dev), *to_dev(dev, codes, scales), out)
        torch.cuda.synchronize()
        want = x[:, 5:6].double().numpy() * R.values(codes, scales, k)[None, :, 5]
        assert np.array_equal(out.double().cpu().numpy(), want), t
    # rows of x: one value, its bits from 2^-133 on, by 2^100
    codes[:], scales[:] = 0, 127
    codes[:, 2], scales[:, 0] = 2 << 4, 227
    tiny = [2.0 ** -126, 1.5 * 2.0 ** -127, 2.0 ** -130, 2.0 ** -133, -3 * 2.0 ** -133, (1 + 2.0 ** -7) * 2.0 ** -126]
    f32 = tiny + [(1 + 2.0 ** -13) * 2.0 ** -120, -(1 + 2.0 ** -7 + 2.0 ** -20) * 2.0 ** -113, (2 - 2.0 ** -23) * 2.0 ** -110]
    for t, values in ((torch.bfloat16, tiny), (torch.float32, f32)):
        x = torch.zeros(len(values), k, dtype=torch.float64)
        x[:, 5] = torch.tensor(values, dtype=torch.float64)
        assert torch.equal(x.to(t).double(), x)
        out = torch.empty(len(values), n, device=dev)
        ff.mx4_linear(x.to(t).to(dev), *to_dev(dev, codes, scales), out)
        torch.cuda.synchronize()
        want = np.repeat(np.array(values)[:, None] * 2.0 ** 100, n, axis=1)
        assert np.array_equal(out.double().cpu().numpy(), want), t


def test_matmul_longest_rows(dev):
    """K beyond 2^24 with too many results for small tiles alone: a few columns of K, the first and
    last among them, hold values."""
    import torch
    import fufft_amd as ff
    m, n, k = 530, 520, (1 << 24) + 1000
    kp = R.padded(k)
    cols = torch.tensor([0, 1, 4095, 4096, 70000, (1 << 23) + 5, (1 << 24) - 1, 1 << 24, k - 33, k - 2, k - 1], device=dev)
    made = []
    for rows in (m, n):
        codes = torch.zeros(rows, kp // 2, dtype=torch.uint8, device=dev)
        scales = torch.full((rows, kp // 32), 127, dtype=torch.uint8, device=dev)
        q = torch.randint(0, 16, (rows, len(cols)), dtype=torch.uint8, device=dev)
        for i, c in enumerate(cols.tolist()):
            codes[:, c // 2] |= q[:, i] << (4 * (c % 2))
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=dev)
        made.append((codes, scales, grid[(q & 7).long()] * torch.where(q >= 8, -1.0, 1.0)))
    (a, sa, av), (b, sb, bv) = made
    assert a.nbytes > 1 << 32
    out = torch.empty(m, n, device=dev)
    ff.mx4_matmul(a, sa, b, sb, out, k)
    torch.cuda.synchronize()
    assert torch.equal(out.double(), av @ bv.t().contiguous())


@pytest.mark.parametrize("m", [3, 70, 300])
def test_products_beyond_4gib_exact(dev, m):
    """A weight of 4.3 GiB of codes: the results of its last rows, whose sums are exact."""
    import torch
    import fufft_amd as ff
    n, k = 70144, 131072
    codes = torch.zeros(n, k // 2, dtype=torch.uint8, device=dev)
    assert codes.nbytes > 1 << 32
    codes[-50:] = torch.randint(0, 256, (50, k // 2), dtype=torch.uint8, device=dev)
    scales = torch.full((n, k // 32), 127, dtype=torch.uint8, device=dev)
    x = torch.randint(-1, 2, (m, k), device=dev).bfloat16()
    q = ff.mx4_empty(m, k)
    ff.mx4_quantize(x, *q)
    out, lin = torch.empty(m, n, device=dev), torch.empty(m, n, device=dev)
    ff.mx4_matmul(*q, codes, scales, out, k)
    ff.mx4_linear(x, codes, scales, lin)
    torch.cuda.synchronize()
    w = torch.from_numpy(R.values(codes[-50:].cpu().numpy(), scales[-50:].cpu().numpy(), k)).to(dev)
    want = x.double() @ w.t().contiguous()
    for got in (out, lin):
        assert bool((got[:, :-50] == 0).all())
        assert torch.equal(got[:, -50:].double(), want)


# two sequences beyond 2048 channels and three beyond 1280 take a kernel of their own
@pytest.mark.parametrize("channels,lens", [(2050, [300, 7]), (2304, [300, 0]), (2561, [1, 300]), (1300, [300, 0, 299]),
                                           (1537, [17, 300, 1]), (1792, [0, 300, 33]), (4100, [64, 300])])
@pytest.mark.parametrize("kind", TYPES)
def test_conv_two_and_three_sequences(dev, rng, channels, lens, kind):
    import torch
    import fufft_amd as ff
    print(f"case cache conv {len(lens)} sequences of {channels} channels, {kind}", flush=True)
    page, length = 16, 300
    width, batch = -(-length // page), len(lens)
    pages = batch * width + 2
    codes, scales = make_cache(rng, pages, page, channels)
    table = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)
    table[0, 0] = -1
    table[1, -1] = pages
    lens = np.array(lens, dtype=np.int32)
    h, h64 = typed(rng.standard_normal((310, channels)), kind, dev)
    h64 = h64[:length]
    args = to_dev(dev, codes, scales, table, lens)
    want, mag = np.zeros((batch, channels)), np.zeros((batch, channels))
    for b in range(batch):
        want[b], mag[b] = R.conv_step(R.history(codes, scales, table[b], lens[b], channels), h64)
    for out_kind, splits in (("f32", 0), ("f32", 2), (kind, 64), ("f16", 3)):
        out = torch.full((batch + 1, channels), 7.0, dtype=torch_type(out_kind), device=dev)
        work = None if splits == 0 else torch.full((splits, batch, channels), float("nan"), device=dev)
        ff.mx4_cache_conv(*args, h, out[:batch], work=work)
        torch.cuda.synchronize()
        assert R.within(out[:batch], want, mag, length + 64, out.dtype)
        assert bool((out[batch] == 7).all())


@pytest.mark.parametrize("kind,bits", [("f16", 11), ("bf16", 8)])
@pytest.mark.parametrize("rule,top", [("fit", 6.0), ("floor", 4.0)])
def test_every_random_byte_at_every_16_bit_magnitude(dev, kind, bits, rule, top):
    """All magnitudes of the type from 2^-24 to 6 (8 under "floor") in units of the block's
    power, under every byte, along rows and along columns."""
    import torch
    import fufft_amd as ff
    end = 6.0 if rule == "fit" else 8.0
    mant = np.arange(1 << (bits - 1), 1 << bits) / (1 << (bits - 1))
    mag = (mant[None] * 2.0 ** np.arange(-24, 3)[:, None]).reshape(-1)
    # for fp16, magnitudes below the type's normal range are in its reach in units of a larger power
    unit = 2.0 ** 10 if kind == "f16" else 1.0
    mag = np.r_[0.0, mag[mag <= end] if rule == "fit" else mag[mag < end]]
    cols = -(-len(mag) // 31) * 32
    row = np.zeros((cols // 32, 32))
    row[:, 0] = top                                              # the block's power is 1
    body = np.zeros(cols // 32 * 31)
    body[:len(mag)] = mag
    row[:, 1:] = body.reshape(-1, 31)
    x64 = np.tile(row.reshape(1, -1) * unit, (256, 1)) * np.where(np.arange(256) % 2, -1.0, 1.0)[:, None]
    x = torch.from_numpy(x64).to(torch_type(kind))
    assert np.array_equal(x.double().numpy(), x64)
    rand = np.repeat(np.arange(256, dtype=np.uint8)[:, None], cols, axis=1)
    codes, scales = R.quantize(x64, rule, rand)
    q = ff.mx4_empty(256, cols)
    dx, drand = x.to(dev), to_dev(dev, rand)[0]
    ff.mx4_quantize(dx, *q, rand=drand, rule=rule)
    torch.cuda.synchronize()
    assert np.array_equal(q[1].cpu().numpy(), scales) and np.array_equal(q[0].cpu().numpy(), codes)
    q = ff.mx4_empty(256, cols)
    ff.mx4_quantize(dx.t().contiguous(), None, None, *q, rand=drand.t().contiguous(), rule=rule)
    torch.cuda.synchronize()
    assert np.array_equal(q[1].cpu().numpy(), scales) and np.array_equal(q[0].cpu().numpy(), codes)
