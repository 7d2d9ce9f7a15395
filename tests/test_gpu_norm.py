"""GPU tests of fufft_rms_norm and fufft_rms_norm_grad against the 64-bit forms of
tests/layer_reference.py, with the bounds of fp32 sums that are derived there."""
import numpy as np
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu

# around every change of a row's lanes and vectors
WIDTHS = [1, 7, 8, 9, 127, 128, 129, 500, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096, 4101, 8192, 8193, 16384, 16391,
          32768, 32775, 65536, 65531]
EPS = 1e-6


def rows_for(k):
    return 5 if k <= 4096 else 2


def signal(rng, rows, k):
    return rng.standard_normal((rows, k)) * 10.0 ** rng.uniform(-2, 2, (rows, 1))


def pool(kind, sum_kind):
    return kind if sum_kind == "same" else "f32"


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("sum_kind", [None, "same", "f32"])
def test_norm(dev, rng, k, kind, sum_kind):
    import torch
    import fufft_amd as ff
    rows = rows_for(k)
    print(f"case norm {rows}x{k} {kind} residual={sum_kind}", flush=True)
    x, x64 = R.typed(signal(rng, rows, k), kind, dev)
    w = torch.from_numpy(rng.standard_normal(k).astype(np.float32)).to(dev) if k % 2 else None
    h, res, total = x64, None, None
    if sum_kind:
        res, r64 = R.typed(signal(rng, rows, k), pool(kind, sum_kind), dev)
        h, total = x64 + r64, torch.empty_like(res)
    want, rel = R.norm(h, None if w is None else w.double().cpu().numpy(), EPS)
    rel += R.EPS24 * (sum_kind is not None)
    out = torch.empty_like(x)
    codes, scales = ff.i8_empty(rows, k)
    codes.fill_(77)
    for view in (x, R.with_stride(x)):
        ff.rms_norm(view, w, out, codes=codes, scales=scales, residual=res, total=total, eps=EPS)
        assert R.inside(out, want, rel * np.abs(want))
        if sum_kind:
            assert R.inside(total, h, R.EPS24 * np.abs(h))
        top = np.abs(want).max(1)
        c, s = codes.cpu().numpy(), scales.double().cpu().numpy()
        assert np.all(np.abs(s - top / 127) <= (rel + 2 * R.EPS24) * top / 127)
        # the code is the nearest to 127 y / max|y|, both known to `rel`
        assert np.all(np.abs(c[:, :k] - 127 * want / np.where(top > 0, top, 1)[:, None]) <= 0.5 + 127 * 2.1 * rel)
        assert not c[:, k:].any()
        # each output alone is the same
        o2, c2, s2 = torch.empty_like(x), torch.empty_like(codes), torch.empty_like(scales)
        ff.rms_norm(view, w, o2, residual=res, eps=EPS)
        ff.rms_norm(view, w, codes=c2, scales=s2, residual=res, eps=EPS)
        assert torch.equal(o2, out) and torch.equal(c2, codes) and torch.equal(s2, scales)


@pytest.mark.parametrize("k", [24, 1000, 3000, 9000])
@pytest.mark.parametrize("kind", R.TYPES)
def test_norm_in_place(dev, rng, k, kind):
    """total in the residual's place, or in x's; out in x's."""
    import torch
    import fufft_amd as ff
    print(f"case norm in place {k} {kind}", flush=True)
    x, _ = R.typed(signal(rng, 6, k), kind, dev)
    res, _ = R.typed(signal(rng, 6, k), kind, dev)
    out, total = torch.empty_like(x), torch.empty_like(x)
    ff.rms_norm(x, None, out, residual=res, total=total)
    a, r = x.clone(), res.clone()
    ff.rms_norm(a, None, a, residual=r, total=r)
    assert torch.equal(a, out) and torch.equal(r, total)
    a = x.clone()
    codes, scales = ff.i8_empty(6, k)
    ff.rms_norm(a, None, codes=codes, scales=scales, residual=res, total=a)
    assert torch.equal(a, total)
    w = R.with_stride(x.clone())
    ff.rms_norm(w, None, w)
    ff.rms_norm(x, None, out)
    assert torch.equal(w, out)


def test_norm_range(dev):
    """Squares beyond fp32's range, up and down, zeros, and rows with NaN or infinities, among
    ordinary ones, which they leave alone."""
    import torch
    import fufft_amd as ff
    for k in (40, 900, 3000, 10000):
        g = torch.Generator().manual_seed(k)
        x = torch.randn(8, k, generator=g)
        x[1] *= 1e30
        x[2] *= 1e-30
        x[3] = 0
        x[4, 3] = float("nan")
        x[5, 7] = float("inf")
        x[6] *= 3e37 / x[6].abs().max()
        d = x.to(dev)
        out = torch.empty_like(d)
        codes, scales = ff.i8_empty(8, k)
        ff.rms_norm(d, None, out, codes=codes, scales=scales, eps=0.0)
        got, c, s = out.cpu(), codes.cpu(), scales.cpu()
        x64 = x.double()
        want = x64 / x64.square().mean(1, keepdim=True).sqrt()
        for r in (0, 1, 2, 6, 7):
            assert R.inside(got[r], want[r].numpy(), (R.ROOT + 6) * R.EPS24 * want[r].abs().numpy()), (k, r)
            assert abs(int(c[r, :k].abs().max())) == 127
        assert got[3].isnan().all()                 # 0 / 0, asked for by eps = 0
        assert got[4].isnan().all() and s[4].isnan() and not c[4].any()
        assert got[5, 7].isnan() and s[5].isnan() and not c[5].any()
        ff.rms_norm(d, None, out, codes=codes, scales=scales)
        assert not out[3].any() and not codes[3].any() and scales[3] == 0


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("sum_kind,through,wide", [("same", False, False), ("same", True, False), ("f32", True, False),
                                                   ("f32", False, True)])
def test_grad(dev, rng, k, kind, sum_kind, through, wide):
    import torch
    import fufft_amd as ff
    print(f"case norm_grad {k} {kind} {sum_kind} through={through} wide={wide}", flush=True)
    for rows, splits in ((rows_for(k), 64), (37 if k <= 8192 else 5, 3)):
        h, h64 = R.typed(signal(rng, rows, k), pool(kind, sum_kind), dev)
        dy, dy64 = R.typed(rng.standard_normal((rows, k)) / 50, kind, dev)
        w = torch.from_numpy(rng.standard_normal(k).astype(np.float32)).to(dev) if k % 2 == 0 else None
        dt, dt64 = R.typed(rng.standard_normal((rows, k)) / 50, pool(kind, sum_kind), dev) if through else (None, None)
        dx64, err, dw64, mags = R.norm_grad(dy64, h64, None if w is None else w.double().cpu().numpy(), dt64, EPS)
        work = torch.full((splits, k), float("nan"), device=dev)
        dw = torch.empty(k, device=dev)
        for strided in (False, True):
            dx = torch.empty(rows, k, dtype=h.dtype if wide else dy.dtype, device=dev)
            view = R.with_stride if strided else (lambda t: t)
            ff.rms_norm_grad(view(dy), view(h), w, dx, dw, work, dtotal=None if dt is None else view(dt), eps=EPS)
            assert R.inside(dx, dx64, err)
            assert R.inside(dw, dw64, R.EPS24 * (R.ROOT + 4 + rows + 40) * mags)
        alone = torch.empty_like(dx)
        ff.rms_norm_grad(dy, h, w, alone, dtotal=dt, eps=EPS)
        assert torch.equal(alone, dx)
        # dx in dy's place, or dtotal's
        if dx.dtype == dy.dtype:
            a = dy.clone()
            ff.rms_norm_grad(a, h, w, a, dtotal=dt, eps=EPS)
            assert torch.equal(a, dx)
        if dt is not None and dx.dtype == dt.dtype:
            a = dt.clone()
            ff.rms_norm_grad(dy, h, w, a, dtotal=a, eps=EPS)
            assert torch.equal(a, dx)


def test_grad_against_differences(dev):
    """dx and dweight against central differences of a sum over the plain form's outputs."""
    import torch
    import fufft_amd as ff
    g = torch.Generator().manual_seed(3)
    h, dy, w = torch.randn(3, 33, generator=g).double(), torch.randn(3, 33, generator=g), torch.randn(33, generator=g)

    def loss(h, w):
        return float((dy.double() * h / (h.square().mean(1, keepdim=True) + 0.1).sqrt() * w).sum())
    dx, dw = torch.empty(3, 33, device=dev), torch.empty(33, device=dev)
    h32 = h.float()
    ff.rms_norm_grad(dy.to(dev), h32.to(dev), w.to(dev), dx, dw, torch.empty(4, 33, device=dev), eps=0.1)
    step = 2.0 ** -17
    for i, j in ((0, 0), (1, 17), (2, 32)):
        e = torch.zeros(3, 33, dtype=torch.float64)
        e[i, j] = step
        # the difference is off by step^2 times a third derivative of a few units, and 2^-53 of the sum over the step
        assert abs((loss(h32.double() + e, w.double()) - loss(h32.double() - e, w.double())) / (2 * step) - float(dx[i, j])) < 1e-5
        e1 = torch.zeros(33, dtype=torch.float64)
        e1[j] = step
        assert abs((loss(h32.double(), w.double() + e1) - loss(h32.double(), w.double() - e1)) / (2 * step) - float(dw[j])) < 1e-5


def test_empty(dev):
    import torch
    import fufft_amd as ff
    x = torch.empty(0, 64, device=dev)
    ff.rms_norm(x, None, torch.empty_like(x))
    dw = torch.full((64,), 5.0, device=dev)
    ff.rms_norm_grad(x, x, None, torch.empty_like(x), dw, torch.empty(2, 64, device=dev))
    assert not dw.any()
    y = torch.empty(4, 0, device=dev)
    ff.rms_norm(y, None, torch.empty_like(y))


def test_many_narrow_rows(dev):
    import torch
    import fufft_amd as ff
    x = torch.randn(300000, 16, device=dev)
    out, dw = torch.empty_like(x), torch.empty(16, device=dev)
    ff.rms_norm(x, None, out)
    want = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    assert float((out.double() - want).abs().max()) < 50 * R.EPS24 * 4
    ff.rms_norm_grad(x, x, None, torch.empty_like(x), dw, torch.empty(512, 16, device=dev))
    terms = x.double() * want
    assert float((dw.double() - terms.sum(0)).abs().max()) < R.EPS24 * float(terms.sum(0).max()) * (300000 / 512 + 100)
